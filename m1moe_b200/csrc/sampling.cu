// sampling.cu — C ABI of the sampler (include/m1moe_cuda.h, m1moe_cuda_sample).
#include <cuda_runtime.h>

#include <algorithm>

#include "m1moe_cuda.h"
#include "sampling.cuh"

// The error helpers and launch counter of m1moe_cuda.cu (one library).
namespace m1abi {
m1moe_status fail(m1moe_status st, const char *fmt, ...);
m1moe_status cuda_fail(cudaError_t e, const char *what);
void count_launch();
}  // namespace m1abi

using m1abi::cuda_fail;
using m1abi::fail;

namespace {
constexpr size_t kDynCap = 184 * 1024;  // dynamic shared memory beside the histograms
}

extern "C" {

m1moe_status m1moe_cuda_sample(const void *d_logits, int32_t dtype, int64_t row_stride, int32_t rows, int32_t vocab,
                               const float *d_u, const float *d_temperature, float temperature,
                               const int32_t *d_top_k, int32_t top_k, const float *d_top_p, float top_p,
                               const float *d_min_p, float min_p, int32_t *d_tokens, void *stream) {
    if (dtype != M1MOE_DTYPE_F32 && dtype != M1MOE_DTYPE_BF16)
        return fail(M1MOE_ERR_INVALID_ARG, "dtype must be F32 (0) or BF16 (1)");
    if (rows < 0 || vocab <= 0 || vocab > (1 << 20))
        return fail(M1MOE_ERR_INVALID_ARG, "rows %d, vocab %d: rows >= 0, vocab 1 to %d", rows, vocab, 1 << 20);
    if (row_stride < vocab) return fail(M1MOE_ERR_INVALID_ARG, "row_stride is below vocab");
    if (!(temperature >= 0.f) || !(top_p >= 0.f) || !(min_p >= 0.f && min_p <= 1.f))
        return fail(M1MOE_ERR_INVALID_ARG, "temperature and top_p must be >= 0, min_p in [0, 1]");
    if (rows == 0) return M1MOE_OK;
    if (!d_logits || !d_u || !d_tokens) return fail(M1MOE_ERR_INVALID_ARG, "NULL pointer");
    m1::SampleParams p{};
    p.logits = d_logits;
    const bool bf16 = dtype == M1MOE_DTYPE_BF16;
    p.stride = row_stride;
    p.vocab = vocab;
    p.u = d_u;
    p.temperature = d_temperature;
    p.top_k = d_top_k;
    p.top_p = d_top_p;
    p.min_p = d_min_p;
    p.temperature1 = temperature;
    p.top_k1 = top_k;
    p.top_p1 = top_p;
    p.min_p1 = min_p;
    p.tokens = d_tokens;
    const size_t size = bf16 ? 2 : 4;
    auto bytes_of = [&](int c) {  // a CTA's slice, 16 bytes of skew, and the own bins of a long one
        const int slice = (vocab + c - 1) / c;
        return ((size_t)slice * size + 16 + 15) / 16 * 16 +
               (slice > m1::kSampleLong ? (size_t)m1::kSampleWide * m1::kSampleThreads * 8 : 0);
    };
    // CTAs per row: enough for the slice to fit in shared memory, while most
    // SMs would be idle, and for short slices where four make them so.  us for
    // 1, 2, 4 and 8 CTAs a row: 192 rows of 32000 f32 95, 81, 73, 176; 256 of
    // 50304 141, 128, 191, 234; one of 50304 35, 15, 12, 10; 48 of 150001 bf16
    // 374, 216, 114, 132.
    int c = 1;
    while (c < m1::kSampleMaxCluster && (bytes_of(c) > kDynCap || (long long)rows * c * 2 <= 74)) c *= 2;
    if (c < 4 && vocab > m1::kSampleLong) c = (vocab + 3) / 4 <= m1::kSampleLong ? 4 : 2;
    if ((long long)rows * c > 0x7FFFFFFFLL) return fail(M1MOE_ERR_UNSUPPORTED, "%d rows are too many", rows);
    p.slice = (vocab + c - 1) / c;
    const bool in_smem = bytes_of(c) <= kDynCap;
    const size_t bytes = in_smem ? bytes_of(c) : (size_t)m1::kSampleWide * m1::kSampleThreads * 8;
    auto kern = bf16 ? (in_smem ? m1::k_sample<uint16_t, true> : m1::k_sample<uint16_t, false>)
                       : (in_smem ? m1::k_sample<float, true> : m1::k_sample<float, false>);
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kDynCap);
    if (e != cudaSuccess) return cuda_fail(e, "k_sample shared memory");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * c);
    cfg.blockDim = dim3(m1::kSampleThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = c;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return cuda_fail(e, "k_sample launch");
    m1abi::count_launch();
    return M1MOE_OK;
}

}  // extern "C"
