// paged.cu — C ABI of the paged key/value cache (include/m1moe_cuda.h,
// m1moe_cuda_paged_*): the batch plan, the append of new tokens and the
// attention over the pages.  Stateless: the caller owns the pools, the page
// table and the plan buffer.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <utility>

#include "m1moe_cuda.h"
#include "paged.cuh"
#include "paged_rows16.cuh"
#include "paged_rows256.cuh"

// The error helpers and launch counter of m1moe_cuda.cu (one library).
namespace m1abi {
m1moe_status fail(m1moe_status st, const char *fmt, ...);
m1moe_status cuda_fail(cudaError_t e, const char *what);
void count_launch();
m1moe_status paged_last_rows(const m1moe_paged_cfg *cfg, void *d_plan, const float *x, int h, float *out,
                             cudaStream_t st);
}  // namespace m1abi

using m1abi::cuda_fail;
using m1abi::fail;

namespace {

#define P_CK(call)                                          \
    do {                                                    \
        cudaError_t e_ = (call);                            \
        if (e_ != cudaSuccess) return cuda_fail(e_, #call); \
    } while (0)

inline cudaStream_t as_stream(void *s) { return reinterpret_cast<cudaStream_t>(s); }

template <typename... KArgs, typename... Args>
m1moe_status launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const char *what,
                        Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
    if (e != cudaSuccess) return cuda_fail(e, what);
    m1abi::count_launch();
    return M1MOE_OK;
}

int sm_count(int *out) {
    static thread_local int cached_dev = -1, cached = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    if (dev != cached_dev) {
        if (cudaDeviceGetAttribute(&cached, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
        cached_dev = dev;
    }
    *out = cached;
    return 0;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The kernels' shape, checked; `ctas` = SMs.
m1moe_status make_shape(const m1moe_paged_cfg *c, int ctas, m1::PagedShape &s) {
    if (!c) return fail(M1MOE_ERR_INVALID_ARG, "cfg is NULL");
    if (c->num_heads <= 0 || c->num_kv_heads <= 0 || c->num_heads % c->num_kv_heads)
        return fail(M1MOE_ERR_INVALID_ARG, "%d heads over %d KV heads: positive, a multiple", c->num_heads,
                    c->num_kv_heads);
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(M1MOE_ERR_UNSUPPORTED, "head_dim %d: 64 or 128", c->head_dim);
    const int group = c->num_heads / c->num_kv_heads;
    if (group > 16) return fail(M1MOE_ERR_UNSUPPORTED, "%d heads per KV head: at most 16", group);
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return fail(M1MOE_ERR_UNSUPPORTED, "page_size %d: a power of two, 16 to 1024", c->page_size);
    if (c->num_pages <= 0 || c->num_seqs <= 0 || c->max_pages_per_seq <= 0 || c->total_q < 0 || c->max_q < 0)
        return fail(M1MOE_ERR_INVALID_ARG, "pages, sequences and pages per sequence must be positive, tokens >= 0");
    if (c->max_q > c->total_q || (long long)c->max_q * c->num_seqs < c->total_q)
        return fail(M1MOE_ERR_INVALID_ARG, "max_q %d does not fit %d tokens of %d sequences", c->max_q, c->total_q,
                    c->num_seqs);
    if (c->window < 0 || c->shared_prefix < 0 || c->shared_prefix % c->page_size)
        return fail(M1MOE_ERR_INVALID_ARG, "window %d must be >= 0, shared_prefix %d a multiple of the page size",
                    c->window, c->shared_prefix);
    // (each product of 32-bit sizes is compared before the next factor joins it)
    if ((long long)c->num_pages * c->page_size > 0x7FFFFFFFLL / c->num_kv_heads ||
        (long long)c->max_pages_per_seq * c->page_size > 0x7FFFFF00LL)
        return fail(M1MOE_ERR_UNSUPPORTED, "the pool's rows and a sequence's positions must fit 31 bits");
    if (c->shared_prefix > (long long)c->max_pages_per_seq * c->page_size)
        return fail(M1MOE_ERR_INVALID_ARG, "shared_prefix %d is longer than a page table row", c->shared_prefix);
    s = m1::PagedShape{};
    s.nh = c->num_heads;
    s.nkv = c->num_kv_heads;
    s.group = group;
    s.by_group = m1::make_fastdiv(group);
    s.hd = c->head_dim;
    s.page_size = c->page_size;
    while ((1 << s.page_shift) < c->page_size) ++s.page_shift;
    s.num_pages = c->num_pages;
    s.num_seqs = c->num_seqs;
    s.max_pages = c->max_pages_per_seq;
    s.total_q = c->total_q;
    s.max_q = c->max_q;
    s.window = c->window;
    s.ctas = ctas;
    // 16-row items while a sequence's rows fit one, 256-row ones beyond (64
    // decode sequences: 113 us with 16 rows; a 8192-token prompt: 4226 us with
    // 16 rows, 518 with 256)
    const bool small = (long long)group * c->max_q <= m1::kPagedRowsSmall;
    s.rows = small ? m1::kPagedRowsSmall : m1::kPagedRowsLarge;
    s.unit = small ? m1::kPagedUnitSmall : m1::kPagedUnitLarge;
    s.workers = small ? ctas * m1::kPagedWarps : ctas;
    s.min_per = small ? m1::kPagedWarps : 1;
    const long long items = c->num_seqs + (long long)c->total_q * group / s.rows;
    const long long cap = (long long)c->max_pages_per_seq * c->page_size;
    if (items * (cap / s.unit + 1 + m1::kPagedItemCost) > 0x7FFF0000LL / c->num_kv_heads)
        return fail(M1MOE_ERR_UNSUPPORTED, "the batch's work (%lld items of up to %lld positions) does not fit 31 bits",
                    items, cap);
    s.max_items = (int)items;
    // A prefix is shared where reading it once saves 200 MB of reads: the extra
    // pass and its partials cost what those take from L2 (us without and with
    // it, n sequences over a prefix: 4 over 1504, 16/16 heads, 37 MB: 18 and 28;
    // 16, 185 MB: 34.8 and 35.3; 32, 382 MB: 58.9 and 37.1; 24 over 2048, 32/8
    // heads, 193 MB: 35.1 and 35.8; 8 over 8192, 235 MB: 42.5 and 40.7; 200 over
    // 16384, 53 GB: 1549 and 195).
    // Its pass takes 16-row items up to 128 rows a KV head, 256-row ones beyond
    // (16-row and 256-row, 32/8 heads over 4096: 64 rows 39.7 and 45.4 us, 128
    // rows 46.1 and 46.2, 256 rows 70.1 and 58.6).
    // The plan keeps room for the pass whenever a prefix is named, so that its
    // size does not jump as sequences join the batch.
    s.prefix_room = small && c->window == 0 && c->num_seqs > 1 && c->shared_prefix > 0;
    const long long saved = (long long)(c->num_seqs - 1) * c->shared_prefix * c->num_kv_heads * c->head_dim * 4;
    s.prefix = s.prefix_room && saved >= 200000000LL ? c->shared_prefix : 0;
    s.prefix_rows = (long long)c->total_q * group > 128 ? m1::kPagedRowsLarge : m1::kPagedRowsSmall;
    return M1MOE_OK;
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// The plan's arrays in its buffer: the main split and, with a shared prefix,
// the prefix's; returns the buffer's bytes.
size_t plan_view(const m1::PagedShape &s, void *base, m1::PagedPlanView &v, m1::PagedPlanView &v2,
                 m1::PagedPrefixView &pre) {
    uint8_t *b = static_cast<uint8_t *>(base);
    size_t at = 0;
    auto take = [&](auto *&ptr, size_t bytes) {
        ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(b + at);
        at = align256(at + bytes);
    };
    const bool large = s.rows == m1::kPagedRowsLarge;
    const size_t part_rows = large ? s.rows : std::max(1, s.group * s.max_q);
    take(v.header, m1::kPhWords * 4);
    v.status = v.header + m1::kPhStatus;
    take(v.cu_q, (size_t)(s.num_seqs + 1) * 4);
    take(v.kv_len, (size_t)s.num_seqs * 4);
    take(v.tokens, (size_t)s.total_q * 8);
    take(v.items, (size_t)s.max_items * sizeof(m1::PagedItem));
    take(v.item_at, (size_t)(s.num_seqs + 1) * 4);
    take(v.unit_at, (size_t)(s.max_items + 1) * 4);
    take(v.start, (size_t)s.workers * 4);
    take(v.count, large ? 0 : (size_t)s.nkv * s.max_items * 4);
    take(v.part_ml, (size_t)2 * s.ctas * part_rows * 8);
    take(v.part, (size_t)2 * s.ctas * part_rows * s.hd * 4);
    v2 = v;
    if (!s.prefix_room) return at;
    const size_t rows2 = s.prefix_rows, items2 = ((size_t)s.total_q * s.group + rows2 - 1) / rows2;
    const bool small2 = s.prefix_rows == m1::kPagedRowsSmall;
    take(v2.header, m1::kPhWords * 4);
    take(v2.items, items2 * sizeof(m1::PagedItem));
    take(v2.unit_at, (items2 + 1) * 4);
    take(v2.start, (size_t)s.ctas * 4 * (small2 ? m1::kPagedWarps : 1));
    take(v2.count, small2 ? (size_t)s.nkv * items2 * 4 : 0);
    take(v2.part_ml, (size_t)2 * s.ctas * rows2 * 8);
    take(v2.part, (size_t)2 * s.ctas * rows2 * s.hd * 4);
    take(pre.ml, (size_t)s.total_q * s.nh * 8);
    take(pre.part, (size_t)s.total_q * s.nh * s.hd * 4);
    return at;
}

struct Plan {
    m1::PagedShape s;
    m1::PagedPlanView v, v2;
    m1::PagedPrefixView pre;
    size_t bytes;
};

m1moe_status open_plan(const m1moe_paged_cfg *cfg, void *d_plan, Plan &p) {
    int sms = 0;
    if (sm_count(&sms)) return fail(M1MOE_ERR_CUDA, "no CUDA device");
    p = Plan{};
    if (m1moe_status st = make_shape(cfg, sms, p.s)) return st;
    if (!d_plan || (reinterpret_cast<uintptr_t>(d_plan) & 255))
        return fail(M1MOE_ERR_INVALID_ARG, "the plan buffer is NULL or not 256-byte aligned");
    p.bytes = plan_view(p.s, d_plan, p.v, p.v2, p.pre);
    return M1MOE_OK;
}

constexpr size_t kRows16SmemCap = 224 * 1024;  // of the CTA's 227 KB; the rest is static

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A pool as rows of hd elements; a box is 64 columns of a page's rows (128 at
// most), 128-byte swizzled.
m1moe_status pool_map(const m1::PagedShape &s, const uint16_t *pool, CUtensorMap *map) {
    static const EncodeTiledFn encode = []() -> EncodeTiledFn {  // one address for the process
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q{};
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
        return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(fn) : nullptr;
    }();
    if (!encode) return fail(M1MOE_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[2] = {(cuuint64_t)s.hd, (cuuint64_t)s.num_pages * s.nkv * s.page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)s.hd * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)std::min(s.page_size, m1::kPagedUnitLarge)}, one[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t *>(pool), dims, strides, box,
                              one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(M1MOE_ERR_CUDA, "page pool tensor map: error %d", (int)r);
    return M1MOE_OK;
}

template <int HD>
m1moe_status launch_rows256(const m1::PagedShape &s, const m1::PagedPlanView &v, const m1::RowsParams &r,
                            const m1::PagedPrefixView *pre, cudaStream_t st) {
    m1::Rows256Params a{};
    a.r = r;
    if (pre) {
        a.prefix_run = 1;
        a.partial = pre->part;
        a.partial_ml = pre->ml;
    }
    CUtensorMap kmap, vmap;
    if (m1moe_status e = pool_map(s, r.k, &kmap)) return e;
    if (m1moe_status e = pool_map(s, r.v, &vmap)) return e;
    auto kern = m1::k_paged_rows256<HD>;
    constexpr int smem = m1::Rows256<HD>::kSmem;
    // the register split of the warpgroups waits for ever if the block is
    // launched with fewer registers than it hands out
    static const int regs = [] {
        cudaFuncAttributes at{};
        return cudaFuncGetAttributes(&at, m1::k_paged_rows256<HD>) == cudaSuccess ? at.numRegs : 0;
    }();
    if (regs * m1::kRows256Threads < 128 * 2 * (m1::kRegsSoftmax + m1::kRegsOther))
        return fail(M1MOE_ERR_CUDA, "k_paged_rows256 was built with %d registers", regs);
    P_CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (m1moe_status e = launch_pdl(kern, dim3(s.ctas), dim3(m1::kRows256Threads), (size_t)smem, st,
                                    "k_paged_rows256 launch", s, v, a, kmap, vmap))
        return e;
    return launch_pdl(m1::k_paged_join<HD>, dim3(std::max(1, s.ctas - 1), 2, HD / 32), dim3(m1::kTileRows), 0, st,
                      "k_paged_join launch", s, v, a);
}

template <int HD, bool kCap, bool kMany>
m1moe_status launch_rows16(const m1::PagedShape &s, const m1::PagedPlanView &v, m1::RowsParams a, cudaStream_t st) {
    // the ring takes what the partials' rows leave, 2 to 4 stages a warp
    const int unit = m1::rows16_unit_bytes<HD>(), part = a.part_rows * HD * 4;
    const int budget = (int)(kRows16SmemCap / m1::kPagedWarps);
    a.stages = std::min(4, (budget - part) / unit);
    const size_t smem = (size_t)m1::kPagedWarps * (a.stages * unit + part);
    auto kern = m1::k_paged_rows16<HD, kCap, kMany>;
    P_CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRows16SmemCap));
    return launch_pdl(kern, dim3(s.ctas), dim3(m1::kPagedWarps * 32), smem, st, "k_paged_rows16 launch", s, v, a);
}

template <int HD>
m1moe_status launch_rows16(const m1::PagedShape &s, const m1::PagedPlanView &v, const m1::RowsParams &a,
                           cudaStream_t st) {
    const bool many = s.max_q > 1 && !a.partial;  // (all rows see all of a shared prefix)
    if (a.cap > 0.f) return many ? launch_rows16<HD, true, true>(s, v, a, st) : launch_rows16<HD, true, false>(s, v, a, st);
    return many ? launch_rows16<HD, false, true>(s, v, a, st) : launch_rows16<HD, false, false>(s, v, a, st);
}

template <int HD>
m1moe_status attention(const Plan &p, m1::RowsParams a, cudaStream_t st) {
    if (p.s.rows == m1::kPagedRowsLarge) return launch_rows256<HD>(p.s, p.v, a, nullptr, st);
    if (p.s.prefix > 0) {
        // one partial per row over the prefix, then the sequences' own parts
        m1::RowsParams b = a;
        b.part_rows = m1::kPagedRowsSmall;
        b.partial = p.pre.part;
        b.partial_ml = p.pre.ml;
        if (m1moe_status e = p.s.prefix_rows == m1::kPagedRowsLarge ? launch_rows256<HD>(p.s, p.v2, a, &p.pre, st)
                                                                    : launch_rows16<HD>(p.s, p.v2, b, st))
            return e;
        a.prefix_part = p.pre.part;
        a.prefix_ml = p.pre.ml;
    }
    return launch_rows16<HD>(p.s, p.v, a, st);
}

}  // namespace

// The last new token's row of each sequence (for dense.cu).
m1moe_status m1abi::paged_last_rows(const m1moe_paged_cfg *cfg, void *d_plan, const float *x, int h, float *out,
                                    cudaStream_t st) {
    Plan p;
    if (m1moe_status e = open_plan(cfg, d_plan, p)) return e;
    return launch_pdl(m1::k_paged_last, dim3(p.s.num_seqs), dim3(256), 0, st, "k_paged_last launch", p.v, x, h, out);
}

extern "C" {

size_t m1moe_cuda_paged_plan_bytes(const m1moe_paged_cfg *cfg) {
    int sms = 0;
    if (sm_count(&sms)) {
        cudaGetLastError();
        sms = 148;
    }
    Plan p{};
    if (make_shape(cfg, sms, p.s)) return 0;
    return plan_view(p.s, nullptr, p.v, p.v2, p.pre);
}

m1moe_status m1moe_cuda_paged_plan(const m1moe_paged_cfg *cfg, const int32_t *d_cu_q, const int32_t *d_kv_len,
                                   const int32_t *d_page_table, void *d_plan, size_t plan_bytes, void *stream) {
    if (!d_cu_q || !d_kv_len || !d_page_table) return fail(M1MOE_ERR_INVALID_ARG, "NULL pointer");
    Plan p;
    if (m1moe_status st = open_plan(cfg, d_plan, p)) return st;
    if (plan_bytes < p.bytes)
        return fail(M1MOE_ERR_INVALID_ARG, "plan buffer: %zu bytes, %zu needed", plan_bytes, p.bytes);
    const m1::PagedShape &s = p.s;
    const m1::PagedPlanView &v = p.v;
    if (m1moe_status st = launch_pdl(m1::k_paged_plan, dim3(1), dim3(1024), 0, as_stream(stream), "k_paged_plan launch",
                                     s, v, (const int *)d_cu_q, (const int *)d_kv_len, (const int *)d_page_table, p.v2))
        return st;
    if (s.total_q == 0) return M1MOE_OK;
    return launch_pdl(m1::k_paged_tokens, dim3((s.total_q + 255) / 256), dim3(256), 0, as_stream(stream),
                      "k_paged_tokens launch", s, v);
}

m1moe_status m1moe_cuda_paged_append(const m1moe_paged_cfg *cfg, const void *d_plan, const int32_t *d_page_table,
                                     const void *d_qkv, int32_t qkv_dtype, int64_t qkv_stride,
                                     const uint16_t *d_q_norm, const uint16_t *d_k_norm, float eps,
                                     const float *d_rope, int32_t rope_rows, int32_t rot_dim, int32_t rope_pairs,
                                     uint16_t *d_k_pages, uint16_t *d_v_pages, uint16_t *d_q_out, void *stream) {
    if (!d_page_table || !d_qkv || !d_rope || !d_k_pages || !d_v_pages || !d_q_out)
        return fail(M1MOE_ERR_INVALID_ARG, "NULL pointer");
    if (qkv_dtype != M1MOE_DTYPE_F32 && qkv_dtype != M1MOE_DTYPE_BF16)
        return fail(M1MOE_ERR_INVALID_ARG, "dtype must be F32 (0) or BF16 (1)");
    Plan p;
    if (m1moe_status st = open_plan(cfg, const_cast<void *>(d_plan), p)) return st;
    const m1::PagedShape &s = p.s;
    const m1::PagedPlanView &v = p.v;
    const int heads = s.nh + 2 * s.nkv;
    const bool bf = qkv_dtype == M1MOE_DTYPE_BF16;
    if (qkv_stride < (int64_t)heads * s.hd || qkv_stride % (bf ? 8 : 4))
        return fail(M1MOE_ERR_INVALID_ARG, "qkv_stride %lld: at least %d, in whole 16 bytes", (long long)qkv_stride,
                    heads * s.hd);
    if (rot_dim < 0 || rot_dim > s.hd || rot_dim % 16)
        return fail(M1MOE_ERR_UNSUPPORTED, "rot_dim %d: a multiple of 16 up to head_dim %d", rot_dim, s.hd);
    if (rope_rows <= 0) return fail(M1MOE_ERR_INVALID_ARG, "the rotation table has no rows");
    for (const void *ptr : {d_qkv, (const void *)d_rope, (const void *)d_k_pages, (const void *)d_v_pages,
                            (const void *)d_q_out, (const void *)d_q_norm, (const void *)d_k_norm})
        if (!aligned16(ptr)) return fail(M1MOE_ERR_INVALID_ARG, "pointers must be 16-byte aligned");
    if (s.total_q == 0) return M1MOE_OK;
    m1::AppendParams a{};
    a.qkv = d_qkv;
    a.qkv_stride = qkv_stride;
    a.q_norm = d_q_norm;
    a.k_norm = d_k_norm;
    a.eps = eps;
    a.rope = reinterpret_cast<const float2 *>(d_rope);
    a.rope_rows = rope_rows;
    a.rot = rot_dim;
    a.pairs = rope_pairs != 0;
    a.k = d_k_pages;
    a.v = d_v_pages;
    a.q_out = d_q_out;
    a.table = d_page_table;
    // one head a group of lanes while that leaves SMs idle, up to 4 (a token's
    // place and angles are then looked up once for them)
    const int L = s.hd / 8;
    const long long lanes = (long long)s.total_q * heads * L;
    if (lanes > (1LL << 38)) return fail(M1MOE_ERR_UNSUPPORTED, "%d tokens are too many for one call", s.total_q);
    a.heads_per_group = (int)std::min<long long>(4, std::max<long long>(1, lanes / (s.ctas * 2048LL * 2)));
    a.groups = (heads + a.heads_per_group - 1) / a.heads_per_group;
    const dim3 grid((unsigned)(((long long)s.total_q * a.groups * L + 255) / 256));
    auto kern = s.hd == 128 ? (bf ? m1::k_paged_append<128, true> : m1::k_paged_append<128, false>)
                            : (bf ? m1::k_paged_append<64, true> : m1::k_paged_append<64, false>);
    return launch_pdl(kern, grid, dim3(256), 0, as_stream(stream), "k_paged_append launch", s, v, a);
}

m1moe_status m1moe_cuda_paged_attention(const m1moe_paged_cfg *cfg, void *d_plan, const int32_t *d_page_table,
                                        const uint16_t *d_q, int64_t q_stride, const uint16_t *d_k_pages,
                                        const uint16_t *d_v_pages, float scale, float softcap, void *d_out,
                                        int32_t out_dtype, int64_t out_stride, void *stream) {
    if (!d_page_table || !d_q || !d_k_pages || !d_v_pages || !d_out)
        return fail(M1MOE_ERR_INVALID_ARG, "NULL pointer");
    if (out_dtype != M1MOE_DTYPE_F32 && out_dtype != M1MOE_DTYPE_BF16)
        return fail(M1MOE_ERR_INVALID_ARG, "dtype must be F32 (0) or BF16 (1)");
    Plan p;
    if (m1moe_status st = open_plan(cfg, d_plan, p)) return st;
    const m1::PagedShape &s = p.s;
    const int64_t width = (int64_t)s.nh * s.hd;
    if (q_stride < width || q_stride % 8 || out_stride < width || out_stride % 8)
        return fail(M1MOE_ERR_INVALID_ARG, "q and out strides: at least %lld, multiples of 8 elements",
                    (long long)width);
    if (!(scale > 0.f) || !std::isfinite(scale) || !(softcap >= 0.f) || !std::isfinite(softcap))
        return fail(M1MOE_ERR_INVALID_ARG, "scale must be positive and softcap >= 0, both finite");
    for (const void *ptr : {(const void *)d_q, (const void *)d_k_pages, (const void *)d_v_pages, (const void *)d_out})
        if (!aligned16(ptr)) return fail(M1MOE_ERR_INVALID_ARG, "pointers must be 16-byte aligned");
    if (s.total_q == 0) return M1MOE_OK;
    m1::RowsParams a{};
    a.q = d_q;
    a.q_stride = q_stride;
    a.k = d_k_pages;
    a.v = d_v_pages;
    a.table = d_page_table;
    a.scale = scale;
    a.cap = softcap;
    a.out = d_out;
    a.out_bf16 = out_dtype == M1MOE_DTYPE_BF16;
    a.out_stride = out_stride;
    a.part_rows = std::min(s.rows, s.group * s.max_q);
    return s.hd == 128 ? attention<128>(p, a, as_stream(stream)) : attention<64>(p, a, as_stream(stream));
}

m1moe_status m1moe_cuda_paged_status(void *d_plan, void *stream) {
    if (!d_plan) return fail(M1MOE_ERR_INVALID_ARG, "NULL pointer");
    int word = 0;
    P_CK(cudaMemcpyAsync(&word, d_plan, 4, cudaMemcpyDeviceToHost, as_stream(stream)));
    P_CK(cudaStreamSynchronize(as_stream(stream)));
    if (!word) return M1MOE_OK;
    P_CK(cudaMemsetAsync(d_plan, 0, 4, as_stream(stream)));
    P_CK(cudaStreamSynchronize(as_stream(stream)));
    return fail(M1MOE_ERR_DEVICE, "paged batch status 0x%x (1: lengths out of range, 2: a page id outside the pool, "
                                  "4: a position outside the rotation table, 8: a wait gave up)", word);
}

}  // extern "C"
