// sampling.cuh — the next token of each logit row by temperature, top-k,
// top-p and min-p from one given uniform number per row (sm_100a).
//
// A token's weight is the whole number w = floor(2^36 exp((l - max) / T)), so
// every sum below is a sum of integers: exact, and the same whatever order
// threads add in.  Tokens rank by logit, equal logits by index.  Kept are
// the top_k first; of these the shortest run of first ones whose weight
// reaches top_p of theirs; of these the ones with exp(...) >= min_p.  The
// token is the first by index whose running kept weight exceeds u of the
// kept weight.  Both cuts are a (key, how many tokens of exactly that key)
// pair, found without sorting: a histogram of counts and weights over 512
// bins of the distance to the maximum, the bin in which the cut falls, and
// then the same over the keys of that bin, 512 at a time, until one key is
// left (two rounds for logits of ordinary size).
//
// A cluster of CTAs shares a row: each keeps its slice in shared memory
// (read from HBM once) and makes its own histogram; after one cluster
// barrier every CTA adds up all of them through distributed shared memory
// and draws the same conclusions, so nothing is broadcast.  A bin's weight
// is held as two 18-bit limbs in 32-bit words (native shared-memory
// atomics), folded into 64-bit registers every 8192 tokens, before a limb
// could overflow.
#pragma once

#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "pipeline.cuh"

namespace m1 {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = kSampleThreads;  // a thread per bin
constexpr int kSampleFold = 8192;            // tokens between folds: 8192 * 2^18 < 2^32
constexpr float kSampleSpan = 25.f;          // exp(-25) * 2^36 < 1: beyond it every weight is 0
constexpr int kSampleMaxCluster = 8;

struct SampleParams {
    const void *logits;
    int bf16;
    long long stride;  // elements between rows
    int vocab, slice;  // slice: tokens per CTA of the cluster
    int in_smem;       // the slice fits in shared memory
    const float *u;
    const float *temperature, *top_p, *min_p;  // per row, or NULL: the scalar below
    const int *top_k;
    float temperature1, top_p1, min_p1;
    int top_k1;
    int *tokens;
};

// Monotone map of a float (no NaN) to unsigned, +0 and -0 alike.
__device__ __forceinline__ uint32_t sample_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// floor(total * f / 2^24) for total < 2^60 and f <= 2^24.
__device__ __forceinline__ unsigned long long mul24(unsigned long long total, uint32_t f) {
    return (total >> 24) * f + (((total & 0xFFFFFFu) * f) >> 24);
}

struct SampleShared {
    uint32_t hist[3][3][kSampleBins];  // three buffers in turn of counts, low and high limbs
    float red_v[kSampleWarps];
    int red_i[kSampleWarps];
    float cta_top;
    int cta_arg;
    unsigned long long scan_w[kSampleWarps];
    uint32_t scan_n[kSampleWarps];
    unsigned long long above_w, bin_w;
    uint32_t above_n, bin_n;
    int bin;
    unsigned long long cta_w;  // kept weight above the cut, and
    uint32_t cta_n;            // tokens of the cut's key, of this CTA
    unsigned long long warp_w[kSampleWarps];
    uint32_t warp_n[kSampleWarps];
};

// Inclusive scan over the block of (n, w), in thread order.
__device__ __forceinline__ void sample_scan(SampleShared &sm, uint32_t &n, unsigned long long &w) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, n, o);
        const unsigned long long b = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) n += a, w += b;
    }
    __syncthreads();
    if (lane == 31) sm.scan_n[warp] = n, sm.scan_w[warp] = w;
    __syncthreads();
    uint32_t pn = 0;
    unsigned long long pw = 0;
    for (int i = 0; i < warp; ++i) pn += sm.scan_n[i], pw += sm.scan_w[i];
    n += pn;
    w += pw;
}

__global__ void __launch_bounds__(kSampleThreads) k_sample(const SampleParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ float slice[];
    __shared__ SampleShared sm;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / C;
    pdl_wait();
    const int i0 = min(p.vocab, rank * p.slice), n = min(p.vocab, i0 + p.slice) - i0;
    const long long base = (long long)row * p.stride + i0;
    auto fetch = [&](int i) {
        float v = load_act(p.logits, p.bf16, (size_t)(base + i));
        return v != v ? -INFINITY : v;  // NaN: never chosen
    };
    auto logit = [&](int i) { return p.in_smem ? slice[i] : fetch(i); };

    // 1. the largest logit and its first index
    float best = -INFINITY;
    int arg = 0x7FFFFFFF;
    for (int i = tid; i < n; i += kSampleThreads) {
        const float v = fetch(i);
        if (p.in_smem) slice[i] = v;
        if (v > best) best = v, arg = i0 + i;
    }
    auto better = [](float v, int a, float &bv, int &ba) {
        if (v > bv || (v == bv && a < ba)) bv = v, ba = a;
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, arg, o), best, arg);
    if (lane == 0) sm.red_v[warp] = best, sm.red_i[warp] = arg;
    for (int b = 0; b < 3; ++b)
        for (int k = 0; k < 3; ++k) sm.hist[b][k][tid] = 0;
    __syncthreads();
    if (tid == 0) {
        for (int w = 0; w < kSampleWarps; ++w) better(sm.red_v[w], sm.red_i[w], best, arg);
        sm.cta_top = best;
        sm.cta_arg = arg;
    }
    cluster.sync();
    float top = -INFINITY;
    arg = 0x7FFFFFFF;
    for (int c = 0; c < C; ++c) {
        const SampleShared *o = cluster.map_shared_rank(&sm, c);
        better(o->cta_top, o->cta_arg, top, arg);
    }
    const float temp = p.temperature ? p.temperature[row] : p.temperature1;
    if (top == -INFINITY || !(temp > 0.f)) {  // nothing to choose from; greedy
        if (rank == 0 && tid == 0) p.tokens[row] = top == -INFINITY ? -1 : arg;
        cluster.sync();  // no CTA leaves while another reads its shared memory
        return;
    }
    const int k = p.top_k ? p.top_k[row] : p.top_k1;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p1;
    float min_p = p.min_p ? p.min_p[row] : p.min_p1;
    if (!(min_p <= 1.f)) min_p = 1.f;  // the largest logit always stays
    const float inv_t = 1.0f / temp, u = p.u[row];
    const uint32_t part = top_p >= 1.f ? 1u << 24 : (top_p > 0.f ? (uint32_t)(top_p * 16777216.f) : 0u);
    const uint32_t uf = u > 0.f ? min((uint32_t)(fminf(u, 1.f) * 16777216.f), 0xFFFFFFu) : 0u;
    auto prob = [&](float l) { return l == top ? 1.f : expf((l - top) * inv_t); };
    auto weight = [&](float e) { return (unsigned long long)(e * 68719476736.f); };
    const float bin_scale = inv_t * ((float)kSampleBins / kSampleSpan);
    // monotone in l; the last bin takes the rest
    auto bin_of = [&](float l) { return l == top ? 0 : (int)fminf((top - l) * bin_scale, (float)(kSampleBins - 1)); };

    // One histogram round over the tokens that sel accepts (their bin, or -1):
    // afterwards thread t holds the row's count and weight of bin t.
    int round = 0;
    auto histogram = [&](auto sel, uint32_t &cnt, unsigned long long &wt) {
        const int b = round % 3;
        uint32_t(*h)[kSampleBins] = sm.hist[b];
        unsigned long long fold_w = 0;
        for (int a = 0; a < n; a += kSampleFold) {
            const int e = min(n, a + kSampleFold);
            for (int i = a + tid; i < e; i += kSampleThreads) {
                const float l = logit(i);
                const int j = sel(l);
                if (j < 0) continue;
                const unsigned long long w = weight(prob(l));
                if (w == 0) continue;
                atomicAdd(&h[0][j], 1u);
                atomicAdd(&h[1][j], (uint32_t)(w & 0x3FFFFu));
                atomicAdd(&h[2][j], (uint32_t)(w >> 18));
            }
            __syncthreads();
            fold_w += (unsigned long long)h[1][tid] + ((unsigned long long)h[2][tid] << 18);
            h[1][tid] = h[2][tid] = 0;
            __syncthreads();
        }
        h[1][tid] = (uint32_t)fold_w;
        h[2][tid] = (uint32_t)(fold_w >> 32);
        // clear the next round's buffer: it was last read two rounds ago, and
        // every CTA has passed the barrier of the last round since
        for (int q = 0; q < 3; ++q) sm.hist[(round + 1) % 3][q][tid] = 0;
        cluster.sync();
        cnt = 0;
        wt = 0;
        for (int c = 0; c < C; ++c) {
            const uint32_t(*o)[kSampleBins] = cluster.map_shared_rank(&sm, c)->hist[b];
            cnt += o[0][tid];
            wt += (unsigned long long)o[1][tid] | ((unsigned long long)o[2][tid] << 32);
        }
        ++round;
    };
    // The first bin at which the running count or weight (on top of `above`)
    // reaches the goal; false if none does.
    auto cross = [&](uint32_t cnt, unsigned long long wt, uint32_t above_n, unsigned long long above_w, bool by_count,
                     unsigned long long goal) {
        uint32_t in = cnt;
        unsigned long long iw = wt;
        if (tid == 0) sm.bin = -1;
        sample_scan(sm, in, iw);  // its barriers order the line above
        const unsigned long long now = by_count ? above_n + in : above_w + iw;
        const unsigned long long before = by_count ? above_n + in - cnt : above_w + iw - wt;
        if (now >= goal && before < goal) {
            sm.bin = tid;
            sm.above_n = above_n + in - cnt;
            sm.above_w = above_w + iw - wt;
            sm.bin_n = cnt;
            sm.bin_w = wt;
        }
        __syncthreads();
        return sm.bin >= 0;
    };
    // The cut's key and how many tokens of that key it takes.
    struct Cut {
        uint32_t key, quota;
        uint32_t above_n;
        unsigned long long above_w, key_w;  // above the key, and one token of the key
    };
    auto refine = [&](bool by_count, unsigned long long goal) {
        // sm.bin, sm.above_*: the bin of the first histogram
        const int bin = sm.bin;
        const uint32_t an0 = sm.above_n;
        const unsigned long long aw0 = sm.above_w;
        uint32_t an = an0;
        unsigned long long aw = aw0;
        // keys of the bin, a little wider than its edges' rounding
        const float hi_l = fminf(top, top - (float)bin / bin_scale * (1.f - 1e-5f) + 1e-5f * fabsf(top));
        const float lo_l = bin == kSampleBins - 1 ? -INFINITY
                                                   : top - (float)(bin + 1) / bin_scale * (1.f + 1e-5f) - 1e-5f * fabsf(top);
        uint32_t khi = sample_key(hi_l), klo = sample_key(lo_l);
        if (isinf(top)) khi = klo = sample_key(top);  // only the tokens at +inf weigh anything
        // at most one round that misses and then four of 9 bits each
        for (int i = 0; i < 8; ++i) {
            const int bits = 32 - __clz((khi - klo) | 1u);
            const int shift = max(0, bits - 9);  // 512 bins
            uint32_t cnt;
            unsigned long long wt;
            histogram(
                [&](float l) {
                    const uint32_t key = sample_key(l);
                    if (key > khi || key < klo || bin_of(l) != bin) return -1;
                    return (int)((khi - key) >> shift);
                },
                cnt, wt);
            if (!cross(cnt, wt, an, aw, by_count, goal)) {
                // the estimated key range missed the cut: take all keys
                an = an0;
                aw = aw0;
                khi = 0xFFFFFFFFu;
                klo = 0u;
                __syncthreads();
                continue;
            }
            const int j = sm.bin;
            an = sm.above_n;
            aw = sm.above_w;
            khi -= (uint32_t)j << shift;
            if (shift == 0) {
                Cut c;
                c.key = khi;
                c.above_n = an;
                c.above_w = aw;
                c.key_w = sm.bin_n ? sm.bin_w / sm.bin_n : 0;
                const unsigned long long need = goal - (by_count ? an : aw);
                c.quota = (uint32_t)(by_count ? need : (need + c.key_w - 1) / max(c.key_w, 1ull));
                __syncthreads();
                return c;
            }
            klo = max(klo, khi - ((1u << shift) - 1u));
            __syncthreads();
        }
        return Cut{0u, 0u, 0u, 0ull, 0ull};
    };

    // 2. the cuts; without one every token that weighs anything is kept
    Cut cut = {0u, 0u, 0u, 0ull, 0ull};
    bool have = false;
    if (k > 0 || part < (1u << 24)) {
        uint32_t cnt;
        unsigned long long wt;
        histogram(bin_of, cnt, wt);
        unsigned long long total;
        if (k > 0 && cross(cnt, wt, 0, 0, true, (unsigned long long)k)) {
            have = true;
            cut = refine(true, (unsigned long long)k);
            total = cut.above_w + (unsigned long long)cut.quota * cut.key_w;
        } else {
            uint32_t in = cnt;
            total = wt;
            sample_scan(sm, in, total);
            if (tid == kSampleThreads - 1) sm.above_w = total;
            __syncthreads();
            total = sm.above_w;
            __syncthreads();
        }
        if (part < (1u << 24)) {
            // at least the first rank stays
            const unsigned long long goal = max(mul24(total, part), 1ull);
            if (cross(cnt, wt, 0, 0, false, goal)) {
                cut = refine(false, goal);
                have = true;
            }
        }
    }

    // 3. the kept weight, warp by warp over contiguous tokens
    const int seg = (p.slice + kSampleWarps - 1) / kSampleWarps;
    const int s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
    auto kept = [&](float l, bool &tie) {  // weight of a token above the cut; ties apart
        const uint32_t key = sample_key(l);
        tie = have && key == cut.key;
        if (tie || (have && key < cut.key)) return 0ull;
        const float e = prob(l);
        return e >= min_p ? weight(e) : 0ull;
    };
    unsigned long long w = 0, tie_w = 0;
    uint32_t ties = 0;
    for (int i = s0 + lane; i < s1; i += 32) {
        bool tie;
        w += kept(logit(i), tie);
        ties += tie;
    }
    if (have) {
        const uint32_t b = cut.key;
        const float l = __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
        const float e = prob(l);
        tie_w = e >= min_p ? weight(e) : 0ull;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        w += __shfl_xor_sync(0xffffffffu, w, o);
        ties += __shfl_xor_sync(0xffffffffu, ties, o);
    }
    if (lane == 0) sm.warp_w[warp] = w, sm.warp_n[warp] = ties;
    __syncthreads();
    if (tid == 0) {
        unsigned long long a = 0;
        uint32_t b = 0;
        for (int i = 0; i < kSampleWarps; ++i) a += sm.warp_w[i], b += sm.warp_n[i];
        sm.cta_w = a;
        sm.cta_n = b;
    }
    cluster.sync();
    unsigned long long before = 0, all = 0;
    uint32_t n_before = 0, n_all = 0;
    for (int c = 0; c < C; ++c) {
        const SampleShared *o = cluster.map_shared_rank(&sm, c);
        const unsigned long long cw = o->cta_w;
        const uint32_t cn = o->cta_n;
        // the cut's tokens are taken in index order
        const uint32_t take = min(cn, cut.quota - min(n_all, cut.quota));
        if (c < rank) before += cw + take * tie_w, n_before += cn;
        all += cw + take * tie_w;
        n_all += cn;
    }
    cluster.sync();  // every CTA has read the others' sums
    const unsigned long long target = mul24(all, uf);
    // 4. the token: this warp's tokens hold the target, or another's do
    for (int i = 0; i < warp; ++i) {
        const uint32_t take = min(sm.warp_n[i], cut.quota - min(n_before, cut.quota));
        before += sm.warp_w[i] + take * tie_w;
        n_before += sm.warp_n[i];
    }
    {
        const uint32_t take = min(sm.warp_n[warp], cut.quota - min(n_before, cut.quota));
        const unsigned long long after = before + sm.warp_w[warp] + take * tie_w;
        if (!(before <= target && target < after)) return;
    }
    for (int a = s0; a < s1; a += 32) {
        const int i = a + lane;
        bool tie = false;
        unsigned long long x = i < s1 ? kept(logit(i), tie) : 0ull;
        const unsigned m = __ballot_sync(0xffffffffu, tie);
        if (tie && n_before + __popc(m & ((1u << lane) - 1u)) < cut.quota) x = tie_w;
        n_before += __popc(m);
        unsigned long long run = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + run > target);
        if (hit) {
            if (lane == __ffs(hit) - 1) p.tokens[row] = i0 + i;
            return;
        }
        before += __shfl_sync(0xffffffffu, run, 31);
    }
}

}  // namespace m1
