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
// pair, found without sorting: counts and weights over bins of the distance
// to the maximum, the bin in which the cut falls, and then the same over the
// keys of that bin, 512 at a time, until one key is left (two or three rounds
// for logits of ordinary size).
//
// The top_k cut needs counts alone, so no exponential is taken for the tokens
// below it; the top_p cut looks at the tokens above the first one only.  The
// first bins see every token, the later ones a few (kept as a list).  A short
// slice adds into 512 shared bins with atomics.  A long one, where the bulk of
// the tokens would queue up on a few dozen bins, takes bins that each thread
// keeps for itself: 128 counts of 8 bits, or 16 weights.
//
// A cluster of CTAs shares a row: each keeps its slice in shared memory
// (read from HBM once) and makes its own histogram; after one cluster
// barrier every CTA adds up all of them through distributed shared memory
// and draws the same conclusions, so nothing is broadcast.  A bin's weight
// is held as two 18-bit limbs in 32-bit words (native shared-memory
// atomics), folded into 64-bit registers before a limb could overflow.
//
// Measured: one row of 50,304 f32 11 us back to back (16 to 30 us amid other
// kernels: the code is read again), 192 rows of 32,000 f32 with mixed settings
// 73 us, 48 rows of 150,001 bf16 114 us (107 to 124 amid others); 4 us and 2 us
// at HBM rate.  What
// bounds it is the passes over the slice in shared memory (the maximum, the
// first bins, one or two refinements, the tokens from the cut on), each at 10
// to 20 instructions a token, and a block or cluster barrier a round.  One
// rolled copy of each loop (70 to 100 KB of code instead of 220 to 340) came
// out slower, 88 to 109 us for the 192 rows.
#pragma once

#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"
#include "pipeline.cuh"

namespace m1 {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = kSampleThreads;  // a thread per bin
constexpr int kSampleFold = 16000;           // tokens between folds: 16000 limbs below 2^18 fit 32 bits
constexpr float kSampleSpan = 25.2f;  // exp(-24.96) * 2^36 < 1: every weight is 0 in the last of 128 bins and beyond
constexpr int kSampleMaxCluster = 8;

constexpr int kSampleWide = 16;              // a thread's own bins of a long slice
constexpr int kSampleLong = 8192;            // tokens of a slice from which it is long
constexpr int kSampleCounts = 128;           // its bins of counts
constexpr int kSampleList = 1024;            // keys a CTA keeps of a bin that is being refined
constexpr int kSampleKeep = 128;             // tokens from a cut on that a warp keeps, in index order
constexpr int kSampleOwn = 120;              // a thread's tokens between folds there: 7 bits of count above 25 of limbs

struct SampleParams {
    const void *logits;
    long long stride;  // elements between rows
    int vocab, slice;  // slice: tokens per CTA of the cluster
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

// Its inverse.
__device__ __forceinline__ float sample_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
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
    uint32_t list[kSampleList];
    float keep_l[kSampleWarps][kSampleKeep];
    int keep_i[kSampleWarps][kSampleKeep];
    uint32_t listed;
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
    // every warp adds up the totals of those before it
    uint32_t pn = lane < warp ? sm.scan_n[lane] : 0;
    unsigned long long pw = lane < warp ? sm.scan_w[lane] : 0;
#pragma unroll
    for (int o = kSampleWarps / 2; o > 0; o >>= 1) {
        pn += __shfl_xor_sync(0xffffffffu, pn, o);
        pw += __shfl_xor_sync(0xffffffffu, pw, o);
    }
    n += __shfl_sync(0xffffffffu, pn, 0);
    w += __shfl_sync(0xffffffffu, pw, 0);
}

// floor(2^36 e) of 0 <= e <= 1: the 24-bit significand shifted to its place.
__device__ __forceinline__ unsigned long long sample_weight(float e) {
    const uint32_t b = __float_as_uint(e), down = 127u - (b >> 23);
    const unsigned long long m = (unsigned long long)((b & 0x7FFFFFu) | 0x800000u) << 13;
    return down < 40u ? m >> down : 0ull;
}

template <class T>
__device__ __forceinline__ float sample_float(T v);
template <>
__device__ __forceinline__ float sample_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float sample_float<uint16_t>(uint16_t v) {
    return bf16_bits(v);
}

// T: float or bf16 bits.  kSmem: the slice is kept in shared memory.
template <class T, bool kSmem>
__global__ void __launch_bounds__(kSampleThreads) k_sample(const SampleParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ SampleShared sm;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / C;
    auto row_sync = [&]() {  // of the row's CTAs
        if (C > 1)
            cluster.sync();
        else
            __syncthreads();
    };
    auto peer = [&](int c) { return C > 1 ? cluster.map_shared_rank(&sm, c) : &sm; };
    pdl_wait();
    const int i0 = min(p.vocab, rank * p.slice), n = min(p.vocab, i0 + p.slice) - i0;
    const T *src = reinterpret_cast<const T *>(p.logits) + (long long)row * p.stride + i0;
    const bool wide = p.slice > kSampleLong;
    uint32_t *own = reinterpret_cast<uint32_t *>(dyn);  // [2][kSampleWide][threads] of a long slice
    // the copy keeps the source's offset within 16 bytes
    const int skew = (int)(reinterpret_cast<uintptr_t>(src) & 15) / (int)sizeof(T);
    T *slice = reinterpret_cast<T *>(dyn + (wide ? kSampleWide * kSampleThreads * 8 : 0)) + skew;
    const T *data = kSmem ? slice : src;
    // The slice in whole 16-byte pieces, with single elements before and after.
    // (A NaN needs no care: it is never above, at or between anything.)
    constexpr int kPer = 16 / (int)sizeof(T);
    const int head = min(n, skew ? kPer - skew : 0), pieces = (n - head) / kPer, tail = head + pieces * kPer;
    auto unpack = [&](const uint4 &w, float (&v)[kPer]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            if constexpr (sizeof(T) == 4)
                v[e] = __uint_as_float(u[e]);
            else
                v[e] = sample_float<uint16_t>((uint16_t)(u[e >> 1] >> (16 * (e & 1))));
        }
    };
    auto piece = [&](int k, float (&v)[kPer]) { unpack(*reinterpret_cast<const uint4 *>(data + head + k * kPer), v); };
    // f(logit) of this thread's share of pieces [k0, k1), two at a time, then g() of the single elements
    auto scan = [&](int k0, int k1, bool singles, auto f) {
        int k = k0 + tid;
        for (; k + kSampleThreads < k1; k += 2 * kSampleThreads) {
            float v[2][kPer];
            piece(k, v[0]);
            piece(k + kSampleThreads, v[1]);
#pragma unroll
            for (int e = 0; e < 2 * kPer; ++e) f(v[e / kPer][e % kPer]);
        }
        if (k < k1) {
            float v[kPer];
            piece(k, v);
#pragma unroll
            for (int e = 0; e < kPer; ++e) f(v[e]);
        }
        if (singles) {
            if (tid < head) f(sample_float<T>(data[tid]));
            if (tid < n - tail) f(sample_float<T>(data[tail + tid]));
        }
    };

    // 1. the largest logit and its first index
    float best = -INFINITY;
    int arg = 0x7FFFFFFF;
    {
        auto see = [&](float v, int i) {
            if (v > best || (v == best && i0 + i < arg)) best = v, arg = i0 + i;
        };
        auto one = [&](int i) {
            const T t = src[i];
            if (kSmem) slice[i] = t;
            see(sample_float<T>(t), i);
        };
#pragma unroll 4
        for (int k = tid; k < pieces; k += kSampleThreads) {
            const uint4 w = *reinterpret_cast<const uint4 *>(src + head + k * kPer);
            if (kSmem) *reinterpret_cast<uint4 *>(slice + head + k * kPer) = w;
            float v[kPer];
            unpack(w, v);
#pragma unroll
            for (int e = 0; e < kPer; ++e) see(v[e], head + k * kPer + e);
        }
        if (tid < head) one(tid);
        if (tid < n - tail) one(tail + tid);
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
    row_sync();
    float top = -INFINITY;
    arg = 0x7FFFFFFF;
#pragma unroll 1
    for (int c = 0; c < C; ++c) {
        const SampleShared *o = peer(c);
        better(o->cta_top, o->cta_arg, top, arg);
    }
    const float temp = p.temperature ? p.temperature[row] : p.temperature1;
    if (top == -INFINITY || !(temp > 0.f)) {  // nothing to choose from; greedy
        if (rank == 0 && tid == 0) p.tokens[row] = top == -INFINITY ? -1 : arg;
        row_sync();  // no CTA leaves while another reads its shared memory
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
    auto weight = [&](float e) { return sample_weight(e); };
    // the first bins: distances to the largest logit, monotone in l, the last one takes the rest
    int bins = kSampleBins;
    float bin_scale = 0.f, last_bin = 0.f;
    auto set_bins = [&](int count, float span) {  // span: a distance in logits
        bins = count;
        bin_scale = (float)count / span;
        last_bin = (float)(count - 1);
    };
    auto bin_of = [&](float l) { return l == top ? 0 : (int)fminf((top - l) * bin_scale, last_bin); };

    // A histogram round over the tokens that sel accepts (their bin, or -1), of
    // the slice or of the listed keys: afterwards thread t holds the row's
    // count and (kW) weight of bin t.
    int round = 0;
    auto gather = [&](bool weights, uint32_t &cnt, unsigned long long &wt) {
        const int b = round % 3;
        // clear the next round's buffer: it was last read two rounds ago, and
        // every CTA has passed the barrier of the last round since
        for (int q = 0; q < 3; ++q) sm.hist[(round + 1) % 3][q][tid] = 0;
        row_sync();
        cnt = 0;
        wt = 0;
#pragma unroll 1
        for (int c = 0; c < C; ++c) {
            const uint32_t(*o)[kSampleBins] = peer(c)->hist[b];
            cnt += o[0][tid];
            if (weights) wt += (unsigned long long)o[1][tid] | ((unsigned long long)o[2][tid] << 32);
        }
        ++round;
    };
    // The tokens from a cut on, in index order, 16 warps' contiguous parts: if
    // they fit, the later steps go over them instead of the slice.
    const int share = (pieces + kSampleWarps - 1) / kSampleWarps;
    const int s0 = min(pieces, warp * share), s1 = min(pieces, s0 + share);
    bool kept_few = false;
    int keep_n = 0;  // this warp's
    auto keep_from = [&](float cut_l) {
        keep_n = 0;
        auto group = [&](const float *v, int per, int at, bool valid) {
            int pos = keep_n;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const unsigned m = __ballot_sync(0xffffffffu, valid && e < per && v[e] >= cut_l);
                pos += __popc(m & ((1u << lane) - 1u));
                keep_n += __popc(m);
            }
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                if (valid && e < per && v[e] >= cut_l) {
                    if (pos < kSampleKeep) sm.keep_l[warp][pos] = v[e], sm.keep_i[warp][pos] = at + e;
                    ++pos;
                }
            }
        };
        auto single = [&](int from, int m) {
            float v[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[e] = lane < m ? sample_float<T>(data[from + lane]) : -INFINITY;
            group(v, 1, from + lane, lane < m);
        };
        if (warp == 0) single(0, head);
#pragma unroll 2
        for (int a = s0; a < s1; a += 32) {
            const int k = a + lane;
            float v[kPer];
            piece(min(k, s1 - 1), v);
            group(v, kPer, head + k * kPer, k < s1);
        }
        if (warp == kSampleWarps - 1) single(tail, n - tail);
        kept_few = __syncthreads_and(keep_n <= kSampleKeep);
    };
    // f(logit) of the kept tokens, or of all
    auto scan_kept = [&](auto f) {
        if (kept_few)
            for (int i = lane; i < keep_n; i += 32) f(sm.keep_l[warp][i]);
        else
            scan(0, pieces, true, f);
    };
    auto histogram = [&](auto kW, bool listed, auto sel, uint32_t &cnt, unsigned long long &wt) {
        uint32_t(*h)[kSampleBins] = sm.hist[round % 3];
        unsigned long long fold_w = 0;
        auto add = [&](float l) {
            const int j = sel(l);
            if (j < 0) return;
            if constexpr (kW.value) {
                const unsigned long long w = weight(prob(l));
                if (w == 0) return;
                atomicAdd(&h[1][j], (uint32_t)(w & 0x3FFFFu));
                atomicAdd(&h[2][j], (uint32_t)(w >> 18));
            }
            atomicAdd(&h[0][j], 1u);
        };
        auto fold = [&]() {
            __syncthreads();
            if constexpr (kW.value) {
                fold_w += (unsigned long long)h[1][tid] + ((unsigned long long)h[2][tid] << 18);
                h[1][tid] = h[2][tid] = 0;
                __syncthreads();
            }
        };
        if (listed) {
            for (int i = tid; i < (int)sm.listed; i += kSampleThreads) add(sample_value(sm.list[i]));
            fold();
        } else if (kept_few) {
            scan_kept(add);
            fold();
        } else {
            constexpr int kStep = kSampleFold / kPer;
            for (int a = 0; a == 0 || a < pieces; a += kStep) {
                scan(a, min(pieces, a + kStep), a == 0, add);
                fold();
            }
        }
        if constexpr (kW.value) {
            h[1][tid] = (uint32_t)fold_w;
            h[2][tid] = (uint32_t)(fold_w >> 32);
        }
        gather(kW.value, cnt, wt);
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
        unsigned long long key_w;  // weight of one token of the key
    };
    auto refine = [&](auto kW, unsigned long long goal) {
        // sm.bin, sm.above_*: the bin of the first histogram
        const int bin = sm.bin;
        const uint32_t an0 = sm.above_n;
        const unsigned long long aw0 = sm.above_w;
        uint32_t an = an0;
        unsigned long long aw = aw0;
        // keys of the bin, a little wider than its edges' rounding
        const float hi_l = fminf(top, top - (float)bin / bin_scale * (1.f - 1e-5f) + 1e-5f * fabsf(top));
        const float lo_l =
            bin == bins - 1 ? -INFINITY : top - (float)(bin + 1) / bin_scale * (1.f + 1e-5f) - 1e-5f * fabsf(top);
        uint32_t khi = sample_key(hi_l), klo = sample_key(lo_l);
        if (isinf(top)) khi = klo = sample_key(top);  // only the tokens at +inf weigh anything
        bool listed = false;
        // at most one round that misses and then four of 9 bits each
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const int bits = 32 - __clz((khi - klo) | 1u);
            const int shift = max(0, bits - 9);  // 512 bins
            const float from = sample_value(klo), to = sample_value(khi);
            uint32_t cnt;
            unsigned long long wt;
            auto sel = [&](float l) {
                // (a NaN bound, of a key past infinity, leaves it to the keys)
                if (l < from || l > to) return -1;
                const uint32_t key = sample_key(l);
                if (key > khi || key < klo || bin_of(l) != bin) return -1;
                return (int)((khi - key) >> shift);
            };
            if (!listed) {
                __syncthreads();
                if (tid == 0) sm.listed = 0;
                __syncthreads();
                scan_kept([&](float l) {
                    if (sel(l) < 0) return;
                    const uint32_t at = atomicAdd(&sm.listed, 1u);
                    if (at < kSampleList) sm.list[at] = sample_key(l);
                });
                __syncthreads();
                listed = sm.listed <= kSampleList;  // (a CTA whose list overflows goes on with its slice)
            }
            histogram(kW, listed, sel, cnt, wt);
            if (!cross(cnt, wt, an, aw, !kW.value, goal)) {
                // the estimated key range missed the cut: take all keys
                an = an0;
                aw = aw0;
                khi = 0xFFFFFFFFu;
                klo = 0u;
                listed = false;
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
                c.key_w = weight(prob(sample_value(khi)));
                const unsigned long long need = goal - (kW.value ? aw : an);
                c.quota = (uint32_t)(kW.value ? (need + c.key_w - 1) / max(c.key_w, 1ull) : need);
                __syncthreads();
                return c;
            }
            klo = max(klo, khi - ((1u << shift) - 1u));
            __syncthreads();
        }
        return Cut{0u, 0u, 0ull};
    };
    // The row's weight above a logit.
    auto above_cut = [&](float cut_l) {
        unsigned long long w = 0;
        scan_kept([&](float l) {
            if (l > cut_l) w += weight(prob(l));
        });
        uint32_t none = 0;
        sample_scan(sm, none, w);
        if (tid == kSampleThreads - 1) sm.cta_w = w;
        row_sync();
        w = 0;
#pragma unroll 1
        for (int c = 0; c < C; ++c) w += peer(c)->cta_w;
        row_sync();  // (used again below)
        return w;
    };
    // The first bins of a long slice, by threads of their own: counts.
    auto own_counts = [&](uint32_t &cnt) {
        // 8-bit counters, four bins to a word
        for (int b = 0; b < kSampleCounts / 4; ++b) own[b * kSampleThreads + tid] = 0;
        constexpr int kStep = 240 / kPer * kSampleThreads;  // pieces: at most 242 tokens a thread
        constexpr int kWords = kSampleCounts / 4 / kSampleWarps;  // a warp's words
        uint32_t c[kWords][4] = {};
        for (int a = 0; a == 0 || a < pieces; a += kStep) {
            scan(a, min(pieces, a + kStep), a == 0, [&](float l) {
                const int b = bin_of(l);
                // (nobody else's word: nothing is returned or waited for)
                atomicAdd(own + (b >> 2) * kSampleThreads + tid, 1u << (8 * (b & 3)));
            });
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                for (int t = lane; t < kSampleThreads; t += 32) {
                    const uint32_t v = own[(warp * kWords + w) * kSampleThreads + t];
                    own[(warp * kWords + w) * kSampleThreads + t] = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[w][e] += v >> (8 * e) & 0xFFu;
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) c[w][e] += __shfl_xor_sync(0xffffffffu, c[w][e], o);
                if (lane == 0) sm.hist[round % 3][0][(warp * kWords + w) * 4 + e] = c[w][e];
            }
        unsigned long long none;
        gather(false, cnt, none);
    };
    // The same for weights: two words a bin, the weight's low 18 bits, and its
    // high ones with the count above them.
    auto own_weights = [&](uint32_t &cnt, unsigned long long &wt) {
        uint32_t *lo = own, *hi = own + kSampleWide * kSampleThreads;
        for (int b = 0; b < 2 * kSampleWide; ++b) own[b * kSampleThreads + tid] = 0;
        constexpr int kStep = kSampleOwn / kPer * kSampleThreads;  // pieces
        uint32_t c = 0;
        unsigned long long w = 0;
        for (int a = 0; a == 0 || a < pieces; a += kStep) {
            scan(a, min(pieces, a + kStep), a == 0, [&](float l) {
                const unsigned long long x = weight(prob(l));
                const int at = bin_of(l) * kSampleThreads + tid;
                if (x) {
                    atomicAdd(lo + at, (uint32_t)(x & 0x3FFFFu));
                    atomicAdd(hi + at, (uint32_t)(x >> 18) + (1u << 25));
                }
            });
            __syncthreads();
            static_assert(kSampleWide == kSampleWarps, "a warp per bin");
            for (int t = warp * kSampleThreads + lane; t < (warp + 1) * kSampleThreads; t += 32) {
                const uint32_t h = hi[t];
                c += h >> 25;
                w += ((unsigned long long)(h & 0x1FFFFFFu) << 18) + lo[t];
                hi[t] = lo[t] = 0;
            }
            __syncthreads();
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            c += __shfl_xor_sync(0xffffffffu, c, o);
            w += __shfl_xor_sync(0xffffffffu, w, o);
        }
        if (lane == 0) {
            uint32_t(*h)[kSampleBins] = sm.hist[round % 3];
            h[0][warp] = c;
            h[1][warp] = (uint32_t)w;
            h[2][warp] = (uint32_t)(w >> 32);
        }
        gather(true, cnt, wt);
    };

    // 2. the cuts; without one every token that weighs anything is kept
    const std::false_type counts;
    const std::true_type weights;
    const float span = kSampleSpan * temp;  // beyond it every weight is 0
    Cut cut = {0u, 0u, 0ull};
    bool have = false;
    uint32_t cnt = 0;
    unsigned long long wt = 0;
    if (k > 0) {
        set_bins(wide ? kSampleCounts : kSampleBins, span);
        if (wide)
            own_counts(cnt);
        else
            histogram(counts, false, bin_of, cnt, wt);
        // a cut in the last bin, where nothing weighs, changes nothing
        if (tid == bins - 1) cnt = 0;
        if (cross(cnt, 0, 0, 0, true, (unsigned long long)k)) {
            cut = refine(counts, (unsigned long long)k);
            have = true;
            keep_from(sample_value(cut.key));
        }
    }
    if (part < (1u << 24)) {
        const float cut_l = sample_value(cut.key);
        const bool few = have && k <= kSampleLong;  // tokens above the first cut
        if (few) {
            set_bins(kSampleBins, fminf(fmaxf(top - cut_l, 1e-30f), span));
            histogram(weights, false, [&](float l) { return l > cut_l ? bin_of(l) : -1; }, cnt, wt);
        } else if (wide) {
            // (tokens below a first cut join in: the second one's goal lies above them)
            set_bins(kSampleWide, span);
            own_weights(cnt, wt);
        } else {
            set_bins(kSampleBins, span);
            histogram(weights, false, bin_of, cnt, wt);
        }
        unsigned long long total = wt;
        {
            uint32_t in = cnt;
            sample_scan(sm, in, total);
            if (tid == kSampleThreads - 1) sm.above_w = total;
            __syncthreads();
            total = sm.above_w;
            __syncthreads();
        }
        if (have && !few) total = above_cut(cut_l);
        if (have) total += (unsigned long long)cut.quota * cut.key_w;
        // at least the first rank stays
        const unsigned long long goal = max(mul24(total, part), 1ull);
        if (cross(cnt, wt, 0, 0, false, goal)) {
            cut = refine(weights, goal);
            if (!have) keep_from(sample_value(cut.key));
            have = true;
        } else if (have) {  // among the first cut's own tokens
            const unsigned long long need = goal - (total - (unsigned long long)cut.quota * cut.key_w);
            cut.quota = (uint32_t)((need + cut.key_w - 1) / max(cut.key_w, 1ull));
        }
    }

    // 3. the kept weight, warp by warp over contiguous pieces (the elements
    //    before them are the first warp's, those after them the last one's)
    const float cut_l = sample_value(cut.key);
    auto kept = [&](float l, bool &tie) {  // weight of a token above the cut; ties apart
        tie = have && l == cut_l;
        if (have && !(l > cut_l)) return 0ull;
        const float e = prob(l);
        return e >= min_p ? weight(e) : 0ull;
    };
    unsigned long long w = 0, tie_w = 0;
    uint32_t ties = 0;
    auto count = [&](float l) {
        bool tie;
        w += kept(l, tie);
        ties += tie;
    };
    if (kept_few) {
        for (int i = lane; i < keep_n; i += 32) count(sm.keep_l[warp][i]);
    } else {
#pragma unroll 2
        for (int k = s0 + lane; k < s1; k += 32) {
            float v[kPer];
            piece(k, v);
#pragma unroll
            for (int e = 0; e < kPer; ++e) count(v[e]);
        }
        if (warp == 0 && lane < head) count(sample_float<T>(data[lane]));
        if (warp == kSampleWarps - 1 && lane < n - tail) count(sample_float<T>(data[tail + lane]));
    }
    if (have) {
        const float e = prob(cut_l);
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
    row_sync();
    unsigned long long before = 0, all = 0;
    uint32_t n_before = 0, n_all = 0;
#pragma unroll 1
    for (int c = 0; c < C; ++c) {
        const SampleShared *o = peer(c);
        const unsigned long long cw = o->cta_w;
        const uint32_t cn = o->cta_n;
        // the cut's tokens are taken in index order
        const uint32_t take = min(cn, cut.quota - min(n_all, cut.quota));
        if (c < rank) before += cw + take * tie_w, n_before += cn;
        all += cw + take * tie_w;
        n_all += cn;
    }
    row_sync();  // every CTA has read the others' sums
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
    // kPer (or 1) consecutive elements a lane, from index `at`; true once the token is found
    auto search = [&](const float *v, int per, int at, bool valid) {
        unsigned long long x[kPer], run = 0;
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            bool tie = false;
            x[e] = valid && e < per ? kept(v[e], tie) : 0ull;
            if (tie) x[e] = ~0ull, ++mine;
        }
        uint32_t t = mine;  // ties of the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += y;
        }
        uint32_t nth = n_before + t - mine;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            if (x[e] == ~0ull) x[e] = nth++ < cut.quota ? tie_w : 0ull;
            run += x[e];
        }
        const unsigned long long lane_w = run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + run > target);
        if (hit && lane == __ffs(hit) - 1) {
            unsigned long long r = before + run - lane_w;
            int i = 0;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                r += x[e];
                if (r <= target) i = e + 1;
            }
            p.tokens[row] = i0 + at + i;
        }
        before += __shfl_sync(0xffffffffu, run, 31);
        n_before += __shfl_sync(0xffffffffu, t, 31);
        return hit != 0;
    };
    auto search1 = [&](float l, int at, bool valid) {
        float v[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[e] = l;
        return search(v, 1, at, valid);
    };
    if (kept_few) {
        for (int a = 0; a < keep_n; a += 32) {
            const int i = min(a + lane, keep_n - 1);
            if (search1(sm.keep_l[warp][i], sm.keep_i[warp][i], a + lane < keep_n)) return;
        }
        return;
    }
    auto single = [&](int from, int m) {
        return search1(lane < m ? sample_float<T>(data[from + lane]) : -INFINITY, from + lane, lane < m);
    };
    if (warp == 0 && single(0, head)) return;
    for (int a = s0; a < s1; a += 32) {
        const int k = a + lane;
        float v[kPer];
        piece(min(k, s1 - 1), v);
        if (search(v, kPer, head + k * kPer, k < s1)) return;
    }
    if (warp == kSampleWarps - 1) single(tail, n - tail);
}

}  // namespace m1
