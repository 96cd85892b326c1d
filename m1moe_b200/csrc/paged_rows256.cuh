// paged_rows256.cuh — attention of up to 256 rows (new tokens x heads of one
// KV head) per item over a paged cache, on the tensor cores: prompts, prompt
// chunks, mixed batches, and a batch's rows against its shared prefix
// (sm_100a).
//
// The formula of paged_rows16.cuh.  Here the two products and the exponentials
// bound it: a 128 x 128 tile of scores at hd 128 is 2 x 2.1 M multiply-adds
// (512 cycles each of a tcgen05 pipe) and 16,384 exponentials (1,024 cycles
// of an SM's 16 special-function lanes a cycle).
//
// One persistent CTA per SM walks its run of 128-position units (paged.cuh).
// An item's 256 rows are two M-tiles of 128 that share every K and V tile:
//   warps 0-3, 4-7   softmax of M-tile 0 and 1, a thread per row: scores from
//                    tensor memory, running maximum and sum, weights back to
//                    tensor memory as bf16, over the scores they came from
//   warps 8-11       K and V tiles from the pages into a ring of shared memory
//   warps 12-15      warp 12 issues the products: S = Q K^T (both operands in shared
//                    memory), O += P V (P from tensor memory, V as it lies:
//                    MN-major)
// While one M-tile's warps take exponentials, the tensor cores run the other
// one's products.  Tensor memory: S0, S1, O0, O1, 128 columns each.
//
// A tile whose 128 positions all belong to the item comes by TMA, one box per
// page (or 128 rows of one) and 64 columns.  A tile at an item's edge is
// copied with cp.async, 16 bytes a lane, with zeros in the rows outside: what
// lies in a page's unused rows may be anything, and 0 * NaN is NaN.  The
// writing thread's fence.proxy.async makes those copies visible to the tensor
// cores.
//
// A row's accumulator keeps the reference maximum it was started with until
// the true maximum is more than 2^8 above it in the weights' scale; only then
// is it rescaled.  Weights are at most 2^8 (bf16 has the same relative error
// there), sums are fp32.
//
// Measured: 8192 tokens of 32/8 heads at hd 128, 518 us back to back = 1061
// TFLOP/s over the visible pairs, 65 % of the measured GEMM rate (585 us = 940
// in turn with other kernels); 4096 tokens 161 us; about 4,000 cycles a unit
// against 2,048 of products.  The chain of one M-tile (scores out 170,
// maximum 260, exponentials 1,400, weights in 120, the two products 1,130 and
// their hand-offs) is what bounds it: with every column of tensor memory
// taken, the next scores cannot be computed beside it.  Tried and slower: two
// threads a row (747 us against 647 then: the exponentials of a tile take as
// long), a polynomial for a quarter to a half of the exponentials (515 to
// 551), five ring stages without the output staging (588 against 558), the
// products' loops rolled (672).
#pragma once

#include <type_traits>

#include "paged_rows16.cuh"
#include "umma.cuh"

namespace m1 {

constexpr int kTileRows = 128;              // an M-tile
constexpr int kRows256Threads = 16 * 32;
constexpr int kRows256Loaders = 128;
constexpr float kRescaleLog2 = 8.f;
constexpr uint32_t kDrainLimit = 1u << 16;  // polls, for copies that take microseconds
// Registers a thread: the block is launched with 128 each (65,536 / 512); the
// loader and product warpgroups give theirs up to the two softmax ones, which
// hold a row of 128 scores: 2 * 200 + 2 * 56 = 4 * 128.
constexpr int kRegsSoftmax = 200, kRegsOther = 56;
static_assert(2 * kRegsSoftmax + 2 * kRegsOther <= 4 * 128, "the split must fit the launch's registers");

template <int HD>
struct Rows256 {
    static constexpr int kHalves = HD / 64;                    // 128-byte columns of a tile
    static constexpr int kTile = 128 * HD * 2;                 // bytes of a Q M-tile, K tile or V tile
    static constexpr int kStages = 4;  // the products' turns are written out for four
    static constexpr int kPairs = kStages / 2;  // V of a tile and K of the next are given back together
    static constexpr int kStageOut = 8 * 1024;                  // 32 rows of 32 bytes a softmax warp, for the output
    static constexpr int kSmem = (2 + kStages) * kTile + kStageOut + 1024;
};

struct Rows256Params {
    RowsParams r;
    int prefix_run;      // this launch is the shared prefix: all rows see [0, prefix)
    float *partial;      // there: [total_q][nh][hd] weighted values and
    float2 *partial_ml;  // [total_q][nh] maxima and sums
};

// Shared-memory descriptors, 128-byte swizzle, as two words: the high one
// (stride byte offset 1024 between 8-row groups, version 1, layout type 2) is
// the same for all operands here, the low one names the start address and
// the leading byte offset (bits 16-29).  K-major operands do not use that
// offset.  An MN-major one (V as it lies: rows along K, 64 elements of N per
// 128-byte row) has its 64-element column blocks `lead` bytes apart.
constexpr uint32_t kUmmaDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t umma_desc_lo(uint32_t smem, uint32_t lead) {
    return ((smem >> 4) & 0x3FFFu) | ((lead >> 4) << 16);
}

// True in one lane of the warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r != 0;
}

// 2-D tiled load of the map's box at element coordinates (x, y); completes the
// box's bytes on `bar`.
__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}

// Instruction descriptor of kind::f16 with bf16 operands and fp32
// accumulators; b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t umma_idesc_bf16(int M, int N, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

// D[tmem] (+)= A[smem] . B[smem]^T, operands by their descriptors' low words.
__device__ __forceinline__ void umma_bf16_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                             bool accumulate) {
    asm volatile(
        "{ .reg .pred p; .reg .b64 da, db; setp.ne.b32 p, %4, 0; mov.b64 da, {%1, %5}; mov.b64 db, {%2, %5}; "
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p; }" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "r"(kUmmaDescHi)
        : "memory");
}

// D[tmem] (+)= A[tmem] . B[smem]: A holds two bf16 of K per 32-bit column.
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc,
                                             bool accumulate) {
    asm volatile(
        "{ .reg .pred p; .reg .b64 db; setp.ne.b32 p, %4, 0; mov.b64 db, {%2, %5}; "
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p; }" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "r"(kUmmaDescHi)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

template <int N>
__device__ __forceinline__ void regs_more() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_less() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// The same, NaN if an operand is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 32 raw scores capped, in units of log2: by the polynomial, two at a time,
// while |x| <= 1 throughout the warp, and score by score where not.  Up to a
// cap of kFarCap the second form serves there for the small scores too: its
// error, 1e-7 of the cap, is at most 4e-5 of a score's units, beside a weight's
// rounding of 2^-9 (4096 tokens of 32/8 heads with scores mostly above the cap:
// 328 us so, 374 with both forms of each).
constexpr float kFarCap = 256.f;
__device__ __forceinline__ void cap_scores(uint32_t (&v)[32], float scale_log2, float cap, float cs) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 32; ++e) top = fmaxf(top, fabsf(__uint_as_float(v[e])));
    if (__all_sync(0xffffffffu, top * cs <= 1.f)) {
        const uint64_t c2 = pack2(cs, cs), s2 = pack2(scale_log2, scale_log2);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            const uint64_t d = pack2(__uint_as_float(v[e]), __uint_as_float(v[e + 1]));
            const uint64_t x = mul2(d, c2), y = mul2(x, x);
            uint64_t t = fma2(pack2(kTanh5, kTanh5), y, pack2(kTanh4, kTanh4));
            t = fma2(t, y, pack2(kTanh3, kTanh3));
            t = fma2(t, y, pack2(kTanh2, kTanh2));
            t = fma2(t, y, pack2(kTanh1, kTanh1));
            t = fma2(t, y, pack2(kTanh0, kTanh0));
            float a, b;
            unpack2(mul2(mul2(d, s2), t), a, b);
            v[e] = __float_as_uint(a);
            v[e + 1] = __float_as_uint(b);
        }
    } else if (cap <= kFarCap) {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(cap_far(__uint_as_float(v[e]) * cs, cap));
    } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(cap_score(__uint_as_float(v[e]), scale_log2, cap, cs));
    }
}

// The weights of a row's 128 scores, over the scores in tensor memory as bf16;
// returns their fp32 sum.  All scores are scaled first, then taken eight pairs
// at a time, a batch's exponentials ahead of the last batch's sums and
// conversions, so that the special-function unit always has work queued.
__device__ __forceinline__ float row_weights(uint32_t (&v)[4][32], float mult, float ref, uint32_t ts) {
    const uint64_t mult2 = pack2(mult, mult), ref2 = pack2(-ref, -ref);
    uint64_t sum[4] = {0, 0, 0, 0};
    auto f = [&](int e) { return __uint_as_float(v[e >> 5][e & 31]); };
#pragma unroll
    for (int e = 0; e < 128; e += 2) {
        float x0, x1;
        unpack2(fma2(pack2(f(e), f(e + 1)), mult2, ref2), x0, x1);
        v[e >> 5][e & 31] = __float_as_uint(x0);
        v[e >> 5][(e & 31) + 1] = __float_as_uint(x1);
    }
    uint32_t w[16];
#pragma unroll
    for (int b = 0; b <= 8; ++b) {
        if (b < 8) {
#pragma unroll
            for (int e = 16 * b; e < 16 * b + 16; ++e) v[e >> 5][e & 31] = __float_as_uint(exp2_approx(f(e)));
        }
        if (b > 0) {
            const int e0 = 16 * (b - 1);
#pragma unroll
            for (int e = e0; e < e0 + 16; e += 2) {
                sum[(e >> 1) & 3] = add2(sum[(e >> 1) & 3], pack2(f(e), f(e + 1)));
                w[(e & 31) >> 1] = pack_bf16(f(e), f(e + 1));
            }
            if ((b & 1) == 0) tmem_st16(ts + 8 * (b - 2), w);
        }
    }
    float a, b;
    unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), a, b);
    return a + b;
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait; once one has given up (the CTA's abort flag), all return false
// at once and the roles go through the rest of their motions without touching
// tensor memory or issuing copies, so that every barrier still matches.
__device__ __forceinline__ bool paged_wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *status) {
#pragma unroll 1
    for (uint32_t i = 0; i < kWaitLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort) return false;
    }
    *abort = 1;
    atomicOr(status, kPagedErrWait);
    return false;
}

// One segment of a CTA's run: tiles [ja, jb) of an item, for the rows of one
// or two M-tiles.
struct Rows256Segment {
    int g, item, u0, u1, seg0, seg1;       // its units, the item's units
    int seq, row0, nrows, q0, len, first;  // first: position of the sequence's first new token
    int ja, jb, lo;                        // lo: first position any row sees
};

// The roles walk the same segments, each on its own.
struct Rows256Walk {
    int u, end, g, item, units, items;
    __device__ __forceinline__ void start(const PagedShape &s, const PagedPlanView &p, int cta) {
        units = p.header[kPhUnits];
        items = p.header[kPhItems];
        const int per = p.header[kPhPer], all = units * s.nkv;
        u = min(cta * per, all);
        end = min(all, u + per);
        g = u < end ? u / units : 0;
        item = u < end ? p.start[cta] : 0;
    }
    __device__ __forceinline__ bool next(const PagedShape &s, const PagedPlanView &p, const Rows256Params &a,
                                         Rows256Segment &x) {
        PagedItem it;
        for (;;) {
            if (u >= end) return false;
            it = p.items[item];
            x.g = g;
            x.item = item;
            // (the item's first kPagedItemCost units stand for its overhead; a run
            // that ends in them leaves the item to the next CTA)
            x.seg0 = g * units + p.unit_at[item] + kPagedItemCost;
            x.seg1 = g * units + p.unit_at[item + 1];
            x.u0 = max(u, x.seg0);
            x.u1 = min(end, x.seg1);
            u = x.u1;
            if (u == x.seg1 && ++item == items) item = 0, ++g;
            if (x.u0 < x.u1) break;
        }
        x.seq = it.seq;
        x.row0 = it.row0;
        x.nrows = it.nrows;
        x.ja = it.unit0 + x.u0 - x.seg0;
        x.jb = it.unit0 + x.u1 - x.seg0;
        if (a.prefix_run) {
            x.q0 = 0;
            x.len = p.header[kPhPrefix];
            x.first = 0;
            x.lo = 0;
        } else {
            x.q0 = it.q0;
            x.len = it.len;
            x.first = it.len - it.nq;
            x.lo = first_seen(x.first + fdiv(it.row0, s.by_group), s.window);
        }
        // the next item's record, for the next call
        asm volatile("prefetch.global.L1 [%0];" ::"l"(p.items + item));
        asm volatile("prefetch.global.L1 [%0];" ::"l"(p.unit_at + item + 1));
        return true;
    }
};

template <int HD>
__global__ void __launch_bounds__(kRows256Threads, 1) k_paged_rows256(const PagedShape s, const PagedPlanView p,
                                                                      const Rows256Params a,
                                                                      const __grid_constant__ CUtensorMap kmap,
                                                                      const __grid_constant__ CUtensorMap vmap) {
    using T = Rows256<HD>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t kv_full[T::kStages], kv_empty[T::kPairs], q_full[2], q_empty[2], s_full[2], p_full[2], o_done[2], drain;
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sq = smem, *skv = smem + 2 * T::kTile;
    uint8_t *sout = skv + T::kStages * T::kTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *status = p.status;
    if (threadIdx.x == 0) {
        for (int i = 0; i < T::kStages; ++i) {
            mbar_init(&kv_full[i], kRows256Loaders);
            if (i < T::kPairs) mbar_init(&kv_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], kRows256Loaders);
            mbar_init(&q_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], kTileRows);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(&drain, 1);
        mbar_fence_init();
        abort_flag = 0;
    }
    if (warp == 12) {
        tmem_alloc(&tmem_base, 512);
        tmem_relinquish();
        tc_fence_before_sync();
    }
    __syncthreads();
    tc_fence_after_sync();
    // All 512 columns are this block's, so they start at address 0, which lets
    // the products' operands be constants.
    constexpr uint32_t tmem = 0;
    if (threadIdx.x == 0 && tmem_base != 0) {
        abort_flag = 1;
        atomicOr(p.status, kPagedErrWait);
    }
    pdl_wait();
    Rows256Walk walk;
    walk.start(s, p, blockIdx.x);
    Rows256Segment x;

    if (warp >= 8 && warp < 12) {
        // ------------------------------------------------------ K and V tiles
        regs_less<kRegsOther>();
        const int t = threadIdx.x - 256;
        constexpr int kChunks = HD / 8;                    // 16-byte chunks per row
        constexpr int kRowsAtOnce = kRows256Loaders / kChunks;
        const int c = t % kChunks, r0 = t / kChunks;
        const uint32_t kv_addr = smem_addr(skv);
        const int box_shift = min(s.page_shift, 7), boxes = 128 >> box_shift;  // rows of a box, boxes along a tile
        int tile = 0, issued = 0;  // K and V tiles so far, K first; and those whose copies were issued
        bool ok = true;
        auto claim = [&]() {  // the next tile's stage, free
            const int st = tile % T::kStages;
            // its last tile, tile - kStages, went with pair (tile - kStages + 1) / 2
            const int pair = (tile - T::kStages + 1) / 2;
            if (ok && tile >= T::kStages)
                ok = paged_wait(&kv_empty[pair % T::kPairs], (pair / T::kPairs) & 1, &abort_flag, status);
            ok = __all_sync(0xffffffffu, ok);
            ++tile;
            if (ok) issued = tile;
            return st;
        };
        int nq0 = 0, nq1 = 0;  // times each M-tile's Q was loaded
        auto nq_of = [&](int i) { return i ? nq1 : nq0; };
        while (walk.next(s, p, a, x)) {
            // the rows of Q, HD / 8 lanes a row, zeros past the item's rows,
            // as soon as the last segment's scores are done with the buffers
            const int tiles = x.nrows > kTileRows ? 2 : 1;
            for (int i = 0; i < tiles; ++i) {
                if (ok && nq_of(i) > 0) ok = paged_wait(&q_empty[i], (nq_of(i) - 1) & 1, &abort_flag, status);
                ok = __all_sync(0xffffffffu, ok);
                const uint32_t base = smem_addr(sq) + i * T::kTile + (c >> 3) * 16384;
#pragma unroll 4
                for (int k = 0; k < 128 / kRowsAtOnce; ++k) {
                    const int r = r0 + k * kRowsAtOnce, pr = x.row0 + i * kTileRows + r;
                    const bool in = i * kTileRows + r < x.nrows;
                    const int pt = fdiv(pr, s.by_group);
                    const long long src = in ? (long long)(x.q0 + pt) * a.r.q_stride +
                                                   (long long)(x.g * s.group + pr - pt * s.group) * HD + c * 8
                                             : 0;
                    if (ok) cp_async16(base + sw128_offset(r, c & 7), a.r.q + src, in);
                }
            }
            cp_async_commit();
            ++nq0;
            nq1 += tiles == 2;
            bool q_sent = false;
            auto send_q = [&]() {  // after a wait that covers the copies of Q
                fence_proxy_async_smem();
                for (int i = 0; i < tiles; ++i) mbar_arrive(&q_full[i]);
                q_sent = true;
            };
            for (int j = x.ja; j < x.jb; ++j) {
                const int pos0 = j * kPagedUnitLarge;
                // every warp looks up all of the tile's pages: lane b that of box b
                int mine = -1;
                bool inside = pos0 >= x.lo && pos0 + kPagedUnitLarge <= x.len;
                if (inside && lane < boxes)
                    mine = paged_row(s, a.r.table, x.seq, x.g, pos0 + (lane << box_shift), status);
                inside = inside && __all_sync(0xffffffffu, lane >= boxes || mine >= 0);
                if (inside) {
                    // op o = (box, 64-column half) is lane o / 4 of warp o % 4's
                    const int o = lane * 4 + (warp - 8);
                    const bool mine_op = o < boxes * T::kHalves;
                    const int box = mine_op ? o / T::kHalves : 0, half = o % T::kHalves;
                    const int row = __shfl_sync(0xffffffffu, mine, box);
                    for (int kv = 0; kv < 2; ++kv) {
                        const int st = claim();
                        if (ok) {
                            if (t == 0)
                                mbar_arrive_expect_tx(&kv_full[st], T::kTile);
                            else
                                mbar_arrive(&kv_full[st]);
                            if (mine_op)
                                tma_load_2d(skv + st * T::kTile + half * 16384 + (box << box_shift) * 128,
                                            kv ? &vmap : &kmap, half * 64, row, &kv_full[st]);
                        }
                    }
                    if (!q_sent) {
                        cp_async_wait(0);
                        send_q();
                    }
                } else {
                    int mine8 = -1;  // the page of positions 8 lane .. 8 lane + 7
                    if (lane < 16 && pos0 + 8 * lane < x.len && pos0 + 8 * lane + 7 >= x.lo)
                        mine8 = paged_row(s, a.r.table, x.seq, x.g, pos0 + 8 * lane, status);
                    int st[2];
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        st[kv] = claim();
                        const uint16_t *pool = kv ? a.r.v : a.r.k;
                        const uint32_t base = kv_addr + st[kv] * T::kTile + (c >> 3) * 16384;
#pragma unroll 4
                        for (int i = 0; i < 128 / kRowsAtOnce; ++i) {
                            const int r = r0 + i * kRowsAtOnce;
                            const int row = __shfl_sync(0xffffffffu, mine8, r >> 3);
                            const bool in = row >= 0 && pos0 + r < x.len && pos0 + r >= x.lo;
                            const long long src = in ? ((long long)row + (r & 7)) * HD + c * 8 : 0;
                            if (ok) cp_async16(base + sw128_offset(r, c & 7), pool + src, in);
                        }
                        cp_async_commit();
                    }
                    cp_async_wait(1);
                    if (!q_sent) send_q();
                    fence_proxy_async_smem();
                    mbar_arrive(&kv_full[st[0]]);
                    cp_async_wait(0);
                    fence_proxy_async_smem();
                    mbar_arrive(&kv_full[st[1]]);
                }
            }
        }
        // The last copies land before the CTA leaves: where a wait gave up, here
        // or in another warp, no product may be waiting for them.
        cp_async_wait(0);
        for (int m = max(0, issued - T::kStages); m < issued; ++m)
            for (uint32_t i = 0; i < kDrainLimit && !mbar_try_wait(&kv_full[m % T::kStages], (m / T::kStages) & 1); ++i) {
            }
    } else if (warp >= 12) {
        // ---------------------------------------------------------- products
        // The whole warp follows the schedule; one elected lane issues.
        regs_less<kRegsOther>();
        if (warp == 12) {
            constexpr uint32_t kIdQK = umma_idesc_bf16(128, 128, false), kIdPV = umma_idesc_bf16(128, HD, true);
            const bool elected = elect_one();
            const uint32_t q_lo = umma_desc_lo(smem_addr(sq), 16), k_lo = umma_desc_lo(smem_addr(skv), 16);
            const uint32_t v_lo = umma_desc_lo(smem_addr(skv), 16384);
            uint32_t phase = 0;  // bits 0, 1: next parity of q_full; 2, 3: of p_full
            bool ok = true;
            // (only the elected lane's `ok` counts; the others keep it company)
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                if (ok) ok = paged_wait(bar, parity & 1, &abort_flag, status);
            };
            // Tile after tile, across segments: S of the next tile (the next
            // segment's first one, while this one's rows are still being
            // finished) goes behind each P V.  The first turn has no P V.
            bool more = walk.next(s, p, a, x);
            int tiles = 1, both = 0, j = 0, tile = -2;
            bool begun = false;
            // One turn: O_i += P_i V of a tile, S_i = Q_i K^T of the next.  kPar: the
            // turn's parity, which fixes the stages (tile is 4 n - 2 + 2 kPar), so
            // that operands are constants: what the issuing warp computes between
            // two products is what the tensor cores wait for.
            auto turn_of = [&](auto kPar, auto kMiddle) {
                constexpr int vs = (2 * kPar.value + 3) % 4, ks = 2 * kPar.value % 4;
                static_assert(T::kStages == 4, "two tiles a turn, two parities");
                // (most turns are amid an item's tiles, with both M-tiles at work)
                constexpr bool mid = kMiddle.value;
                const bool ends = !mid && j + 1 == tiles, follows = mid || !ends || more;
                const int next_tiles = x.jb - x.ja, next_both = more && x.nrows > kTileRows;
                const bool gives_q = !mid && (ends ? next_tiles == 1 : j + 2 == tiles);
                const bool works = mid || begun, two = mid || both;
                // both tiles first: nothing then stands between the weights and the products
                if (works) wait(&kv_full[vs], (tile + 1) / 4);
                if (follows) wait(&kv_full[ks], (tile + 2) / 4);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (works && (i == 0 || two)) {
                        wait(&p_full[i], phase >> (2 + i));
                        tc_fence_after_sync();
                        phase ^= 4u << i;
                        if (ok && elected) {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                umma_bf16_ts(256 + i * 128, i * 128 + 8 * k, v_lo + ((vs * T::kTile + k * 2048) >> 4),
                                             kIdPV, !(j == 0 && k == 0));
                            // (before that, the next scores' commit tells that O is up to date)
                            if (ends) umma_commit(&o_done[i]);
                        }
                    }
                    if (follows && (i == 0 || (ends ? next_both : two))) {
                        if (ends) {
                            wait(&q_full[i], phase >> i);
                            phase ^= 1u << i;
                        }
                        if (ok && elected) {
#pragma unroll
                            for (int k = 0; k < HD / 16; ++k) {
                                const uint32_t step = (k >> 2) * 16384 + (k & 3) * 32;
                                umma_bf16_ss(i * 128, q_lo + ((i * T::kTile + step) >> 4),
                                             k_lo + ((ks * T::kTile + step) >> 4), kIdQK, k > 0);
                            }
                            umma_commit(&s_full[i]);
                            // the segment's last scores: the next one's rows may come
                            if (gives_q) umma_commit(&q_empty[i]);
                        }
                    }
                }
                // V of this turn and K of the next are done with together
                if (ok && elected) umma_commit(&kv_empty[kPar.value]);
                tile += 2;
                if (!ends) {
                    ++j;
                } else {
                    tiles = next_tiles;
                    both = next_both;
                    j = 0;
                    begun = true;
                    if (!more) return false;
                    more = walk.next(s, p, a, x);
                }
                return true;
            };
            auto turn = [&](auto kPar) {
                if (begun && both && j + 2 < tiles) return turn_of(kPar, std::true_type{});
                return turn_of(kPar, std::false_type{});
            };
            if (more) {
                const std::integral_constant<int, 0> even;
                const std::integral_constant<int, 1> odd;
                while (turn(even) && turn(odd)) {
                }
            }
            // every product has ended before tensor memory is given back
            if (elected) umma_commit(&drain);
            __syncwarp();
            for (uint32_t i = 0; i < kWaitLimit && !mbar_try_wait(&drain, 0); ++i) {
            }
        }
    } else {
        // ----------------------------------------------------------- softmax
        regs_more<kRegsSoftmax>();
        const int i = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + i * 128 + lanes, to = tmem + 256 + i * 128 + lanes;
        const bool capped = a.r.cap > 0.f;
        const float mult = capped ? 1.f : a.r.scale * kLog2e;
        uint8_t *stage = sout + warp * 1024;
        int ns = 0, nseg = 0;  // score tiles, segments so far
        bool ok = true;
        while (walk.next(s, p, a, x)) {
            const int n = min(kTileRows, x.nrows - i * kTileRows);  // rows of this M-tile
            if (n <= 0) continue;
            const int r = x.row0 + i * kTileRows + row, tok = fdiv(r, s.by_group);  // packed row and its token
            const int head = x.g * s.group + r - tok * s.group;
            const bool live = row < n;
            const int hi = a.prefix_run ? x.len - 1 : x.first + tok;
            const int lo = a.prefix_run ? 0 : first_seen(hi, s.window);
            // limits that hold for the M-tile's every row
            const int rf = x.row0 + i * kTileRows;
            const int min_hi = a.prefix_run ? x.len - 1 : x.first + fdiv(rf, s.by_group);
            const int max_lo = a.prefix_run ? 0 : first_seen(x.first + fdiv(rf + n - 1, s.by_group), s.window);
            const int warp_hi = __shfl_sync(0xffffffffu, hi, 0), warp_lo = __shfl_sync(0xffffffffu, lo, 31);
            float m = -INFINITY, l = 0.f;  // the reference maximum (raw scale) and the sum
            for (int j = x.ja; j < x.jb; ++j) {
                if (ok) ok = paged_wait(&s_full[i], ns & 1, &abort_flag, status);
                ok = __all_sync(0xffffffffu, ok);
                if (ok) {
                    tc_fence_after_sync();
                    const int pos0 = j * kPagedUnitLarge;
                    const bool masked = pos0 < max_lo || pos0 + kPagedUnitLarge - 1 > min_hi;
                    if (capped || masked) {
                        // 32 scores at a time through tensor memory (rolled: the unrolled
                        // code would not fit the instruction cache)
#pragma unroll 1
                        for (int q = 0; q < 4; ++q) {
                            const int at = pos0 + 32 * q;
                            // some row of this warp does not see all of the 32 positions
                            const bool hides = at + 31 > warp_hi || at < warp_lo;
                            if (!capped && !hides) continue;
                            uint32_t y[32];
                            tmem_ld32(ts + 32 * q, y);
                            tmem_wait_ld();
                            if (capped) cap_scores(y, a.r.scale * kLog2e, a.r.cap, a.r.scale / a.r.cap);
                            if (hides) {
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (at + e > hi || at + e < lo) y[e] = 0xFF800000u;  // -inf
                            }
                            tmem_st32(ts + 32 * q, y);
                        }
                        tmem_wait_st();
                    }
                    uint32_t v[4][32];  // the row's 128 scores
#pragma unroll
                    for (int q = 0; q < 4; ++q) tmem_ld32(ts + 32 * q, v[q]);
                    tmem_wait_ld();
                    float mx4[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        mx4[q] = fmaxf(__uint_as_float(v[q][0]), __uint_as_float(v[q][1]));
#pragma unroll
                        for (int e = 2; e < 32; e += 2)
                            mx4[q] = max3(mx4[q], __uint_as_float(v[q][e]), __uint_as_float(v[q][e + 1]));
                    }
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                    bool grow = false;
                    float f = 1.f;
                    if (m == -INFINITY) {
                        m = mx;
                    } else if ((mx - m) * mult > kRescaleLog2) {
                        grow = true;
                        f = exp2_approx((m - mx) * mult);
                        m = mx;
                        l *= f;
                    }
                    // j > a: the products of the tiles before are in O
                    if (__any_sync(0xffffffffu, grow) && j > x.ja) {
                        {  // (these scores' products came after those of P V)
#pragma unroll 1
                            for (int q = 0; q < HD / 16; ++q) {
                                uint32_t y[16];
                                tmem_ld16(to + 16 * q, y);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * f);
                                tmem_st16(to + 16 * q, y);
                            }
                            tmem_wait_st();
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : m * mult;
                    l += row_weights(v, mult, ref, ts);
                    tmem_wait_st();
                    tc_fence_before_sync();
                }
                mbar_arrive(&p_full[i]);
                ++ns;
            }
            // ------------------------------------------------ the segment's end
            if (ok) ok = paged_wait(&o_done[i], nseg++ & 1, &abort_flag, status);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) tc_fence_after_sync();
            const bool whole = x.u0 == x.seg0 && x.u1 == x.seg1;
            const long long token = x.q0 + tok;
            const bool narrow = !a.prefix_run && a.r.out_bf16;  // bf16 rows; else f32
            uint8_t *out_row = a.prefix_run ? reinterpret_cast<uint8_t *>(a.partial + (token * s.nh + head) * HD)
                                            : reinterpret_cast<uint8_t *>(a.r.out) +
                                                  (token * a.r.out_stride + (long long)head * HD) * (narrow ? 2 : 4);
            const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
            // 32 bytes of each of the warp's rows, at byte `at` of the row: through
            // shared memory, so that two lanes store a whole sector
            auto store32 = [&](uint4 y0, uint4 y1, int at) {
                const int sw = (lane >> 2) & 1;
                *reinterpret_cast<uint4 *>(stage + lane * 32 + (sw << 4)) = y0;
                *reinterpret_cast<uint4 *>(stage + lane * 32 + ((sw ^ 1) << 4)) = y1;
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int rr = 16 * k + (lane >> 1), c = lane & 1;
                    const uint4 y = *reinterpret_cast<const uint4 *>(stage + rr * 32 + ((c ^ ((rr >> 2) & 1)) << 4));
                    uint8_t *d = reinterpret_cast<uint8_t *>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out_row), rr));
                    if (live_rows >> rr & 1) *reinterpret_cast<uint4 *>(d + at + 16 * c) = y;
                }
                __syncwarp();
            };
            auto put = [&](float f, int col, const float (&o)[16]) {  // columns col .. col + 15 of this thread's row
                if (narrow) {
                    store32(make_uint4(pack_bf16(o[0] * f, o[1] * f), pack_bf16(o[2] * f, o[3] * f),
                                       pack_bf16(o[4] * f, o[5] * f), pack_bf16(o[6] * f, o[7] * f)),
                            make_uint4(pack_bf16(o[8] * f, o[9] * f), pack_bf16(o[10] * f, o[11] * f),
                                       pack_bf16(o[12] * f, o[13] * f), pack_bf16(o[14] * f, o[15] * f)),
                            2 * col);
                } else {
                    auto word = [&](int e) { return __float_as_uint(o[e] * f); };
#pragma unroll
                    for (int e = 0; e < 16; e += 8)
                        store32(make_uint4(word(e), word(e + 1), word(e + 2), word(e + 3)),
                                make_uint4(word(e + 4), word(e + 5), word(e + 6), word(e + 7)), 4 * (col + e));
                }
            };
            // partials: [slot][M-tile][hd / 4][row] float4, so that a warp's rows are one run
            auto part_at = [&](int slot) {
                return reinterpret_cast<float4 *>(p.part) + ((size_t)slot * 2 + i) * (HD / 4) * kTileRows + row;
            };
            auto part_ml_at = [&](int slot) { return p.part_ml + ((size_t)slot * 2 + i) * kTileRows + row; };
            const int slot = 2 * blockIdx.x + (x.u0 == x.seg0 ? 1 : 0);
            const float mm = m == -INFINITY ? m : m * mult, ll = l;  // the row's maximum (log2 scale) and sum
            auto read_o = [&](int q, float (&o)[16]) {  // 16 columns of O
                uint32_t v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = 0;
                if (ok) {
                    tmem_ld16(to + 16 * q, v);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __uint_as_float(v[e]);
            };
            const float f = a.prefix_run ? 1.f : ll == 0.f ? 0.f : 1.f / ll;
            float odd[2] = {0.f, 0.f};  // the largest |element| of O; NaN if one is
#pragma unroll 1
            for (int q = 0; q < HD / 16; ++q) {
                float o[16];
                read_o(q, o);
#pragma unroll
                for (int e = 0; e < 16; e += 2) odd[e >> 3] = max3_nan(odd[e >> 3], fabsf(o[e]), fabsf(o[e + 1]));
                if (whole) {
                    put(f, 16 * q, o);
                } else if (live) {
                    float4 *d = part_at(slot) + 4 * q * kTileRows;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        d[e * kTileRows] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
            }
            // A row's weight of a position that it does not see is 0, and so is its
            // product with that position's V, unless V is infinite or NaN there:
            // k_paged_join then sums such rows again.
            if (!(odd[0] + odd[1] < INFINITY) && live && !a.prefix_run) p.header[kPhOdd] = 1;
            if (live) {
                if (!whole)
                    *part_ml_at(slot) = make_float2(mm, ll);
                else if (a.prefix_run)
                    a.partial_ml[token * s.nh + head] = make_float2(mm, ll);
            }
            if (ok) tc_fence_before_sync();
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
}

// Where k_paged_rows256 met infinities or NaN: the rows of the items that the
// split did not cut whose results are such, again by the formula.  Blocks take
// the items in turn.
template <int HD>
__device__ __noinline__ void mend_whole_items(const PagedShape s, const PagedPlanView p, const RowsParams a) {
    const int i = blockIdx.y, col = 32 * blockIdx.z, row = threadIdx.x;
    const int units = p.header[kPhUnits], items = p.header[kPhItems], per = p.header[kPhPer];
    for (int k = blockIdx.x; k < items * s.nkv; k += gridDim.x) {
        const int g = k / items, item = k - g * items;
        const int seg0 = g * units + p.unit_at[item] + kPagedItemCost, seg1 = g * units + p.unit_at[item + 1];
        const PagedItem it = p.items[item];
        if (seg0 / per != (seg1 - 1) / per || i * kTileRows + row >= it.nrows) continue;
        mend_row<HD>(s, a, it, g, it.row0 + i * kTileRows + row, col, 32);
    }
}

// The items that the split cut: block (c, M-tile, 32 columns) joins, in
// position order, the partials of the item that begins in CTA c's run and
// does not end there (a run begins at most one such item).  A thread a row.  Then,
// where there is need, the rows that infinities or NaN have spoilt are mended.
template <int HD>
__device__ __forceinline__ void join_cut_item(const PagedShape &s, const PagedPlanView &p, const Rows256Params &a, int units,
                                              int per, int odd) {
    const int c = blockIdx.x, i = blockIdx.y, col = 32 * blockIdx.z, row = threadIdx.x;
    const int all = units * s.nkv, cut = (c + 1) * per;
    if ((long long)(c + 1) * per >= all) return;
    const int g = cut / units, item = p.start[c + 1];
    const PagedItem it = p.items[item];
    const int seg0 = g * units + p.unit_at[item] + kPagedItemCost, seg1 = g * units + p.unit_at[item + 1];
    if (seg0 >= cut || seg0 / per != c) return;  // it begins later, or began before
    const int last = (seg1 - 1) / per, n = min(kTileRows, it.nrows - i * kTileRows);
    if (row >= n) return;
    const size_t tile = (size_t)kTileRows * (HD / 4);
    const float4 *part = reinterpret_cast<const float4 *>(p.part) + i * tile + (size_t)(col / 4) * kTileRows + row;
    const float2 *ml = p.part_ml + (size_t)i * kTileRows + row;
    auto slot_of = [&](int k) { return (size_t)(2 * k + (k == c ? 1 : 0)) * 2; };  // in M-tiles
    float m = -INFINITY, l = 0.f, o[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = 0.f;
#pragma unroll 2
    for (int k = c; k <= last; ++k) {
        const float2 v = ml[slot_of(k) * kTileRows];
        const float4 *d = part + slot_of(k) * tile;
        float4 y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = d[e * kTileRows];
        const float mn = fmaxf(m, v.x), f = mn == -INFINITY ? 0.f : exp2_approx(m - mn);
        const float w = v.x == -INFINITY ? 0.f : exp2_approx(v.x - mn);
        l = l * f + v.y * w;
        m = mn;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[4 * e] = o[4 * e] * f + y[e].x * w;
            o[4 * e + 1] = o[4 * e + 1] * f + y[e].y * w;
            o[4 * e + 2] = o[4 * e + 2] * f + y[e].z * w;
            o[4 * e + 3] = o[4 * e + 3] * f + y[e].w * w;
        }
    }
    const int r = it.row0 + i * kTileRows + row, tok = fdiv(r, s.by_group), head = g * s.group + r - tok * s.group;
    const long long token = it.q0 + tok;
    if (!a.prefix_run && a.r.out_bf16) {
        const float f = l == 0.f ? 0.f : 1.f / l;
        uint16_t *d = reinterpret_cast<uint16_t *>(a.r.out) + token * a.r.out_stride + (long long)head * HD + col;
#pragma unroll
        for (int e = 0; e < 32; e += 8)
            *reinterpret_cast<uint4 *>(d + e) =
                make_uint4(pack_bf16(o[e] * f, o[e + 1] * f), pack_bf16(o[e + 2] * f, o[e + 3] * f),
                           pack_bf16(o[e + 4] * f, o[e + 5] * f), pack_bf16(o[e + 6] * f, o[e + 7] * f));
    } else {
        const float f = a.prefix_run ? 1.f : l == 0.f ? 0.f : 1.f / l;
        float *d = a.prefix_run ? a.partial + (token * s.nh + head) * HD + col
                                : reinterpret_cast<float *>(a.r.out) + token * a.r.out_stride + (long long)head * HD + col;
#pragma unroll
        for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4 *>(d + e) = make_float4(o[e] * f, o[e + 1] * f, o[e + 2] * f, o[e + 3] * f);
        if (a.prefix_run && col == 0) a.partial_ml[token * s.nh + head] = make_float2(m, l);
    }
    if (odd) mend_row<HD>(s, a.r, it, g, r, col, 32);
}
template <int HD>
__global__ void __launch_bounds__(kTileRows) k_paged_join(const PagedShape s, const PagedPlanView p,
                                                          const Rows256Params a) {
    pdl_wait();
    const int units = p.header[kPhUnits], per = p.header[kPhPer], odd = a.prefix_run ? 0 : p.header[kPhOdd];
    join_cut_item<HD>(s, p, a, units, per, odd);
    if (odd) mend_whole_items<HD>(s, p, a.r);
}

}  // namespace m1
