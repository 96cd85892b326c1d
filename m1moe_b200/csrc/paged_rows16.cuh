// paged_rows16.cuh — attention of at most 16 rows (new tokens x heads of one
// KV head) per item over a paged cache: the decode step's kernel (sm_100a).
//
//   out[r] = sum_p w(r, p) v[p] / sum_p w(r, p),
//   w(r, p) = exp(cap(scale q[r] . k[p]) - m_r) over the positions row r sees.
//
// It reads each K and V row of a (sequence, KV head) once for all the rows
// that share it, so HBM bounds it.  Work is cut evenly in units of 16
// positions (8 KB at hd 128) over every warp of the GPU, whatever the lengths are
// (paged.cuh); a warp streams its run of units through a ring of its own in
// shared memory (cp.async, 16 bytes a lane: pages may be as small as 16
// rows, positions outside the item are filled with zeros, so what lies in a
// page's unused rows never enters a sum) and no warp waits for another
// before its run ends.  A unit is two m16n8k16 products for the scores and
// 16 positions' weights times V; the tile's 16 rows are mostly padding in a
// decode step, which costs nothing while the copies are the bound.  A
// 16-byte chunk c of row r is stored at chunk c ^ (r & 7), so that the eight
// rows of an ldmatrix fall in different banks.  Scores, maxima, sums and
// weighted values are fp32; the weights are rounded to bf16 for the second
// product (the sum takes them unrounded), an error of 2^-9 of each weight
// beside the output's own rounding of 2^-9.
//
// Measured back to back in a CUDA graph: one token over 2048 positions of 16
// heads 12.3 us (four dependent loads, one round of copies and two merges; 2.6
// us at HBM rate); 64 sequences of 37 to 16,000 positions, 32/8 heads, 113 us =
// 5.4 TB/s, 83 % of the measured copy rate; 200 sequences of 20 to 1500, 79 us =
// 4.1 TB/s; 32 sequences of 4 new tokens and up to 8,000 positions, 16/4 heads,
// 28 us = 3.0 TB/s.
#pragma once

#include "paged.cuh"

namespace m1 {

struct RowsParams {
    const uint16_t *q;
    long long q_stride;  // elements between tokens
    const uint16_t *k, *v;
    const int *table;
    float scale, cap;
    void *out;
    int out_bf16;
    long long out_stride;
    int stages;          // ring stages per warp
    int part_rows;       // rows kept of a partial: group * max_q
    const float *prefix_part;  // [total_q][nh][hd] merged in when the header names a prefix
    const float2 *prefix_ml;   // [total_q][nh]
    float *partial;            // not NULL: this launch is the prefix's pass -- all rows see all of it --
    float2 *partial_ml;        // and leaves each row's values and (maximum, sum) here
};

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// tanh(x) / x as a polynomial in y = x^2 for |x| <= 1, degree 5 (least largest
// relative error, 5.9e-7, by Remez exchange).
constexpr float kTanh0 = 0.9999994039535522f, kTanh1 = -0.3332904279232025f, kTanh2 = 0.13281433284282684f,
                kTanh3 = -0.051605675369501114f, kTanh4 = 0.016743114218115807f, kTanh5 = -0.003067060373723507f;

// A capped score in units of log2: cap * tanh(x) * log2(e) with x = score / cap
// = dot * cs; `near` is its value where |x| <= 1: score * log2(e) * tanh(x) / x.
// Beyond, tanh(x) = 1 - 2 / (1 + e^2x).  The error is relative to the score,
// whatever the cap: 1e-7 of the second form is beside a value above 0.76.
__device__ __forceinline__ float cap_far(float x, float cap) {
    return cap * kLog2e * (1.f - __fdividef(2.f, 1.f + exp2_approx(x * (2.f * kLog2e))));
}
__device__ __forceinline__ float cap_score(float x, float near, float cap) {
    const float far = cap_far(x, cap);
    float r;  // (where the compiler branches here, most warps take both sides, element after element)
    asm("{ .reg .pred p; setp.le.f32 p, %1, 0f3F800000; selp.f32 %0, %2, %3, p; }"
        : "=f"(r)
        : "f"(fabsf(x)), "f"(near), "f"(far));
    return r;
}
__device__ __forceinline__ float cap_score(float dot, float scale_log2, float cap, float cs) {
    const float x = dot * cs, y = x * x;
    float t = fmaf(kTanh5, y, kTanh4);
    t = fmaf(t, y, kTanh3);
    t = fmaf(t, y, kTanh2);
    t = fmaf(t, y, kTanh1);
    t = fmaf(t, y, kTanh0);
    return cap_score(x, dot * scale_log2 * t, cap);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Wait until at most n (0..3) of this thread's copy groups are in flight.
__device__ __forceinline__ void cp_async_wait(int n) {
    if (n == 0)
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (n == 1)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (n == 2)
        asm volatile("cp.async.wait_group 2;" ::: "memory");
    else
        asm volatile("cp.async.wait_group 3;" ::: "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Infinities and NaN in V.  A row's weight of a position that it does not see is
// 0, and so is its product with that position's V -- unless V is infinite or NaN
// there.  Where rows of one item see different positions and a row's sums have
// come out infinite or NaN, they are taken again by what follows, one thread a
// row and some columns, over the positions that the row sees and no others.
// (Functions of their own, called after the loops that always run: within these
// their calls cost 4 %, their code 2 to 7 %.)
struct SeenRow {
    const uint16_t *q, *k, *v;  // the row's query; the pools
    const int *pages;           // the sequence's row of the page table
    int nkv, g, page_shift, num_pages, p0, p1;
    float scale_log2, cap, cs, ref;  // ref: the maximum that the row's weights are relative to
};
template <int N>
struct Columns {
    float x[N];
};
// The pool row of position p, or -1 (its K and V count as zeros; the copies have
// reported the page).
__device__ __forceinline__ long long seen_at(const SeenRow &r, int p) {
    const int page = __ldg(r.pages + (p >> r.page_shift));
    if ((unsigned)page >= (unsigned)r.num_pages) return -1;
    return ((long long)page * r.nkv + r.g) << r.page_shift | (p & ((1 << r.page_shift) - 1));
}
// Its score in units of log2.
template <int HD>
__device__ __forceinline__ float seen_score(const SeenRow &r, long long row) {
    const uint32_t *k = reinterpret_cast<const uint32_t *>(r.k + row * HD), *q = reinterpret_cast<const uint32_t *>(r.q);
    float dot = 0.f;
#pragma unroll 4
    for (int d = 0; d < HD / 2; ++d) {
        const uint32_t a = q[d], b = k[d];
        dot = fmaf(__uint_as_float(a << 16), __uint_as_float(b << 16), dot);
        dot = fmaf(__uint_as_float(a & 0xFFFF0000u), __uint_as_float(b & 0xFFFF0000u), dot);
    }
    return r.cap > 0.f ? cap_score(dot, r.scale_log2, r.cap, r.cs) : dot * r.scale_log2;
}
// N columns from `col` on.
template <int HD, int N>
__device__ __noinline__ Columns<N> sum_seen(const SeenRow r, int col) {
    Columns<N> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.x[e] = 0.f;
#pragma unroll 1
    for (int p = r.p0; p <= r.p1; ++p) {
        const long long row = seen_at(r, p);
        if (row < 0) continue;
        const uint32_t *v = reinterpret_cast<const uint32_t *>(r.v + row * HD + col);
        const float w = __bfloat162float(__float2bfloat16_rn(exp2_approx(seen_score<HD>(r, row) - r.ref)));
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const uint32_t b = v[e / 2];
            o.x[e] = fmaf(w, __uint_as_float(b << 16), o.x[e]);
            o.x[e + 1] = fmaf(w, __uint_as_float(b & 0xFFFF0000u), o.x[e + 1]);
        }
    }
    return o;
}
// Row `row` of an item.
template <int HD>
__device__ __forceinline__ SeenRow seen_row(const PagedShape &s, const RowsParams &a, const PagedItem &it, int g, int row) {
    const int tok = fdiv(row, s.by_group);
    SeenRow x;
    x.q = a.q + (long long)(it.q0 + tok) * a.q_stride + (long long)(g * s.group + row - tok * s.group) * HD;
    x.k = a.k, x.v = a.v;
    x.pages = a.table + (size_t)it.seq * s.max_pages;
    x.nkv = s.nkv, x.g = g, x.page_shift = s.page_shift, x.num_pages = s.num_pages;
    x.p1 = it.len - it.nq + tok;
    x.p0 = first_seen(x.p1, s.window);
    x.scale_log2 = a.scale * kLog2e, x.cap = a.cap, x.cs = a.cap > 0.f ? a.scale / a.cap : 0.f;
    x.ref = 0.f;
    return x;
}
// Which of columns col .. col + n - 1 (n even, at most 64) of V at position p are
// infinite or NaN (bits above `from`: 0x7F7F) or NaN alone (0x7F80).
__device__ __forceinline__ unsigned long long odd_columns(const SeenRow &r, int hd, int p, int col, int n,
                                                          uint32_t from = 0x7F7Fu) {
    const long long row = seen_at(r, p);
    if (row < 0) return 0;
    const uint32_t *v = reinterpret_cast<const uint32_t *>(r.v + row * hd + col);
    unsigned long long odd = 0;
#pragma unroll 4
    for (int e = 0; e < n; e += 2) {
        const uint32_t b = v[e / 2];
        odd |= (unsigned long long)(((b & 0x7FFFu) > from ? 1 : 0) | ((b >> 16 & 0x7FFFu) > from ? 2 : 0)) << e;
    }
    return odd;
}
// Columns col .. col + n - 1 (n a multiple of 8, at most 64) of a row's result,
// summed again where they are infinite or NaN and a position that came in with
// the item's units, but that this row does not see, may be why.
template <int HD>
__device__ __noinline__ void mend_row(const PagedShape s, const RowsParams a, const PagedItem it, int g, int row, int col,
                                      int n) {
    const int tok = fdiv(row, s.by_group);
    const long long at = (long long)(it.q0 + tok) * a.out_stride + (long long)(g * s.group + row - tok * s.group) * HD + col;
    __nv_bfloat16 *narrow = reinterpret_cast<__nv_bfloat16 *>(a.out) + at;
    float *wide = reinterpret_cast<float *>(a.out) + at;
    unsigned long long odd = 0, why = 0;
    for (int c = 0; c < n; ++c) {
        const float y = a.out_bf16 ? __bfloat162float(narrow[c]) : wide[c];
        odd |= (unsigned long long)(y * 0.f != 0.f) << c;
    }
    if (!odd) return;
    SeenRow x = seen_row<HD>(s, a, it, g, row);
    // (a NaN at its own position makes the result NaN, whatever else came in)
    if (x.p1 >= 0) odd &= ~odd_columns(x, HD, x.p1, col, n, 0x7F80u);
    const int p0 = it.len - it.nq + fdiv(it.row0, s.by_group), p1 = it.len - it.nq + fdiv(it.row0 + it.nrows - 1, s.by_group);
    const int end = min(it.len, (max(p1, 0) / s.unit + 1) * s.unit);  // of the item's last unit (it has one at least)
    for (int p = first_seen(p0, s.window); p < x.p0; ++p) why |= odd_columns(x, HD, p, col, n);
    for (int p = max(0, x.p1 + 1); p < end; ++p) why |= odd_columns(x, HD, p, col, n);
    odd &= why;
    if (!odd) return;
    float m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int p = x.p0; p <= x.p1; ++p) {
        const long long r = seen_at(x, p);
        const float y = r < 0 ? 0.f : seen_score<HD>(x, r), top = fmaxf(m, y);
        l = l * (m == -INFINITY ? 0.f : exp2_approx(m - top)) + (y == -INFINITY ? 0.f : exp2_approx(y - top));
        m = top;
    }
    x.ref = m == -INFINITY ? 0.f : m;
    const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
    for (int c = 0; c < n; c += 8) {
        if (!(odd >> c & 0xFF)) continue;
        const Columns<8> y = sum_seen<HD, 8>(x, col + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (!(odd >> (c + e) & 1)) continue;
            if (a.out_bf16)
                narrow[c + e] = __float2bfloat16_rn(y.x[e] * f);
            else
                wide[c + e] = y.x[e] * f;
        }
    }
}
// The rows of the items that lie whole in a warp's units [begin, end), half a
// row a lane, and of the items that its CTA joined.
template <int HD>
__device__ __noinline__ void mend_finished(const PagedShape s, const PagedPlanView p, const RowsParams a, int begin, int end,
                                           int item, const int2 *done, int done_n) {
    const int units = p.header[kPhUnits], items = p.header[kPhItems], lane = threadIdx.x & 31;
    for (int g = begin < end ? begin / units : 0; begin < end;) {
        const int seg0 = g * units + p.unit_at[item], seg1 = g * units + p.unit_at[item + 1];
        if (seg1 > end) break;
        const PagedItem it = p.items[item];
        if (seg0 >= begin && (lane & 15) < it.nrows)
            mend_row<HD>(s, a, it, g, it.row0 + (lane & 15), (lane >> 4) * (HD / 2), HD / 2);
        if (seg1 == end) break;
        if (++item == items) item = 0, ++g;
    }
    for (int k = 0; k < done_n; ++k) {
        const PagedItem it = p.items[done[k].y];
        for (int r = threadIdx.x >> 5; r < it.nrows; r += kPagedWarps)
            if (lane < HD / 8) mend_row<HD>(s, a, it, done[k].x, it.row0 + r, lane * 8, 8);
    }
}

// A warp's place in the work: unit u of [u, end) lies in item `item` of KV
// head g; [seg0, seg1) are that item's units.
struct UnitCursor {
    int u, end, g, item, seg0, seg1;
    __device__ __forceinline__ void locate(const PagedPlanView &p, int units) {
        seg0 = g * units + p.unit_at[item];
        seg1 = g * units + p.unit_at[item + 1];
    }
    __device__ __forceinline__ void next_item(const PagedPlanView &p, int units, int items) {
        if (++item == items) item = 0, ++g;
        locate(p, units);
    }
};

// Merge of n partials of one row, 4 (HD 128) or 2 (HD 64) output elements a
// lane; get(i, m, l, o) gives partial i.
template <int HD, class Get>
__device__ __forceinline__ void merge_partials(int n, Get get, float &m, float &l, float (&o)[HD / 32]) {
    constexpr int E = HD / 32;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int i = 0; i < n; ++i) {
        float mi, li, oi[E];
        get(i, mi, li, oi);
        const float mn = fmaxf(m, mi);
        const float c = m == -INFINITY ? 0.f : exp2_approx(m - mn);
        const float ci = mi == -INFINITY ? 0.f : exp2_approx(mi - mn);
        l = l * c + li * ci;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + oi[e] * ci;
        m = mn;
    }
}

template <int HD>
__device__ __forceinline__ void load_vec(const float *p, float (&o)[HD / 32]) {
    if constexpr (HD == 128) {
        const float4 x = *reinterpret_cast<const float4 *>(p);
        o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
    } else {
        const float2 x = *reinterpret_cast<const float2 *>(p);
        o[0] = x.x, o[1] = x.y;
    }
}
template <int HD>
__device__ __forceinline__ void store_vec(float *p, const float (&o)[HD / 32]) {
    if constexpr (HD == 128)
        *reinterpret_cast<float4 *>(p) = make_float4(o[0], o[1], o[2], o[3]);
    else
        *reinterpret_cast<float2 *>(p) = make_float2(o[0], o[1]);
}
template <int HD>
__device__ __forceinline__ void store_out(const RowsParams &a, long long at, const float (&o)[HD / 32]) {
    if (a.out_bf16) {
        uint16_t *p = reinterpret_cast<uint16_t *>(a.out) + at;
        if constexpr (HD == 128)
            *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
        else
            *reinterpret_cast<uint32_t *>(p) = pack_bf16(o[0], o[1]);
    } else {
        store_vec<HD>(reinterpret_cast<float *>(a.out) + at, o);
    }
}

template <int HD>
__device__ __forceinline__ void load_vec_cg(const float *p, float (&o)[HD / 32]) {
    if constexpr (HD == 128) {
        const float4 x = __ldcg(reinterpret_cast<const float4 *>(p));
        o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
    } else {
        const float2 x = __ldcg(reinterpret_cast<const float2 *>(p));
        o[0] = x.x, o[1] = x.y;
    }
}

// One row's end: the shared prefix's partial (if any) joins, then the row is
// divided by its sum and written.  A row that saw nothing is zero.
template <int HD>
__device__ __forceinline__ void finish_row(const PagedShape &s, const RowsParams &a, int prefix, int token, int head,
                                           float m, float l, float (&o)[HD / 32]) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long r = (long long)token * s.nh + head;
    if (a.partial) {
        store_vec<HD>(a.partial + r * HD + lane * E, o);
        if (lane == 0) a.partial_ml[r] = make_float2(m, l);
        return;
    }
    if (prefix > 0) {
        const float2 ml = a.prefix_ml[r];
        float x[E];
        load_vec<HD>(a.prefix_part + r * HD + lane * E, x);
        const float mn = fmaxf(m, ml.x);
        const float c = m == -INFINITY ? 0.f : exp2_approx(m - mn);
        const float ci = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - mn);
        l = l * c + ml.y * ci;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + x[e] * ci;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= inv;
    store_out<HD>(a, (long long)token * a.out_stride + (long long)head * HD + lane * E, o);
}

// Shared memory of one warp: `stages` units of K and V, then the rows of a
// partial that ended before the warp's run did.
template <int HD>
__host__ __device__ constexpr int rows16_unit_bytes() {
    return 2 * kPagedUnitSmall * HD * 2;
}

// What a warp left unfinished: a first segment begun before its run and
// ended in it (`front`, kept apart), and a last one that its run did not end.
struct Rows16Left {
    int front, front_g, front_item;
    int open_right, open_left, g, item;
};

// kCap: scores are capped (a.cap > 0).  kMany: rows of an item may see different
// positions (several new tokens of a sequence).  A kernel of its own each: what
// one step of one short sequence takes is much the first fetch of its code (us in
// one kernel for both caps, and in two: one uncapped token over 2048 positions
// 12.8 and 12.3; 64 sequences to 16,000 114 and 112; 200 on a shared prefix 198
// and 195).
template <int HD, bool kCap, bool kMany>
__global__ void __launch_bounds__(kPagedWarps * 32, 1) k_paged_rows16(const PagedShape s, const PagedPlanView p,
                                                                      const RowsParams a) {
    constexpr int E = HD / 32, KS = HD / 16, NT = HD / 8, CH = HD / 8;  // CH: 16-byte chunks per row
    constexpr int kRow = HD * 2, kHalf = kPagedUnitSmall * kRow, kUnit = 2 * kHalf;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Rows16Left left[kPagedWarps];
    __shared__ float2 ml_front[kPagedWarps][kPagedRowsSmall], ml_last[kPagedWarps][kPagedRowsSmall];
    __shared__ int sm_last;
    __shared__ int2 done[kPagedWarps + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cta = blockIdx.x;
    const int warp_bytes = a.stages * kUnit + a.part_rows * HD * 4;
    uint8_t *ring = smem + (size_t)warp * warp_bytes;
    float *front = reinterpret_cast<float *>(ring + a.stages * kUnit);
    const uint32_t ring_addr = smem_addr(ring);
    pdl_wait();
    const int start = p.start[cta * kPagedWarps + warp];
    const int units = p.header[kPhUnits], items = p.header[kPhItems], per = p.header[kPhPer];
    const int prefix = a.partial ? 0 : p.header[kPhPrefix];
    int *status = p.status;
    const int all = units * s.nkv;
    const int c0 = min(cta * per, all), c1 = min(all, c0 + per);
    const int pw = (c1 - c0 + kPagedWarps - 1) / kPagedWarps;
    UnitCursor cur;
    cur.u = min(c1, c0 + warp * pw);
    cur.end = min(c1, cur.u + pw);
    const bool work = cur.u < cur.end;
    const int begin = cur.u;
    Rows16Left mine = {0, 0, 0, 0, 0, 0, 0};
    [[maybe_unused]] float odd = 0.f;  // NaN once a finished row's sums were infinite or NaN
    if (work) {
        cur.g = cur.u / units;
        cur.item = start;
        cur.locate(p, units);
        UnitCursor ld = cur;  // the loader runs ahead
        PagedItem ld_item = p.items[ld.item];
        auto item_lo = [&](const PagedItem &it) {  // first position any row of the item sees
            return max(prefix, first_seen(it.len - it.nq + fdiv(it.row0, s.by_group), s.window));
        };
        int ld_lo = item_lo(ld_item);
        int slot = 0;
        auto load_unit = [&]() {
            if (ld.u < ld.end) {
                if (ld.u == ld.seg1) {
                    ld.next_item(p, units, items);
                    ld_item = p.items[ld.item];
                    ld_lo = item_lo(ld_item);
                }
                const int pos = (ld_item.unit0 + ld.u - ld.seg0) * kPagedUnitSmall;
                // all 16 positions lie in one page (page sizes are multiples of 16)
                int row = -1;
                if (pos < ld_item.len) row = paged_row(s, a.table, ld_item.seq, ld.g, pos, status);
                const long long at = (long long)max(row, 0) * HD;
                const uint32_t dst = ring_addr + slot * kUnit;
#pragma unroll
                for (int i = 0; i < kPagedUnitSmall * CH / 32; ++i) {
                    const int r = (i * 32 + lane) / CH, c = (i * 32 + lane) % CH;
                    const bool ok = row >= 0 && pos + r < ld_item.len && pos + r >= ld_lo;
                    const uint32_t d = dst + r * kRow + ((c ^ (r & 7)) << 4);
                    const long long src = ok ? at + r * HD + c * 8 : 0;
                    cp_async16(d, a.k + src, ok);
                    cp_async16(d + kHalf, a.v + src, ok);
                }
                ++ld.u;
                if (++slot == a.stages) slot = 0;
            }
            cp_async_commit();
        };
        for (int i = 0; i < a.stages - 1; ++i) load_unit();
        int use = 0;
        uint32_t qf[KS][4];
        float o[NT][4], m[2], l[2];
        int hi[2], lo[2];  // positions the lane's two rows see
        int min_hi = 0, max_lo = 0;
        const float sl2 = a.scale * kLog2e, cs = kCap ? a.scale / a.cap : 0.f;
        PagedItem it;
        auto open_segment = [&]() {
            it = p.items[cur.item];
            const int q0 = it.q0, nq = it.nq, len = it.len;
            const uint16_t *qr[2];
            bool ok[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = lane / 4 + 8 * h;
                ok[h] = r < it.nrows;
                const int row = it.row0 + (ok[h] ? r : 0), tok = fdiv(row, s.by_group);
                qr[h] = a.q + (long long)(q0 + tok) * a.q_stride + (long long)(cur.g * s.group + row - tok * s.group) * HD;
                hi[h] = a.partial ? len - 1 : len - nq + tok;
                lo[h] = max(prefix, first_seen(hi[h], s.window));
                m[h] = -INFINITY;
                l[h] = 0.f;
            }
            min_hi = a.partial ? len - 1 : len - nq + fdiv(it.row0, s.by_group);
            const int max_hi = len - nq + fdiv(it.row0 + it.nrows - 1, s.by_group);
            max_lo = max(prefix, first_seen(max_hi, s.window));
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int h = j & 1, at = 16 * k + 8 * (j >> 1) + 2 * (lane & 3);
                    qf[k][j] = ok[h] ? *reinterpret_cast<const uint32_t *>(qr[h] + at) : 0u;
                }
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        };
        // this lane's part of the row sums joins its quad's
        auto row_sums = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            }
        };
        // the segment's rows as a partial in shared memory
        auto store_partial = [&](float *dst, float2 *ml) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = lane / 4 + 8 * h;
                if (r < it.nrows) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        *reinterpret_cast<float2 *>(dst + r * HD + 8 * n + 2 * (lane & 3)) =
                            make_float2(o[n][2 * h], o[n][2 * h + 1]);
                    if ((lane & 3) == 0) ml[r] = make_float2(m[h], l[h]);
                }
            }
            __syncwarp();
        };
        // the finished rows of an item, straight from the accumulators
        auto write_rows = [&]() {
            const int q0 = it.q0, pre = it.len > 0 ? prefix : 0;  // an idle slot has none
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = lane / 4 + 8 * h;
                if (r >= it.nrows) continue;
                const int row = it.row0 + r, tok = fdiv(row, s.by_group);
                const int token = q0 + tok, head = cur.g * s.group + row - tok * s.group;
                const long long pr = (long long)token * s.nh + head;
                float c = 1.f, ci = 0.f, sum = l[h];
                if (pre > 0) {
                    const float2 ml = a.prefix_ml[pr];
                    const float mn = fmaxf(m[h], ml.x);
                    c = m[h] == -INFINITY ? 0.f : exp2_approx(m[h] - mn);
                    ci = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - mn);
                    sum = sum * c + ml.y * ci;
                }
                const float inv = a.partial ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
                if (a.partial && (lane & 3) == 0) a.partial_ml[pr] = make_float2(m[h], sum);
                const long long at = (long long)token * a.out_stride + (long long)head * HD;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int col = 8 * n + 2 * (lane & 3);
                    float x0 = o[n][2 * h] * c, x1 = o[n][2 * h + 1] * c;
                    if (pre > 0) {
                        const float2 y = *reinterpret_cast<const float2 *>(a.prefix_part + pr * HD + col);
                        x0 += y.x * ci, x1 += y.y * ci;
                    }
                    x0 *= inv, x1 *= inv;
                    if (a.partial)
                        *reinterpret_cast<float2 *>(a.partial + pr * HD + col) = make_float2(x0, x1);
                    else if (a.out_bf16)
                        *reinterpret_cast<uint32_t *>(reinterpret_cast<uint16_t *>(a.out) + at + col) = pack_bf16(x0, x1);
                    else
                        *reinterpret_cast<float2 *>(reinterpret_cast<float *>(a.out) + at + col) = make_float2(x0, x1);
                }
            }
        };
        open_segment();
        for (; cur.u < cur.end; ++cur.u) {
            load_unit();
            if (cur.u == cur.seg1) {
                cur.next_item(p, units, items);
                open_segment();
            }
            cp_async_wait(a.stages - 1);
            __syncwarp();
            const uint32_t kb = ring_addr + use * kUnit, vb = kb + kHalf;
            // scores: two n8 tiles of positions
            float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            {
                const int r = (lane & 7) + ((lane >> 4) << 3), cb = (lane >> 3) & 1;
                const uint32_t base = kb + r * kRow;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t b[4];
                    ldsm4(base + (((2 * k + cb) ^ (r & 7)) << 4), b);
                    mma_bf16(sc[0], qf[k], b[0], b[1]);
                    mma_bf16(sc[1], qf[k], b[2], b[3]);
                }
            }
            const int pos = (it.unit0 + cur.u - cur.seg0) * kPagedUnitSmall;
            float mx[2] = {m[0], m[1]};
            const bool whole = pos >= max_lo && pos + kPagedUnitSmall - 1 <= min_hi;
            if constexpr (kCap) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[t][j] = cap_score(sc[t][j], sl2, a.cap, cs);
            } else {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[t][j] *= sl2;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int h = j >> 1;
                    float x = sc[t][j];
                    if (!whole) {
                        const int at = pos + 8 * t + 2 * (lane & 3) + (j & 1);
                        if (at > hi[h] || at < lo[h]) x = -INFINITY;
                    }
                    sc[t][j] = x;
                    mx[h] = fmaxf(mx[h], x);
                }
            float c[2], ref[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                ref[h] = mx[h] == -INFINITY ? 0.f : mx[h];  // nothing seen yet: all weights are 0
                c[h] = exp2_approx(m[h] - ref[h]);
                m[h] = mx[h];
                l[h] *= c[h];
            }
            uint32_t pf[4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = exp2_approx(sc[t][j] - ref[j >> 1]);
                    l[j >> 1] += w[j];
                }
                pf[2 * t] = pack_bf16(w[0], w[1]);
                pf[2 * t + 1] = pack_bf16(w[2], w[3]);
            }
            if (__any_sync(0xffffffffu, c[0] != 1.f || c[1] != 1.f)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    o[n][0] *= c[0], o[n][1] *= c[0];
                    o[n][2] *= c[1], o[n][3] *= c[1];
                }
            }
            {
                const int r = lane & 15, cb = lane >> 4;
                const uint32_t base = vb + r * kRow;
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b[4];
                    ldsm4_t(base + (((n + cb) ^ (r & 7)) << 4), b);
                    mma_bf16(o[n], pf, b[0], b[1]);
                    mma_bf16(o[n + 1], pf, b[2], b[3]);
                }
            }
            __syncwarp();  // the stage may be filled again
            if (++use == a.stages) use = 0;
            if (cur.u + 1 == cur.seg1) {
                row_sums();
                if (cur.seg0 >= begin) {
                    if constexpr (kMany) {
                        float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int n = 0; n < NT; ++n) z[n & 3] += (o[n][0] + o[n][1]) + (o[n][2] + o[n][3]);
                        odd = fmaf((z[0] + z[1]) + (z[2] + z[3]), 0.f, odd);
                    }
                    write_rows();  // the whole item was this warp's
                } else {
                    store_partial(front, ml_front[warp]);
                    mine.front = 1;
                    mine.front_g = cur.g;
                    mine.front_item = cur.item;
                }
            } else if (cur.u + 1 == cur.end) {
                row_sums();
                store_partial(reinterpret_cast<float *>(ring), ml_last[warp]);  // the ring is drained
                mine.open_right = 1;
                mine.open_left = cur.seg0 < begin;
                mine.g = cur.g;
                mine.item = cur.item;
            }
        }
    }
    if (lane == 0) left[warp] = mine;
    __syncthreads();
    // The items that this CTA joins and finishes (one a warp at most, and two cut by its run's ends).
    int done_n = 0;
    auto note = [&](const float (&o)[E]) {
        if constexpr (kMany) {
#pragma unroll
            for (int e = 0; e < E; ++e) odd = fmaf(o[e], 0.f, odd);
        }
    };
    auto finished = [&](int g, int item) {
        if constexpr (kMany) {
            if (threadIdx.x == 0) done[done_n] = make_int2(g, item);
            ++done_n;
        }
    };
    // The warps' unfinished segments, joined item by item in position order:
    // a group starts at a warp whose last segment begins its item (or at warp
    // 0, whatever it begins with) and runs on over the following warps.
    // Every warp takes every eighth row.
    auto join = [&](int w0, bool from_front, int n, bool closed, bool open_left, int g, int item) {
        const PagedItem it = p.items[item];
        const int pre = it.len > 0 ? prefix : 0;
        const bool whole = closed && !open_left;
        if (whole) finished(g, item);
        const int slot = 2 * cta + (open_left ? 0 : 1);
        for (int r = warp; r < it.nrows; r += kPagedWarps) {
            float m, l, o[E];
            merge_partials<HD>(
                n,
                [&](int i, float &mi, float &li, float (&oi)[E]) {
                    const bool f = from_front || (closed && i == n - 1);
                    const float2 ml = f ? ml_front[w0 + i][r] : ml_last[w0 + i][r];
                    mi = ml.x, li = ml.y;
                    const uint8_t *base = smem + (size_t)(w0 + i) * warp_bytes + (f ? a.stages * kUnit : 0);
                    load_vec<HD>(reinterpret_cast<const float *>(base) + r * HD + lane * E, oi);
                },
                m, l, o);
            const int row = it.row0 + r, tok = fdiv(row, s.by_group);
            if (whole) {
                note(o);
                finish_row<HD>(s, a, pre, it.q0 + tok, g * s.group + row - tok * s.group, m, l, o);
            } else {
                const size_t at = (size_t)slot * a.part_rows + r;
                store_vec<HD>(p.part + at * HD + lane * E, o);
                if (lane == 0) p.part_ml[at] = make_float2(m, l);
            }
        }
    };
    int open_n = 0, open_g[2], open_item[2];  // groups that other CTAs' partials complete
    for (int w = 0; w < kPagedWarps; ++w) {
        const Rows16Left h = left[w];
        if (w == 0 && h.front) {
            join(0, true, 1, true, true, h.front_g, h.front_item);
            open_g[open_n] = h.front_g, open_item[open_n++] = h.front_item;
        }
        if (h.open_right && (w == 0 || !h.open_left)) {
            int n = 1;
            bool closed = false;
            for (; w + n < kPagedWarps && !closed; ++n) {
                const Rows16Left &x = left[w + n];
                if (x.front)
                    closed = true;
                else if (!(x.open_right && x.open_left))
                    break;
            }
            join(w, false, n, closed, h.open_left, h.g, h.item);
            if ((!closed || h.open_left) && open_n < 2) open_g[open_n] = h.g, open_item[open_n++] = h.item;
        }
    }
    for (int i = 0; i < open_n; ++i) {
        const int g = open_g[i], item = open_item[i];
        const int first = (g * units + p.unit_at[item]) / per, last = (g * units + p.unit_at[item + 1] - 1) / per;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            int *cnt = p.count + g * items + item;
            sm_last = atomicAdd(cnt, 1) == last - first;
            if (sm_last) *cnt = 0;  // ready for the next call
        }
        __syncthreads();
        if (!sm_last) continue;
        __threadfence();
        const PagedItem it = p.items[item];
        const int pre = it.len > 0 ? prefix : 0;
        for (int r = warp; r < it.nrows; r += kPagedWarps) {
            float m, l, o[E];
            merge_partials<HD>(
                last - first + 1,
                [&](int k, float &mi, float &li, float (&oi)[E]) {
                    // the item's first CTA begins it, the others begin with it
                    const size_t at = (size_t)(2 * (first + k) + (k == 0 ? 1 : 0)) * a.part_rows + r;
                    const float2 ml = __ldcg(p.part_ml + at);
                    mi = ml.x, li = ml.y;
                    load_vec_cg<HD>(p.part + at * HD + lane * E, oi);
                },
                m, l, o);
            const int row = it.row0 + r, tok = fdiv(row, s.by_group);
            note(o);
            finish_row<HD>(s, a, pre, it.q0 + tok, g * s.group + row - tok * s.group, m, l, o);
        }
        finished(g, item);
    }
    if constexpr (kMany) {
        if (__syncthreads_or(odd != odd)) mend_finished<HD>(s, p, a, work ? begin : 0, work ? cur.end : 0, start, done, done_n);
    }
}

}  // namespace m1
