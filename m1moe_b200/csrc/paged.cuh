// paged.cuh — a paged bf16 key/value cache for a ragged batch: the batch's
// plan and the append of new tokens (sm_100a).
//
// Cache of one layer: K and V, each bf16 [num_pages][nkv][page_size][hd], so
// that the rows of one (page, KV head) are one contiguous run.  Position p of
// sequence b lies in page table[b][p / page_size], row p % page_size.  The
// pool's rows are numbered ((page * nkv) + g) * page_size + row; a row number
// fits 31 bits (checked by the host), a byte offset does not and is formed
// in 64.
//
// Plan (k_paged_plan, k_paged_tokens).  One device buffer per batch, made
// from cu_q and kv_len and used by every layer of a step: a checked copy of
// the lengths, each token's (sequence, position), and the attention's work
// split.  The work is a list of items -- a sequence's rows (token, head of
// the KV head's group), `rows` at a time -- per KV head; an item's cost is
// the number of position units its rows can see; the units of all KV heads'
// items, concatenated, are cut into equal runs, one per CTA (and, for the
// 16-row kernel, per warp), whatever the lengths are.  A run that starts or
// ends inside an item leaves a partial (maximum, sum, weighted values); an
// item's partials are merged in position order -- by the last CTA to finish
// it (16 rows) or by a kernel that follows (256 rows: one CTA would read them
// for longer than the launch takes) -- so the result does not depend on the
// order of events.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "pipeline.cuh"

namespace m1 {

// Status bits of a plan (m1moe_cuda_paged_status).
constexpr int kPagedErrLengths = 1;   // cu_q or kv_len out of range or inconsistent
constexpr int kPagedErrPage = 2;      // a page id outside the pool
constexpr int kPagedErrPosition = 4;  // a position outside the rotation table
constexpr int kPagedErrWait = 8;      // a bounded wait gave up

constexpr int kPagedWarps = 8;      // consumer warps of the 16-row kernel
constexpr int kPagedRowsSmall = 16; // rows of an item there: one m16n8k16 tile
constexpr int kPagedUnitSmall = 16; // positions of a unit there
constexpr int kPagedRowsLarge = 256; // rows of an item of the 256-row kernel: two M-tiles of 128
constexpr int kPagedUnitLarge = 128; // positions of a unit there: one K or V tile
// Units that the split adds to each item of the 256-row kernel for what an
// item costs besides its tiles (rows in and out, the pipeline's start and
// end: about 9,500 cycles beside 4,300 for a unit).
constexpr int kPagedItemCost = 2;

// Words of the plan's header.
enum PagedHeader {
    kPhStatus = 0,
    kPhItems = 1,   // items per KV head
    kPhUnits = 2,   // units per KV head
    kPhPer = 3,     // units per CTA
    kPhPrefix = 4,  // positions of the shared prefix in use (0: none)
    kPhOdd = 5,     // a 256-row item's sums met an infinity or a NaN since the plan was made
    kPhWords = 16
};

// One item: rows row0 .. row0 + nrows - 1 of sequence `seq` (row = token
// offset * group + head offset), seen from position unit0 * unit on; and of
// the sequence the first of its nq new tokens and its length, so that one
// load tells all (a worker's first copies wait for every load before them).
struct __align__(16) PagedItem {
    int seq, row0, nrows, unit0;
    int q0, nq, len, unused;
};

struct PagedPlanView {
    int *status;         // the batch's status word (header word 0 of the main split)
    int *header;
    int *cu_q;           // [B + 1]
    int *kv_len;         // [B]
    int2 *tokens;        // [total_q]: (sequence, position)
    PagedItem *items;    // [max_items]
    int *item_at;        // [B + 1]: first item of each sequence
    int *unit_at;        // [max_items + 1]: units before each item
    int *start;          // [workers]: the item each worker starts in
    int *count;          // [nkv * max_items], 16-row kernel: partials that have arrived
    float *part;         // [2 * ctas][rows][hd] weighted values
    float2 *part_ml;     // [2 * ctas][rows] maximum and sum
};

// The shared prefix's results, one partial per row, which the 16-row kernel
// joins to each sequence's own.
struct PagedPrefixView {
    float *part;   // [total_q][nh][hd]
    float2 *ml;    // [total_q][nh]
};

struct PagedShape {
    int nh, nkv, group, hd;
    FastDiv by_group;
    int page_size, page_shift, num_pages;
    int num_seqs, max_pages, total_q, max_q;
    int window, prefix;
    int rows, unit;      // the attention kernel's item rows and unit positions
    int ctas, workers;   // CTAs of the attention grid, and plan start entries
    int min_per;         // fewest units per CTA
    int max_items;
    int prefix_room;     // the plan has room for the shared prefix's pass
    int prefix_rows;     // item rows of the shared prefix's pass: 16 or 256
};

// First position that a token at position p sees (window 0: all).  Tokens
// before position 0 see nothing, and a window may be as large as an int:
// p - window + 1 is formed only where it cannot pass 31 bits.
__device__ __forceinline__ int first_seen(int p, int window) {
    return window == 0 || p < window ? 0 : p - window + 1;
}

// Pool row of position p of sequence b and KV head g, or -1 (with the status
// bit) if the page table names no page of the pool.
__device__ __forceinline__ int paged_row(const PagedShape &s, const int *table, int b, int g, int p, int *status) {
    const int page = __ldg(table + (size_t)b * s.max_pages + (p >> s.page_shift));
    if ((unsigned)page >= (unsigned)s.num_pages) {
        atomicOr(status, kPagedErrPage);
        return -1;
    }
    return (page * s.nkv + g) * s.page_size + (p & (s.page_size - 1));
}

// Exclusive block scan of one int per thread (1024 threads); returns the
// exclusive prefix and the total.
__device__ __forceinline__ int block_scan_1024(int v, int *sm, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // sm is free
    if (lane == 31) sm[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int y = sm[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        sm[lane] = y;
    }
    __syncthreads();
    total = sm[31];
    return x - v + (warp ? sm[warp - 1] : 0);
}

// Largest i in [0, n) with a[i] <= v (a ascending, a[0] <= v).
__device__ __forceinline__ int upper_index(const int *a, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// One CTA: the checked lengths, the items and the work split of one batch.
// Measured with k_paged_tokens: 6 us for one sequence or a few prompts, 7 for 64
// sequences, 19 for 200 with a shared prefix of 256 pages (whose tables it
// compares); once a step, whatever the number of layers.
// Lengths that cannot be right raise the status bit and make the batch an
// empty one, so that no later kernel leaves the buffers.  A sequence may be
// shorter than its new tokens (an idle slot of a fixed-size batch has none
// at all): the tokens before position 0 see nothing and are stored nowhere.
__global__ void __launch_bounds__(1024) k_paged_plan(const PagedShape s, const PagedPlanView p, const int *cu_q,
                                                     const int *kv_len, const int *table, const PagedPlanView p2) {
    __shared__ int sm[32];
    __shared__ int sm_bad, sm_noprefix, sm_lead;
    const int tid = threadIdx.x;
    if (tid == 0) sm_bad = 0, sm_noprefix = 0, sm_lead = s.num_seqs;
    __syncthreads();
    pdl_wait();
    const int capacity = s.max_pages * s.page_size;
    int items = 0;
    for (int b0 = 0; b0 < s.num_seqs; b0 += 1024) {
        const int b = b0 + tid;
        int n = 0;
        if (b < s.num_seqs) {
            const int q0 = cu_q[b], q1 = cu_q[b + 1], t = kv_len[b];
            const bool good = q0 >= 0 && q1 >= q0 && q1 <= s.total_q && q1 - q0 <= s.max_q && t >= 0 &&
                              t <= capacity && (b > 0 || q0 == 0) && (b + 1 < s.num_seqs || q1 == s.total_q);
            if (!good) sm_bad = kPagedErrLengths;
            p.cu_q[b] = q0;
            p.kv_len[b] = t;
            if (b + 1 == s.num_seqs) p.cu_q[b + 1] = q1;
            n = good ? ((q1 - q0) * s.group + s.rows - 1) / s.rows : 0;
            // an idle slot takes no part in the prefix; the others' new tokens follow it
            if (t > 0) {
                if (t - (q1 - q0) < s.prefix) sm_noprefix = 1;
                atomicMin(&sm_lead, b);
            }
        }
        int total;
        const int at = block_scan_1024(n, sm, total);
        if (b < s.num_seqs) p.item_at[b] = items + at;
        items += total;
    }
    if (tid == 0) p.item_at[s.num_seqs] = items;
    __syncthreads();
    if (sm_bad) {  // an empty batch
        items = 0;
        for (int b = tid; b <= s.num_seqs; b += 1024) {
            p.cu_q[b] = 0;
            if (b < s.num_seqs) p.kv_len[b] = 0;
        }
    }
    // the prefix is shared only where the page tables agree
    const int lead = sm_lead;
    if (s.prefix > 0 && lead < s.num_seqs && !sm_bad) {
        const int np = s.prefix >> s.page_shift;
        for (int b = lead + 1 + (tid >> 5); b < s.num_seqs; b += 32) {
            if (p.kv_len[b] == 0) continue;
            bool same = true;
            for (int j = tid & 31; j < np; j += 32)
                same = same && table[(size_t)b * s.max_pages + j] == table[(size_t)lead * s.max_pages + j];
            if (!same) sm_noprefix = 1;
        }
    }
    __syncthreads();
    const int prefix = sm_noprefix || sm_bad || lead == s.num_seqs ? 0 : s.prefix;
    int units = 0;
    for (int i0 = 0; i0 < items; i0 += 1024) {
        const int i = i0 + tid;
        int n = 0;
        if (i < items) {
            const int b = upper_index(p.item_at, s.num_seqs + 1, i);
            const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1], t = p.kv_len[b];
            const int nrow = (q1 - q0) * s.group, r0 = (i - p.item_at[b]) * s.rows;
            PagedItem it;
            it.seq = b;
            it.row0 = r0;
            it.q0 = q0;
            it.nq = q1 - q0;
            it.len = t;
            it.unused = 0;
            it.nrows = min(s.rows, nrow - r0);
            const int first = t - (q1 - q0) + r0 / s.group;  // position of the first and the last row
            const int last = t - (q1 - q0) + (r0 + it.nrows - 1) / s.group;
            it.unit0 = max(prefix, first_seen(first, s.window)) / s.unit;
            // at least one unit, so that an item whose rows see nothing is still written
            n = max(1, (last + s.unit) / s.unit - it.unit0) + (s.rows == kPagedRowsLarge ? kPagedItemCost : 0);
            p.items[i] = it;
        }
        int total;
        const int at = block_scan_1024(n, sm, total);
        if (i < items) p.unit_at[i] = units + at;
        units += total;
    }
    if (tid == 0) p.unit_at[items] = units;
    for (int i = tid; s.rows == kPagedRowsSmall && i < items * s.nkv; i += 1024) p.count[i] = 0;
    __syncthreads();
    const long long all = (long long)units * s.nkv;
    const int per = (int)max((long long)s.min_per, (all + s.ctas - 1) / s.ctas);
    const int nw = s.workers / s.ctas;
    for (int w = tid; w < s.workers && units > 0; w += 1024) {
        // worker w of CTA c: an equal part of the CTA's run [c * per, ...)
        const int c = w / nw;
        const long long c0 = (long long)c * per, c1 = min(all, c0 + per);
        const int pw = (int)((c1 - c0 + nw - 1) / nw);
        const long long u = c0 + (long long)(w - c * nw) * pw;
        p.start[w] = u < c1 ? upper_index(p.unit_at, items + 1, (int)(u % units)) : 0;
    }
    if (tid == 0) {
        // (bits of earlier steps stay until they are reported)
        if (sm_bad) atomicOr(p.status, sm_bad);
        p.header[kPhItems] = items;
        p.header[kPhUnits] = units;
        p.header[kPhPer] = per;
        p.header[kPhPrefix] = prefix;
        p.header[kPhOdd] = 0;
    }
    if (s.prefix == 0) return;
    // the prefix's own split: all rows of the batch, 16 or 256 at a time,
    // against its positions (no items when it is not shared after all)
    const bool big = s.prefix_rows == kPagedRowsLarge;
    const int rows = s.total_q * s.group, unit2 = big ? kPagedUnitLarge : kPagedUnitSmall;
    const int items2 = prefix ? (rows + s.prefix_rows - 1) / s.prefix_rows : 0;
    const int n2 = (prefix + unit2 - 1) / unit2 + (big ? kPagedItemCost : 0), units2 = items2 * n2;
    for (int i = tid; i <= items2; i += 1024) {
        p2.unit_at[i] = i * n2;
        if (i < items2)
            p2.items[i] = PagedItem{lead, i * s.prefix_rows, min(s.prefix_rows, rows - i * s.prefix_rows), 0,
                                    0, s.total_q, prefix, 0};
    }
    for (int i = tid; !big && i < items2 * s.nkv; i += 1024) p2.count[i] = 0;
    const int all2 = units2 * s.nkv, nw2 = big ? 1 : kPagedWarps;
    const int per2 = max(big ? 1 : kPagedWarps, (all2 + s.ctas - 1) / s.ctas);
    for (int w = tid; w < s.ctas * nw2; w += 1024) {
        const int c = w / nw2;
        const long long c0 = (long long)c * per2, c1 = min((long long)all2, c0 + per2);
        const int pw = (int)((c1 - c0 + nw2 - 1) / nw2);
        const long long u = c0 + (long long)(w - c * nw2) * pw;
        p2.start[w] = u < c1 ? (int)(u % units2) / n2 : 0;
    }
    if (tid == 0) {
        p2.header[kPhItems] = items2;
        p2.header[kPhUnits] = units2;
        p2.header[kPhPer] = per2;
        p2.header[kPhPrefix] = prefix;
    }
}

// Each token's sequence and position, (-1, -1) for a token of no sequence or
// before position 0.
__global__ void __launch_bounds__(256) k_paged_tokens(const PagedShape s, const PagedPlanView p) {
    pdl_wait();
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= s.total_q) return;
    int2 v = make_int2(-1, -1);
    if (t >= p.cu_q[0] && t < p.cu_q[s.num_seqs]) {
        const int b = upper_index(p.cu_q, s.num_seqs + 1, t);
        const int pos = p.kv_len[b] - p.cu_q[b + 1] + t;
        if (b < s.num_seqs && pos >= 0) v = make_int2(b, pos);
    }
    p.tokens[t] = v;
}

// out[b] = x[last new token of sequence b] (f32 rows of h), zeros without one.
__global__ void __launch_bounds__(256) k_paged_last(const PagedPlanView p, const float *x, int h, float *out) {
    pdl_wait();
    const int b = blockIdx.x, t = p.cu_q[b + 1] - 1;
    const bool any = t >= p.cu_q[b];
    for (int i = threadIdx.x; i < h; i += 256) out[(long long)b * h + i] = any ? x[(long long)t * h + i] : 0.f;
}

// ----------------------------------------------------------------- append ----
struct AppendParams {
    const void *qkv;
    long long qkv_stride;  // elements between tokens
    const uint16_t *q_norm, *k_norm;
    float eps;
    const float2 *rope;    // [rope_rows][rot / 2] (cos, sin)
    int rope_rows, rot, pairs;
    uint16_t *k, *v;
    uint16_t *q_out;       // [total_q][nh][hd]
    const int *table;
    int heads_per_group;   // heads one group of lanes does of one token
    int groups;            // groups per token
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Two fp32 values in one 64-bit register (packed arithmetic issues once for both).
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Four elements as two packed pairs.
template <bool BF16>
__device__ __forceinline__ void load4x(const void *x, long long at, uint64_t (&v)[2]) {
    if constexpr (BF16) {
        const uint2 w = __ldg(reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(x) + at));
        v[0] = pack2(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u));
        v[1] = pack2(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
    } else {
        const float4 w = __ldg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(x) + at));
        v[0] = pack2(w.x, w.y);
        v[1] = pack2(w.z, w.w);
    }
}
__device__ __forceinline__ uint2 round4(const uint64_t (&v)[2]) {
    float a, b, c, d;
    unpack2(v[0], a, b);
    unpack2(v[1], c, d);
    return make_uint2(pack_bf16(a, b), pack_bf16(c, d));
}

// Append: y = rotate(x * rsqrt(mean(x^2) + eps) * w) of each new query and key
// head, v as it is; q rows go out bf16, k and v rows into their pages.  A
// group of HD / 8 lanes takes a head, two runs of four elements a lane chosen
// so that both elements of every rotated pair are the lane's: (i, i + rot/2)
// from two runs rot/2 apart, or adjacent pairs from two neighbouring runs; the
// lanes past the rotated part hold eight elements of the rest.  All sums in
// fp32, one rounding at the end.  A group keeps its token's place and angles
// over its heads and has the loads of kAppendAhead heads under way.  HBM
// would bound it; what does is the latency of these loads together with the
// instructions (about 80 a warp and two heads, hence the packed arithmetic):
// waiting for loads is the largest stall, and issue slots are 57 % busy.
// Measured: nine prompts, 13.9 thousand tokens of 48 heads bf16 with norm, 91
// us = 3.75 TB/s (57 % of the measured copy rate; 141 us with a head per group
// of lanes and shuffled halves); 2000 tokens f32, 15 us = 5.0 TB/s; one token
// 3.1 us.
constexpr int kAppendAhead = 2;
template <int HD, bool BF16>
__global__ void __launch_bounds__(256, 4) k_paged_append(const PagedShape s, const PagedPlanView p,
                                                         const AppendParams a) {
    constexpr int L = HD / 8;
    const int gid = (blockIdx.x * 256 + threadIdx.x) / L, l = threadIdx.x % L;
    pdl_wait();
    const int t = gid / a.groups, part = gid - t * a.groups;
    if (t >= s.total_q) return;  // whole groups leave together
    const unsigned mask = (L == 16 ? 0xFFFFu : 0xFFu) << ((threadIdx.x & 31) / L * L);
    const int2 tok = p.tokens[t];
    const bool in_seq = tok.x >= 0;
    int pos = in_seq ? tok.y : 0;
    if (pos >= a.rope_rows) {
        if (l == 0) atomicOr(p.status, kPagedErrPosition);
        pos = 0;
    }
    const int half = a.rot >> 1;
    const bool turns = 8 * l < a.rot;
    const int at0 = turns && !a.pairs ? 4 * l : 8 * l, at1 = turns && !a.pairs ? 4 * l + half : 8 * l + 4;
    uint64_t cs[2], sn[2];  // cosines and sines of this lane's four pairs
    cs[0] = cs[1] = sn[0] = sn[1] = 0;
    if (turns) {
        const float4 *r = reinterpret_cast<const float4 *>(a.rope + (long long)pos * half + 4 * l);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4 w = __ldg(r + i);
            cs[i] = pack2(w.x, w.z);
            sn[i] = pack2(w.y, w.w);
        }
    }
    const int heads = s.nh + 2 * s.nkv;
    const int h0 = part * a.heads_per_group, h1 = min(heads, h0 + a.heads_per_group);
    int row0 = -1;  // the token's pool row for KV head 0
    if (in_seq && h1 > s.nh) row0 = paged_row(s, a.table, tok.x, 0, tok.y, p.status);
    const long long src = (long long)t * a.qkv_stride;
#pragma unroll 1
    for (int kind = 0; kind < 3; ++kind) {  // queries, keys, values
        const int from = kind == 0 ? 0 : s.nh + (kind - 1) * s.nkv;
        const int b0 = max(h0, from), b1 = min(h1, kind == 0 ? s.nh : from + s.nkv);
        if (b0 >= b1 || (kind > 0 && row0 < 0)) continue;
        const uint16_t *w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
        uint64_t g0[2], g1[2];
        if (w) load4x<true>(w, at0, g0), load4x<true>(w, at1, g1);
        uint16_t *out = kind == 0 ? a.q_out + (long long)t * s.nh * HD
                                  : (kind == 1 ? a.k : a.v) + (long long)row0 * HD;
        const long long step = kind == 0 ? HD : (long long)s.page_size * HD;
#pragma unroll 1
        for (int hb = b0; hb < b1; hb += kAppendAhead) {
            uint64_t x0[kAppendAhead][2], x1[kAppendAhead][2];
#pragma unroll
            for (int j = 0; j < kAppendAhead; ++j) {
                const long long at = src + (long long)min(hb + j, b1 - 1) * HD;
                load4x<BF16>(a.qkv, at + at0, x0[j]);
                load4x<BF16>(a.qkv, at + at1, x1[j]);
            }
#pragma unroll
            for (int j = 0; j < kAppendAhead; ++j) {
                if (hb + j >= b1) break;
                uint64_t(&u)[2] = x0[j], (&v)[2] = x1[j];
                if (w) {
                    uint64_t ss2 = mul2(u[0], u[0]);
                    ss2 = fma2(u[1], u[1], ss2);
                    ss2 = fma2(v[0], v[0], ss2);
                    ss2 = fma2(v[1], v[1], ss2);
                    float sa, sb;
                    unpack2(ss2, sa, sb);
                    float ss = sa + sb;
#pragma unroll
                    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
                    const float r = rsqrtf(ss * (1.0f / HD) + a.eps);
                    const uint64_t r2 = pack2(r, r);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        u[i] = mul2(mul2(u[i], r2), g0[i]);
                        v[i] = mul2(mul2(v[i], r2), g1[i]);
                    }
                }
                if (kind < 2 && turns) {
                    const uint64_t neg = pack2(-1.f, -1.f);
                    if (a.pairs) {  // (u0 u1) (u2 u3) | (v0 v1) (v2 v3): each is a pair
                        float p0[4], p1[4];
                        unpack2(u[0], p0[0], p1[0]);
                        unpack2(u[1], p0[1], p1[1]);
                        unpack2(v[0], p0[2], p1[2]);
                        unpack2(v[1], p0[3], p1[3]);
                        float y0[4], y1[4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint64_t f = pack2(p0[2 * i], p0[2 * i + 1]), q = pack2(p1[2 * i], p1[2 * i + 1]);
                            unpack2(fma2(f, cs[i], mul2(mul2(q, neg), sn[i])), y0[2 * i], y0[2 * i + 1]);
                            unpack2(fma2(q, cs[i], mul2(f, sn[i])), y1[2 * i], y1[2 * i + 1]);
                        }
                        u[0] = pack2(y0[0], y1[0]);
                        u[1] = pack2(y0[1], y1[1]);
                        v[0] = pack2(y0[2], y1[2]);
                        v[1] = pack2(y0[3], y1[3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {  // first half a cos - b sin, second half b cos + a sin
                            const uint64_t f = u[i], q = v[i];
                            u[i] = fma2(f, cs[i], mul2(mul2(q, neg), sn[i]));
                            v[i] = fma2(q, cs[i], mul2(f, sn[i]));
                        }
                    }
                }
                uint16_t *d = out + (hb + j - from) * step;
                const uint2 y0 = round4(u), y1 = round4(v);
                if (at1 == at0 + 4) {
                    *reinterpret_cast<uint4 *>(d + at0) = make_uint4(y0.x, y0.y, y1.x, y1.y);
                } else {
                    *reinterpret_cast<uint2 *>(d + at0) = y0;
                    *reinterpret_cast<uint2 *>(d + at1) = y1;
                }
            }
        }
    }
}

}  // namespace m1
