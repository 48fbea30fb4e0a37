// What the attention kernels over the paged cache share (kv_attention.hip: fp16 and
// fp32 caches, kv_attention4.hip: 4 bits): the call's arguments, the items that a batch
// is cut into, and the join of a column's items.
#pragma once

#include "kv_pages.hpp"

#include <climits>
#include <float.h>

namespace pio {

constexpr int KA_THREADS = 256;

struct KaArgs {
    pio_kv_cache c;
    const int32_t *seq, *row_start;
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int layer, n, shared, rows, H, G;
    uint32_t g_magic;        // floor(2^32 / G) + 1, 0 for 1
    float scale;
    bool q16;
    // items of the matrix core kernels
    int pre_items, pre_tiles, pre_splits, pre_keys;   // workgroups; column tiles; runs of keys, keys of each
    int tail_tiles, tail_runs, max_runs;              // column tiles; the most runs beside one for each request, and of one
    float fixed;                                      // rounds of keys that an item costs besides its own
    int slots;                                        // items that the device holds at once
    float pre_work;                                   // rounds of keys that the prefix's items cost
    int tail_items;                                   // workgroups: (run, column tile, kv head), as many as there may be
    bool direct;                                      // one item per column: it writes out itself
    float* part_o;                                    // [pre_splits + max_runs][rows * H][D]
    float* part_ml;                                   // [..][rows * H][2]
    int* part_n;                                      // [rows]: tail runs, 0 for a row that is written already
};

// Column / G.
__device__ __forceinline__ int ka_div(const KaArgs& a, int col) {
    const int r = a.g_magic ? (int)__umulhi((uint32_t)col, a.g_magic) : col;     // at most one too large
    return r - (r * a.G > col);
}

// Rows of request i, kept inside q whatever row_start holds.
__device__ __forceinline__ void ka_rows(const KaArgs& a, int i, int& r0, int& r1) {
    r0 = max(a.row_start[i], 0);
    r1 = min(a.row_start[i + 1], a.rows);
}

__device__ __forceinline__ float ka_q(const KaArgs& a, int64_t at) {
    return a.q16 ? (float)((const _Float16*)a.q)[at] : ((const float*)a.q)[at];
}

// The attention over a cache of 4 bits (kv_attention4.hip).
int ka4_attention(KaArgs& a, int max_rows, hipStream_t st);

typedef float ka_v16 __attribute__((ext_vector_type(16)));
typedef float ka_f4 __attribute__((ext_vector_type(4)));
typedef float ka_f2 __attribute__((ext_vector_type(2)));
typedef _Float16 ka_h8 __attribute__((ext_vector_type(8)));

constexpr float KA_LOG2E = 1.44269504088896340736f;
// A column's reference (the exponent that its weights are relative to) follows its
// maximum only when that has grown by KA_SLACK: rescaling O^T for every new maximum of 32
// columns cost as much as a tile's exponentials. fp16 weights are held times 2^10, so that they
// stay below 2^15, and are normal numbers down to 2^-24 of the reference.
constexpr float KA_LIFT = 10.f, KA_SLACK = 5.f;
// Least maximum of a column that sees a key; one that sees none keeps -FLT_MAX.
constexpr float KA_SEEN = -3.4e38f;

// Maximum over the parts of a column.
template <int COLS>
__device__ __forceinline__ float ka_max(float v) {
    // (the halves of the wave swapped, then neighbouring rows of 16 lanes: no trip through LDS)
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
    if constexpr (COLS == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}

// ---- what an item is: columns of a batch or a request, a run of keys of one kv head
struct KaItem {
    const int32_t* table;    // the table row that the keys are read through
    int g, k0, k1;           // kv head, keys
    int row0, ncols;         // columns: (row0 + c / G, head g * G + c % G), c < ncols
    int first_limit;         // tails: keys that row0 sees, each row behind it one more
    int slot;                // of the workspace
    bool bad;                // no such sequence: the rows become NaN
    bool direct;             // the columns' only item: it writes the result
};

// 4 dimensions from d of column (row, head): an item's part of it, or the result.
__device__ __forceinline__ void ka_out(const KaArgs& a, int D, int row, int head, int d, ka_f4 v) {
    const int64_t at = row * a.out_stride + (int64_t)head * D + d;
    if (a.q16) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        h4 y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = (_Float16)v[e];
        *(h4*)((_Float16*)a.out + at) = y;
    } else {
        *(ka_f4*)((float*)a.out + at) = v;
    }
}
__device__ __forceinline__ void ka_emit(const KaArgs& a, int D, const KaItem& it, int col, int d, ka_f4 v, float m, float l) {
    const int r = ka_div(a, col), row = it.row0 + r, head = it.g * a.G + col - r * a.G;
    if (it.direct) {
        v = v / l;
        if (m == -FLT_MAX && l == 0.f) v = ka_f4{0.f, 0.f, 0.f, 0.f};     // sees no key
        ka_out(a, D, row, head, d, v);
        return;
    }
    const int64_t at = ((int64_t)it.slot * a.rows + row) * a.H + head;
    *(ka_f4*)(a.part_o + at * D + d) = v;
    if (d == 0) *(ka_f2*)(a.part_ml + 2 * at) = ka_f2{m, l};
}

constexpr int KA_ROUND = 128;          // keys that runs are multiples of
// Rounds of keys for each of the runs that `rounds` are cut into, if every run is an item in
// each of `units` places and all else costs `work`: the longest item, fixed + r, takes as
// long as the device's share of all work.
__device__ __forceinline__ float ka_cut(float rounds, float units, float work, float slots, float fixed) {
    const float d = (work + units * rounds) / slots - fixed;
    return 0.5f * (d + sqrtf(d * d + 4.f * fixed * units / slots * rounds));
}

// Sum over the workgroup's threads before this one, and over all.
__device__ __forceinline__ int ka_scan(int v, int* red, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) red[w] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < waves; i++) {
        if (i < w) before += red[i];
        total += red[i];
    }
    return before + x - v;
}

// Which tail items there are: the tails are cut into runs of about equal length,
// however uneven they are (every request with rows has at least one), and a run has the
// column tiles of its request, at most tail_tiles. By the whole workgroup; it gets the
// request, run and geometry of item number `unit` over all runs' tiles (request -1 if
// there are fewer).
struct KaRun {
    int i, z, runs, per;     // request, run of it, runs of it, rounds of KA_ROUND keys of a run
    int ct, tiles;           // column tile, tiles of the request
    int r0, r1, s, L;        // rows, sequence, its length (-1: none such)
};
__device__ __forceinline__ void ka_runs(const KaArgs& a, int unit, KaRun& found, int* red, int cols) {
    const int tid = threadIdx.x, threads = blockDim.x;
    KaRun r{};
    auto rounds = [&](int i) {
        r.i = i;
        if (i >= a.n) return 0;
        ka_rows(a, i, r.r0, r.r1);
        r.s = a.seq[i];
        r.L = kv_seq_len(a.c, r.s);
        if (r.r1 <= r.r0) return 0;
        return r.L <= a.shared ? 1 : (r.L - a.shared + KA_ROUND - 1) / KA_ROUND;
    };
    if (tid == 0) found.i = -1;
    int n = rounds(tid), total, sum;
    ka_scan(n, red, total);
    for (int i0 = threads; i0 < a.n; i0 += threads) {
        ka_scan(rounds(i0 + tid), red, sum);
        total += min(sum, INT_MAX - total);
    }
    const float units = a.c.n_kv_heads * a.tail_tiles;
    // runs that balance the items, or of as many rounds as an item costs besides: the last items to start should be short ones
    // (and at most tail_runs more runs than requests)
    const float cut = fmaxf(fmaxf(1.f, (float)total / a.tail_runs),
                            fminf(a.fixed, ka_cut(total, units, a.pre_work + a.n * units * a.fixed, a.slots, a.fixed)));
    int before = 0;
    for (int i0 = 0; i0 < a.n; i0 += threads) {
        if (a.n > threads) n = rounds(i0 + tid);
        r.per = r.runs = r.tiles = 0;
        if (n > 0) {
            r.tiles = min(a.tail_tiles, ((r.r1 - r.r0) * a.G + cols - 1) / cols);
            r.runs = min(max(1, (int)(n / cut + 0.5f)), a.max_runs);
            r.per = (n + r.runs - 1) / r.runs;
            r.runs = (n + r.per - 1) / r.per;
        }
        const int at = before + ka_scan(r.runs * r.tiles, red, sum);
        before += sum;
        if (unit >= at && unit < at + r.runs * r.tiles) {
            r.z = (unit - at) / r.tiles;
            r.ct = unit - at - r.z * r.tiles;
            found = r;
        }
    }
    __syncthreads();
}

// Keys that each of N rows of the batch from `first` sees, -1 for a row that no
// request has; by the whole workgroup.
__device__ __forceinline__ void ka_limits(const KaArgs& a, int first, int* limit, int N) {
    for (int i = threadIdx.x; i < N; i += blockDim.x) limit[i] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
        const int s = a.seq[i];            // (with its rows, not behind them)
        int r0, r1;
        ka_rows(a, i, r0, r1);
        const int lo = max(r0, first), hi = min(r1, first + N);
        if (lo >= hi) continue;
        const int L = kv_seq_len(a.c, s);
        if (L < 0) continue;
        for (int row = lo; row < hi; row++) limit[row - first] = max(L - (r1 - row) + 1, 0);
    }
    __syncthreads();
}

__device__ __forceinline__ int ka_wave_min(int v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return v;
}

// Keys of its run that a column with row r (of the item) sees; limits: of a prefix's rows from `first`.
__device__ __forceinline__ int ka_limit(const KaItem& it, const int* limits, int first, int r) {
    const int n = limits ? limits[r - first] : it.first_limit + r;
    return limits && n < 0 ? it.k1 : min(n, it.k1);     // (a row that no request has: anything)
}

// The prefix item of a workgroup: false for one beyond them.
__device__ __forceinline__ bool ka_prefix(const KaArgs& a, KaItem& it, int& ct) {
    // the column tiles of a (kv head, run of keys) on one XCD, next to each other: they read the same K and V
    const int x = blockIdx.x & 7, y = blockIdx.x >> 3, unit = (y / a.pre_tiles) * 8 + x;
    ct = y % a.pre_tiles;
    if (unit >= a.c.n_kv_heads * a.pre_splits) return false;
    it.slot = unit / a.c.n_kv_heads;
    it.g = unit - it.slot * a.c.n_kv_heads;
    it.k0 = it.slot * a.pre_keys;
    it.k1 = min(it.k0 + a.pre_keys, a.shared);
    it.row0 = 0;
    it.ncols = a.rows * a.G;
    it.first_limit = 1;
    it.direct = false;
    const int s = a.seq[0];
    it.bad = s < 0 || s >= a.c.max_seqs;
    it.table = a.c.table + (int64_t)(it.bad ? 0 : s) * a.c.max_pages;
    return true;
}
// A run of a request's tail; false: there is none.
__device__ __forceinline__ bool ka_tail(const KaArgs& a, KaItem& it, const KaRun& r, int g) {
    it = KaItem{};
    if (r.i < 0) return false;
    const int keys = r.per * KA_ROUND;
    it.g = g;
    it.k0 = a.shared + r.z * keys;
    it.k1 = max(it.k0, min(it.k0 + keys, r.L));
    it.row0 = r.r0;
    it.ncols = (r.r1 - r.r0) * a.G;
    it.first_limit = r.L - (r.r1 - r.r0) + 1;
    it.slot = a.pre_splits + r.z;
    it.bad = r.L < 0;
    it.direct = r.runs == 1 && a.pre_splits == 0;
    it.table = a.c.table + (int64_t)(it.bad ? 0 : r.s) * a.c.max_pages;
    return true;
}

// A column's items joined: D / 4 lanes have its dimensions, Z groups of them take
// every Z-th item, all loads of a few in flight together. Z = 8: few columns, where
// latency counts (1,024 columns of 5 items 4 us); Z = 1: 8 (16) columns to a workgroup
// (6,752 of 4 items 5.7 us, 3.5 TB/s).
template <int D, int Z>
__global__ __launch_bounds__(256) void ka_merge_kernel(KaArgs a) {
    constexpr int TPC = D / 4, GRP = 256 / TPC, COLS = GRP / Z;
    __shared__ __attribute__((aligned(16))) float so[GRP][D];
    __shared__ float sml[GRP][2];
    const int tid = threadIdx.x, grp = tid / TPC, d = (tid % TPC) * 4, zg = grp % Z;
    // (rows * H < 2^26) Which parts a column has is known later than the first ones' loads are under way: those are
    // read whatever they hold, inside the workspace.
    const uint32_t col = blockIdx.x * COLS + grp / Z;
    const int64_t step = (int64_t)a.rows * a.H, at = col < step ? col : 0;
    const int row = (int)((uint32_t)at / (uint32_t)a.H), head = (int)at - row * a.H, most = a.pre_splits + a.max_runs;
    auto part = [&](int z) { return at + min(z, most - 1) * step; };
    ka_f2 ml = *(const ka_f2*)(a.part_ml + 2 * part(zg));
    ka_f4 o = *(const ka_f4*)(a.part_o + part(zg) * D + d);
    const int runs_of = a.part_n[row];
    const bool has = col < step && row >= a.row_start[0] && row < min(a.row_start[a.n], a.rows);
    // (0: the row's only item wrote it)
    const int runs = has ? min(max(runs_of, 0), a.max_runs) : 0, parts = runs ? a.pre_splits + runs : 0;
    float m = -FLT_MAX, l = 0.f;
    ka_f4 v = {0.f, 0.f, 0.f, 0.f};
    auto add = [&]() {
        const float nm = fmaxf(m, ml[0]), f = __builtin_amdgcn_exp2f(m - nm), fz = __builtin_amdgcn_exp2f(ml[0] - nm);
        l = l * f + ml[1] * fz;
        v = v * f + o * fz;
        m = nm;
    };
    if (zg < parts) add();
#pragma unroll 4
    for (int z = zg + Z; z < parts; z += Z) {
        ml = *(const ka_f2*)(a.part_ml + 2 * part(z));
        o = *(const ka_f4*)(a.part_o + part(z) * D + d);
        add();
    }
    if constexpr (Z > 1) {
        *(ka_f4*)&so[grp][d] = v;
        if (d == 0) {
            sml[grp][0] = m;
            sml[grp][1] = l;
        }
        __syncthreads();
        if (zg) return;
#pragma unroll
        for (int z = 1; z < Z; z++) m = fmaxf(m, sml[grp + z][0]);
        l = 0.f;
        v = ka_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int z = 0; z < Z; z++) {
            const float f = __builtin_amdgcn_exp2f(sml[grp + z][0] - m);
            l += sml[grp + z][1] * f;
            v += *(const ka_f4*)&so[grp + z][d] * f;
        }
    }
    if (parts == 0) return;
    v = v / l;
    if (l == 0.f && m == -FLT_MAX) v = ka_f4{0.f, 0.f, 0.f, 0.f};     // sees no key
    ka_out(a, D, row, head, d, v);
}

}  // namespace pio
