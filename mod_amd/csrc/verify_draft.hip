// Verification of drafted tokens (speculative sampling, tensor_rocm.h): which of
// a request's drafted tokens the target accepts, and the token that follows.
#include "pio_common.hpp"

#include <algorithm>
#include <climits>
#include <float.h>

namespace pio {

constexpr int VD_THREADS = 256;
constexpr int VD_WAVES = VD_THREADS / 64;
constexpr int VD_UNIT = 8 * VD_THREADS;      // tokens whose weights are summed together

struct VdArgs {
    const void *target, *draft;
    int64_t target_stride, draft_stride;
    const int32_t* ids;
    const float *u, *u_next;
    const int32_t* row_start;
    int32_t *accepted, *tokens, *rejected;
    int n, rows, vocab;
    int units, per_block;
    double* sums;          // [n][units]
};

// The weight that the next token is drawn with: p - q where that is positive.
__device__ __forceinline__ double vd_weight(double p, double q) {
    const double w = p - q;
    return w > 0.0 && w <= DBL_MAX ? w : 0.0;     // (false for NaN)
}

struct VdRow {
    int first, count;      // rows of the request (count 0: none)
    int accepted;
    int row;               // the row that the next token is drawn from
    bool rejects;          // from the difference
};

// One request's rows and how many of its drafted tokens hold; by a whole
// workgroup, `sh` its scratch.
template <typename PT>
__device__ __forceinline__ VdRow vd_accept(const VdArgs& a, int i, int* sh) {
    VdRow r;
    const int r0 = min(max(a.row_start[i], 0), a.rows), r1 = min(max(a.row_start[i + 1], r0), a.rows);
    r.first = r0;
    r.count = r1 - r0;
    const int drafted = max(r.count - 1, 0);
    int least = drafted;
    for (int j = threadIdx.x; j < drafted; j += VD_THREADS) {
        const int row = r0 + j, id = a.ids[row];
        bool ok = false;
        if (id >= 0 && id < a.vocab) {
            const double p = (double)((const PT*)a.target)[row * a.target_stride + id];
            const double q = a.draft ? (double)((const PT*)a.draft)[row * a.draft_stride + id] : 1.0;
            ok = (double)a.u[row] * q < p;
        }
        if (!ok) {
            least = j;
            break;
        }
    }
    if (threadIdx.x == 0) *sh = drafted;
    __syncthreads();
    if (least < drafted) atomicMin(sh, least);
    __syncthreads();
    r.accepted = *sh;
    r.row = r0 + r.accepted;
    r.rejects = r.accepted < drafted;
    return r;
}

// 8 consecutive tokens' probabilities from v of a row (0 behind its end). Rows may
// begin at any element, so the wide loads are unaligned ones.
template <typename PT>
__device__ __forceinline__ void vd_load8(const PT* row, int v, int vocab, double (&x)[8]) {
    typedef PT V __attribute__((ext_vector_type(16 / sizeof(PT)), aligned(sizeof(PT))));
    if (v + 8 <= vocab) {
        V r[8 * sizeof(PT) / 16];
#pragma unroll
        for (int i = 0; i < (int)(8 * sizeof(PT) / 16); i++) r[i] = *(const V*)(row + v + i * (16 / (int)sizeof(PT)));
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (double)r[e * sizeof(PT) / 16][e % (16 / sizeof(PT))];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = v + e < vocab ? (double)row[v + e] : 0.0;
    }
}

// The weights of 8 consecutive tokens of a request's row: from the difference, or
// from the target alone.
template <typename PT>
__device__ __forceinline__ void vd_weights(const VdArgs& a, const VdRow& r, int id, bool difference, int v, double (&w)[8]) {
    double p[8];
    vd_load8<PT>((const PT*)a.target + r.row * a.target_stride, v, a.vocab, p);
    if (difference && a.draft) {
        double q[8];
        vd_load8<PT>((const PT*)a.draft + r.row * a.draft_stride, v, a.vocab, q);
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = vd_weight(p[e], q[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = vd_weight(p[e], difference && v + e == id ? 1.0 : 0.0);
    }
}
__device__ __forceinline__ double vd_sum8(const double (&w)[8]) {
    return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
}
// Sum over the workgroup.
__device__ __forceinline__ double vd_block_sum(double x, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
// Sums of the threads before this one; `total` gets the sum of all.
__device__ __forceinline__ double vd_block_scan(double x, double* red, double& total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    double up = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(up, o, 64);
        if (lane >= o) up += y;
    }
    const double before = __shfl_up(up, 1, 64);
    __syncthreads();
    if (lane == 63) red[wv] = up;
    __syncthreads();
    double base = 0.0;
    for (int k = 0; k < wv; k++) base += red[k];
    total = (red[0] + red[1]) + (red[2] + red[3]);
    return lane ? base + before : base;
}

// First launch, (units of a row / per_block, requests): every workgroup finds its
// request's row and sums the weights of a few units of 2048 tokens; the first also
// writes what is accepted. Bytes bound it: 96 rows of 151,936, fp32, target and draft,
// 21 us, 5.6 TB/s. Weights and their sums in 64 bits: the place of u_next in a sum of
// 151,936 would move by tokens with 32.
template <typename PT>
__global__ __launch_bounds__(VD_THREADS) void vd_sum_kernel(VdArgs a) {
    __shared__ int sh;
    __shared__ double red[VD_WAVES];
    const int i = blockIdx.y, tid = threadIdx.x;
    const VdRow r = vd_accept<PT>(a, i, &sh);
    if (blockIdx.x == 0) {
        if (tid == 0) {
            a.accepted[i] = r.accepted;
            if (a.rejected) a.rejected[i] = max(r.count - 1, 0) - r.accepted;
        }
        for (int j = tid; j < r.count; j += VD_THREADS)
            if (j != r.accepted) a.tokens[r.first + j] = j < r.accepted ? a.ids[r.first + j] : -1;
    }
    if (r.count == 0) return;
    const int id = r.rejects ? a.ids[r.row] : -1;
    const int u1 = min(a.units, (int)(blockIdx.x + 1) * a.per_block);
    for (int u = blockIdx.x * a.per_block; u < u1; u++) {
        double w[8];
        vd_weights<PT>(a, r, id, r.rejects, u * VD_UNIT + 8 * tid, w);
        const double s = vd_block_sum(vd_sum8(w), red);
        if (tid == 0) a.sums[(int64_t)i * a.units + u] = s;
    }
}

// Of the workgroup's threads in order: the first one's `first` that is not INT_MAX (its
// `at` in *before), and the last one's `some` that is not -1.
struct VdPlace {
    int first, last;
    double before;
};
__device__ __forceinline__ VdPlace vd_place(int first, double at, int some, VdPlace* sh) {
    const int wv = threadIdx.x >> 6;
    const uint64_t f = __ballot(first != INT_MAX), l = __ballot(some >= 0);
    VdPlace p;
    p.first = f ? __shfl(first, __ffsll((unsigned long long)f) - 1, 64) : INT_MAX;
    p.before = f ? __shfl(at, __ffsll((unsigned long long)f) - 1, 64) : 0.0;
    p.last = l ? __shfl(some, 63 - __clzll((long long)l), 64) : -1;
    if ((threadIdx.x & 63) == 0) sh[wv] = p;
    __syncthreads();
    p = sh[0];
    for (int k = 1; k < VD_WAVES; k++) {
        if (p.first == INT_MAX) {
            p.first = sh[k].first;
            p.before = sh[k].before;
        }
        p.last = max(p.last, sh[k].last);
    }
    return p;
}

// Second launch, one workgroup per request: the unit whose weights reach u_next *
// total, and the token in it. A chain of waits: what a request is and its sums, the
// unit's weights; each thread has a few units in order, so that one scan gives both
// the total and where it is reached. 3.8 us for one request, 4.4 for 96.
template <typename PT>
__global__ __launch_bounds__(VD_THREADS) void vd_pick_kernel(VdArgs a) {
    __shared__ VdPlace sh[2][VD_WAVES];
    __shared__ double red[VD_WAVES];
    const int i = blockIdx.x, tid = threadIdx.x;
    const int per = (a.units + VD_THREADS - 1) / VD_THREADS, first = min(tid * per, a.units), end = min(first + per, a.units);
    double* sums = a.sums + (int64_t)i * a.units;
    VdRow r;
    // (a request without rows has no sums: they are read all the same, with the rest)
    const int s0 = a.row_start[i], s1 = a.row_start[i + 1];
    r.accepted = a.accepted[i];
    const double drawn = (double)a.u_next[i];
    double mine = 0.0;
    for (int u = first; u < end; u++) mine += sums[u];
    const int r0 = min(max(s0, 0), a.rows), r1 = min(max(s1, r0), a.rows);
    if (r1 <= r0) return;
    r.first = r0;
    r.count = r1 - r0;
    r.row = r0 + r.accepted;
    r.rejects = r.accepted < r.count - 1;
    const int id = r.rejects ? a.ids[r.row] : -1;
    bool difference = r.rejects;
    double total, base = vd_block_scan(mine, red, total);
    if (!(total > 0.0) && difference) {
        // nothing is left of the target above the draft: the target's own weights
        difference = false;
        for (int u = 0; u < a.units; u++) {
            double w[8];
            vd_weights<PT>(a, r, id, false, u * VD_UNIT + 8 * tid, w);
            const double s = vd_block_sum(vd_sum8(w), red);
            if (tid == 0) sums[u] = s;
        }
        __syncthreads();
        mine = 0.0;
        for (int u = first; u < end; u++) mine += sums[u];
        base = vd_block_scan(mine, red, total);
    }
    const double bar = drawn * total;
    int some = -1, found = INT_MAX;
    double at = base, before = 0.0;
    for (int u = first; u < end; u++) {
        const double s = per == 1 ? mine : sums[u];
        if (s > 0.0) {
            some = u;
            if (found == INT_MAX && at + s > bar) {
                found = u;
                before = at;
            }
        }
        at += s;
    }
    const VdPlace unit = vd_place(found, before, some, sh[0]);
    // rounding (or u_next = 1) left none: the last one with a weight
    const bool over = unit.first != INT_MAX;
    const int u = over ? unit.first : unit.last;
    int token = -1;
    if (u >= 0) {
        double w[8], all;
        const int v = u * VD_UNIT + 8 * tid;
        vd_weights<PT>(a, r, id, difference, v, w);
        double sum = (over ? unit.before : 0.0) + vd_block_scan(vd_sum8(w), red, all);
        int some = -1, found = INT_MAX;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            sum += w[e];
            if (w[e] > 0.0) {
                some = v + e;
                if (over && sum > bar) found = min(found, v + e);
            }
        }
        const VdPlace place = vd_place(found, 0.0, some, sh[1]);
        token = place.first != INT_MAX ? place.first : place.last;
    }
    if (tid == 0) a.tokens[r.row] = token;
}

}  // namespace pio

using namespace pio;

PIO_EXPORT int pio_verify_draft(const void* target, int64_t target_stride, const void* draft, int64_t draft_stride,
                                int dtype, const int32_t* ids, const float* u, const float* u_next,
                                const int32_t* row_start, int n, int rows, int vocab, int32_t* accepted,
                                int32_t* tokens, int32_t* rejected, void* stream) {
    const char* nm = "pio_verify_draft";
    PIO_REQUIRE(dtype == PIO_F32 || dtype == PIO_F16, "%s: dtype %d (fp32 or fp16)", nm, dtype);
    PIO_REQUIRE(n >= 0 && rows >= 0 && vocab > 0, "%s: %d requests, %d rows, vocabulary of %d", nm, n, rows, vocab);
    PIO_REQUIRE(vocab <= 1 << 30, "%s: a vocabulary of over 2^30", nm);
    if (n == 0) return PIO_OK;
    PIO_REQUIRE(row_start && accepted && u_next, "%s: null pointer", nm);
    PIO_REQUIRE(rows == 0 || (target && ids && u && tokens), "%s: null pointer", nm);
    if (target_stride == 0) target_stride = vocab;
    if (draft_stride == 0) draft_stride = vocab;
    PIO_REQUIRE(target_stride >= vocab && draft_stride >= vocab, "%s: strides %lld, %lld for rows of %d", nm,
                (long long)target_stride, (long long)draft_stride, vocab);
    const size_t esz = dtype_bytes(dtype);
    PIO_REQUIRE((uintptr_t)target % esz == 0 && (uintptr_t)draft % esz == 0, "%s: unaligned probabilities", nm);
    for (const void* p : {(const void*)ids, (const void*)u, (const void*)u_next, (const void*)row_start,
                          (const void*)accepted, (const void*)tokens, (const void*)rejected})
        PIO_REQUIRE(((uintptr_t)p & 3u) == 0, "%s: array not 4-byte aligned", nm);
    VdArgs a{};
    a.target = target;
    a.draft = draft;
    a.target_stride = target_stride;
    a.draft_stride = draft_stride;
    a.ids = ids;
    a.u = u;
    a.u_next = u_next;
    a.row_start = row_start;
    a.accepted = accepted;
    a.tokens = tokens;
    a.rejected = rejected;
    a.n = n;
    a.rows = rows;
    a.vocab = vocab;
    hipStream_t st = pick_stream(stream);
    a.units = ceil_div(vocab, VD_UNIT);
    Scratch ws;
    PIO_TRY(ws.get((size_t)n * a.units * sizeof(double), st));
    a.sums = (double*)ws.ptr;
    // a few thousand workgroups are enough for the device, and each has its row to find first
    a.per_block = (int)std::max<int64_t>(1, (int64_t)n * a.units / 2048);
    for (int i0 = 0; i0 < n; i0 += 65535) {        // the grid's second dimension
        VdArgs b = a;
        b.n = std::min(n - i0, 65535);
        b.u_next += i0;
        b.row_start += i0;
        b.accepted += i0;
        if (b.rejected) b.rejected += i0;
        b.sums += (int64_t)i0 * a.units;
        const dim3 grid(ceil_div(a.units, a.per_block), b.n);
        if (dtype == PIO_F32) {
            vd_sum_kernel<float><<<grid, VD_THREADS, 0, st>>>(b);
            vd_pick_kernel<float><<<b.n, VD_THREADS, 0, st>>>(b);
        } else {
            vd_sum_kernel<_Float16><<<grid, VD_THREADS, 0, st>>>(b);
            vd_pick_kernel<_Float16><<<b.n, VD_THREADS, 0, st>>>(b);
        }
        PIO_LAUNCHED();
    }
    return PIO_OK;
}
