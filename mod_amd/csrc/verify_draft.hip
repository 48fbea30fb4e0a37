// Verification of drafted tokens (speculative sampling, tensor_rocm.h): which of
// a request's drafted tokens the target accepts, and the token that follows.
#include "pio_common.hpp"

#include <algorithm>
#include <climits>
#include <float.h>

namespace pio {

constexpr int VD_THREADS = 256;
constexpr int VD_WAVES = VD_THREADS / 64;

struct VdArgs {
    const void *target, *draft;
    int64_t target_stride, draft_stride;
    const int32_t* ids;
    const float *u, *u_next;
    const int32_t* row_start;
    int32_t *accepted, *tokens, *rejected;
    int n, rows, vocab;
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

// The weight of token v in a request's row: from the difference, or from the
// target alone.
template <typename PT>
__device__ __forceinline__ double vd_at(const VdArgs& a, const VdRow& r, int id, bool difference, int v) {
    const double p = (double)((const PT*)a.target)[r.row * a.target_stride + v];
    double q = 0.0;
    if (difference) q = a.draft ? (double)((const PT*)a.draft)[r.row * a.draft_stride + v] : v == id ? 1.0 : 0.0;
    return vd_weight(p, q);
}

__device__ __forceinline__ double vd_shfl_up(double x, int o) { return __shfl_up(x, o, 64); }

// One workgroup per request: it sums the weights, then walks them again for the
// place. Every thread has a run of consecutive tokens of each piece of the row.
template <typename PT>
__global__ __launch_bounds__(VD_THREADS) void vd_simple_kernel(VdArgs a) {
    __shared__ int sh, place, last;
    __shared__ double red[VD_WAVES];
    const int i = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const VdRow r = vd_accept<PT>(a, i, &sh);
    if (r.count == 0) {
        if (tid == 0) {
            a.accepted[i] = 0;
            if (a.rejected) a.rejected[i] = 0;
        }
        return;
    }
    const int id = r.rejects ? a.ids[r.row] : -1;
    bool difference = r.rejects;
    double total = 0.0;
    for (;;) {
        double sum = 0.0;
        for (int v = tid; v < a.vocab; v += VD_THREADS) sum += vd_at<PT>(a, r, id, difference, v);
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        __syncthreads();
        if (lane == 0) red[wv] = sum;
        __syncthreads();
        total = (red[0] + red[1]) + (red[2] + red[3]);
        if (total > 0.0 || !difference) break;
        difference = false;
    }
    const double bar = (double)a.u_next[i] * total;
    if (tid == 0) {
        place = INT_MAX;
        last = -1;
    }
    double before = 0.0;
    for (int v0 = 0; v0 < a.vocab; v0 += VD_THREADS) {
        const int v = v0 + tid;
        const double w = v < a.vocab ? vd_at<PT>(a, r, id, difference, v) : 0.0;
        double x = w;
        for (int o = 1; o < 64; o <<= 1) {
            const double y = vd_shfl_up(x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) red[wv] = x;
        __syncthreads();
        double base = before;
        for (int k = 0; k < wv; k++) base += red[k];
        if (w > 0.0) atomicMax(&last, v);
        if (w > 0.0 && base + x > bar) atomicMin(&place, v);
        before += (red[0] + red[1]) + (red[2] + red[3]);
        __syncthreads();
        if (place != INT_MAX) break;
    }
    __syncthreads();
    const int drafted = r.count - 1, next = place != INT_MAX ? place : last;
    for (int j = tid; j < r.count; j += VD_THREADS)
        a.tokens[r.first + j] = j < r.accepted ? a.ids[r.first + j] : j == r.accepted ? next : -1;
    if (tid == 0) {
        a.accepted[i] = r.accepted;
        if (a.rejected) a.rejected[i] = drafted - r.accepted;
    }
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
    if (dtype == PIO_F32) vd_simple_kernel<float><<<n, VD_THREADS, 0, st>>>(a);
    else vd_simple_kernel<_Float16><<<n, VD_THREADS, 0, st>>>(a);
    PIO_LAUNCHED();
    return PIO_OK;
}
