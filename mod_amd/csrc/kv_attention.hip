// Causal attention of a batch over the paged cache (kv_pages.hip):
//   out[r, h] = sum_t softmax_t(q[r, h] . k[t] * scale) v[t].
#include "kv_pages.hpp"

#include <algorithm>
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
    float scale;
    bool q16;
};

__device__ __forceinline__ float ka_q(const KaArgs& a, int64_t at) {
    return a.q16 ? (float)((const _Float16*)a.q)[at] : ((const float*)a.q)[at];
}

// One workgroup per (row, head): 256 keys at a time, a thread for each key's
// score, then a thread for each dimension of the weighted sum.
template <typename KT>
__global__ __launch_bounds__(KA_THREADS) void ka_simple_kernel(KaArgs a) {
    __shared__ float qs[256], ps[KA_THREADS], red[4];
    __shared__ const KT* vrow[KA_THREADS];
    __shared__ int req, count0;
    const pio_kv_cache& c = a.c;
    const int tid = threadIdx.x, row = blockIdx.x / a.H, h = blockIdx.x - row * a.H, g = h / a.G, D = c.head_dim;
    const int lg = kv_log2(c.page_size);
    if (tid == 0) req = -1;
    __syncthreads();
    for (int i = tid; i < a.n; i += KA_THREADS) {
        const int r0 = a.row_start[i], r1 = a.row_start[i + 1];
        if (row >= r0 && row < r1) {
            req = i;
            count0 = r1 - row;
        }
    }
    for (int d = tid; d < D; d += KA_THREADS) qs[d] = ka_q(a, row * a.q_stride + h * D + d);
    __syncthreads();
    if (req < 0) return;
    const int s = a.seq[req], s0 = a.seq[0], L = kv_seq_len(c, s);
    const int limit = L - count0 + 1;
    int bad = L < 0 || kv_seq_len(c, s0) < 0;     // the same in every thread, always
    const int64_t head = (int64_t)c.page_size * D, page_e = head * c.n_kv_heads;
    const KT* kb = (const KT*)c.kv + (int64_t)(2 * a.layer) * c.n_pages * page_e + g * head;
    const KT* vb = kb + (int64_t)c.n_pages * page_e;
    float m = -FLT_MAX, l = 0.f, o = 0.f;
    for (int t0 = 0; t0 < limit && !bad; t0 += KA_THREADS) {
        const int t = t0 + tid;
        float sc = -INFINITY;
        const KT* vr = nullptr;
        int wrong = 0;
        if (t < limit) {
            const int page = c.table[(int64_t)(t < a.shared ? s0 : s) * c.max_pages + (t >> lg)];
            if (page < 0 || page >= c.n_pages) {
                wrong = 1;
            } else {
                const int64_t at = page * page_e + (int64_t)(t & (c.page_size - 1)) * D;
                float d = 0.f;
                for (int e = 0; e < D; e += 8) {
                    float x[8];
                    load8<KT>(kb + at + e, x);
#pragma unroll
                    for (int j = 0; j < 8; j++) d = fmaf(x[j], qs[e + j], d);
                }
                sc = d * a.scale;
                vr = vb + at;
            }
        }
        vrow[tid] = vr;
        float mt = wave_max(sc);
        if ((tid & 63) == 0) red[tid >> 6] = mt;
        __syncthreads();
        mt = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        ps[tid] = vr ? expf(sc - mt) : 0.f;
        const float corr = expf(m - mt);
        m = mt;
        o *= corr;
        l *= corr;
        __syncthreads();
        const int keys = min(KA_THREADS, limit - t0);
        for (int u = 0; u < keys; u++) {
            l += ps[u];
            if (tid < D && vrow[u]) o = fmaf(ps[u], (float)vrow[u][tid], o);
        }
        bad = __syncthreads_or(wrong);
    }
    if (tid < D) {
        const float r = bad ? NAN : limit <= 0 ? 0.f : o / l;
        const int64_t at = row * a.out_stride + h * D + tid;
        if (a.q16) ((_Float16*)a.out)[at] = (_Float16)r;
        else ((float*)a.out)[at] = r;
    }
    if (bad && tid == 0) atomicOr(c.work, KV_BAD);
}

}  // namespace pio

using namespace pio;

PIO_EXPORT int pio_kv_attention(const pio_kv_cache* c, int layer, const int32_t* seq, const int32_t* row_start, int n,
                                int shared, const void* q, void* out, int dtype, int rows, int n_heads,
                                int64_t q_stride, int64_t out_stride, int max_rows, float scale, void* stream) {
    const char* nm = "pio_kv_attention";
    PIO_TRY(kv_check(c, nm));
    PIO_REQUIRE(layer >= 0 && layer < c->n_layers, "%s: layer %d of %d", nm, layer, c->n_layers);
    PIO_REQUIRE(dtype == PIO_F32 || dtype == PIO_F16, "%s: dtype %d (fp32 or fp16)", nm, dtype);
    PIO_REQUIRE(n >= 0 && rows >= 0, "%s: %d requests, %d rows", nm, n, rows);
    PIO_REQUIRE(shared >= 0 && shared <= c->max_pages * c->page_size, "%s: %d shared tokens of a table row's %d", nm,
                shared, c->max_pages * c->page_size);
    PIO_REQUIRE(n_heads > 0 && n_heads % c->n_kv_heads == 0, "%s: %d heads over %d", nm, n_heads, c->n_kv_heads);
    PIO_REQUIRE(max_rows >= 1, "%s: max_rows %d", nm, max_rows);
    if (n == 0 || rows == 0) return PIO_OK;
    PIO_REQUIRE(seq && row_start && q && out, "%s: null pointer", nm);
    PIO_REQUIRE(((uintptr_t)seq & 3u) == 0 && ((uintptr_t)row_start & 3u) == 0, "%s: request list not 4-byte aligned",
                nm);
    const int64_t width = (int64_t)n_heads * c->head_dim;
    if (q_stride == 0) q_stride = width;
    if (out_stride == 0) out_stride = width;
    PIO_REQUIRE(q_stride % 8 == 0 && out_stride % 8 == 0 && q_stride >= width && out_stride >= width,
                "%s: strides %lld, %lld (multiples of 8, rows of %lld)", nm, (long long)q_stride, (long long)out_stride,
                (long long)width);
    PIO_REQUIRE(aligned16(q) && aligned16(out), "%s: q or out not 16-byte aligned", nm);
    PIO_REQUIRE((int64_t)rows * n_heads <= INT_MAX, "%s: too many rows", nm);
    KaArgs a{};
    a.c = *c;
    a.seq = seq;
    a.row_start = row_start;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.layer = layer;
    a.n = n;
    a.shared = shared;
    a.rows = rows;
    a.H = n_heads;
    a.G = n_heads / c->n_kv_heads;
    a.scale = scale;
    a.q16 = dtype == PIO_F16;
    hipStream_t st = pick_stream(stream);
    if (c->kv_dtype == PIO_F32) ka_simple_kernel<float><<<rows * n_heads, KA_THREADS, 0, st>>>(a);
    else ka_simple_kernel<_Float16><<<rows * n_heads, KA_THREADS, 0, st>>>(a);
    PIO_LAUNCHED();
    return PIO_OK;
}
