// Causal attention of a batch over a paged cache of 4 bits (tensor_rocm.h: its layout):
//   out[r, h] = sum_t softmax_t(q[r, h] . k[t] * scale) v[t].
#include "kv_attention.hpp"

#include <cmath>

namespace pio {

// Head dimensions other than 64 and 128. One workgroup per (row, head): 256 keys at a time, a thread
// for each key's score, then a thread for each dimension of the weighted sum.
constexpr int KA4_DEEP = 8;
__global__ __launch_bounds__(KA_THREADS) void ka4_simple_kernel(KaArgs a) {
    __shared__ float qs[256], ps[KA_THREADS], red[4];
    __shared__ int64_t vblock[KA_THREADS];     // where the block of a key's value is, -1: nowhere
    __shared__ int vrow[KA_THREADS];           // the key's row in it
    __shared__ int req, count0;
    const pio_kv_cache& c = a.c;
    const int tid = threadIdx.x, row = blockIdx.x / a.H, h = blockIdx.x - row * a.H, g = h / a.G, D = c.head_dim;
    const int lg = kv_log2(c.page_size), P = c.page_size;
    if (tid == 0) req = -1;
    __syncthreads();
    for (int i = tid; i < a.n; i += KA_THREADS) {
        int r0, r1;
        ka_rows(a, i, r0, r1);
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
    // the same in every thread, always; of seq[0] only the table row counts, and only where tokens are shared
    int bad = L < 0 || (a.shared > 0 && (s0 < 0 || s0 >= c.max_seqs));
    const int64_t head = (int64_t)P * kv_token_bytes(c), page_b = head * c.n_kv_heads;
    const char* kb = (const char*)c.kv + (int64_t)(2 * a.layer) * c.n_pages * page_b + g * head;
    const char* vb = kb + (int64_t)c.n_pages * page_b;
    float m = -FLT_MAX, l = 0.f, o = 0.f;
    for (int t0 = 0; t0 < limit && !bad; t0 += KA_THREADS) {
        const int t = t0 + tid;
        float sc = -INFINITY;
        int64_t block = -1;
        int wrong = 0;
        if (t < limit) {
            const int page = c.table[(int64_t)(t < a.shared ? s0 : s) * c.max_pages + (t >> lg)];
            if (page < 0 || page >= c.n_pages) {
                wrong = 1;
            } else {
                block = page * page_b;
                const int r = t & (P - 1);
                const char* codes = kb + block + r * (D / 2);
                const uint8_t* scales = (const uint8_t*)kb + block + P * (D / 2) + r;
                float d = 0.f;
                for (int b = 0; b < D / 32; b++) {
                    const uint4 w = *(const uint4*)(codes + 16 * b);
                    const int scale = scales[b * P];
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        kv_mx4_widen((&w.x)[i], scale, x);
#pragma unroll
                        for (int j = 0; j < 8; j++) d = fmaf(x[j], qs[32 * b + 8 * i + j], d);
                    }
                }
                sc = d * a.scale;
            }
        }
        vblock[tid] = block;
        vrow[tid] = t & (P - 1);
        float mt = wave_max(sc);
        if ((tid & 63) == 0) red[tid >> 6] = mt;
        __syncthreads();
        mt = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        ps[tid] = block >= 0 ? expf(sc - mt) : 0.f;
        const float corr = expf(m - mt);
        m = mt;
        o *= corr;
        l *= corr;
        __syncthreads();
        const int keys = min(KA_THREADS, limit - t0), d = min(tid, D - 1);
        for (int u0 = 0; u0 < keys; u0 += KA4_DEEP) {      // (a key behind the last one has no block and weight 0)
            int code[KA4_DEEP], scale[KA4_DEEP];
#pragma unroll
            for (int i = 0; i < KA4_DEEP; i++) {
                const uint8_t* from = (const uint8_t*)vb + max(vblock[u0 + i], (int64_t)0);
                code[i] = from[vrow[u0 + i] * (D / 2) + d / 2];
                scale[i] = from[P * (D / 2 + d / 32) + vrow[u0 + i]];
            }
#pragma unroll
            for (int i = 0; i < KA4_DEEP; i++) {
                typedef float f2 __attribute__((ext_vector_type(2)));
                const f2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)code[i],
                                                                      __uint_as_float((uint32_t)scale[i] << 23), 0);
                l += ps[u0 + i];
                o = fmaf(ps[u0 + i], vblock[u0 + i] >= 0 ? x[d & 1] : 0.f, o);
            }
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

int ka4_attention(KaArgs& a, int max_rows, hipStream_t st) {
    PIO_REQUIRE((int64_t)a.rows * a.H < 1 << 24, "pio_kv_attention: too many rows");
    ka4_simple_kernel<<<a.rows * a.H, KA_THREADS, 0, st>>>(a);
    PIO_LAUNCHED();
    return PIO_OK;
}

}  // namespace pio
