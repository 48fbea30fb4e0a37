// Causal attention of a batch over the paged cache (kv_pages.hip):
//   out[r, h] = sum_t softmax_t(q[r, h] . k[t] * scale) v[t].
//
// The keys fall in two parts: the prefix that all sequences have in common, whose
// columns (a column is one (query, head) pair) are those of the whole batch, and
// the tails, one per sequence. Both are cut into items of a few columns and a run
// of keys, one launch computes all of them, each item's (max, sum, weighted sum)
// goes to a workspace, and a second launch joins a column's items.
//
// Scores and weighted sums are contractions on the matrix cores, formed
// transposed, S^T = K Q^T and O^T = V^T P^T, as in attention.hip: a column is held
// by lanes c and c + 32, its softmax is arithmetic inside them, and the
// accumulator registers of S^T are, after the exp, operand registers of O^T.
//   fp16 cache: v_mfma_f32_32x32x16_f16. K is read from LDS as operands, V
//     through the transposing LDS read (a lane gets one dimension of 4 keys).
//     fp16 queries: one part of q, weights rounded to fp16 (their sum is not).
//     fp32 queries: q and the weights as two fp16 parts each, 22 bits, q scaled
//     to a fixed exponent per column first (exact).
//   fp32 cache: v_mfma_f32_32x32x2_f32.
// K and V come by direct global -> LDS copies: page ids only change addresses,
// and any mix of pages in a tile costs the same.
#include "gemm_core.hpp"
#include "kv_pages.hpp"

#include <algorithm>
#include <climits>
#include <float.h>
#include <type_traits>

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
    // items of the matrix core kernels
    int pre_items, pre_tiles, pre_splits, pre_keys;   // workgroups; column tiles; runs of keys, keys of each
    int tail_tiles, tail_splits;                      // per (request, kv head)
    bool direct;                                      // one item per column: it writes out itself
    float* part_o;                                    // [pre_splits + tail_splits][rows * H][D]
    float* part_ml;                                   // [..][rows * H][2]
};

// Rows of request i, kept inside q whatever row_start holds.
__device__ __forceinline__ void ka_rows(const KaArgs& a, int i, int& r0, int& r1) {
    r0 = max(a.row_start[i], 0);
    r1 = min(a.row_start[i + 1], a.rows);
}

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

// ------------------------------------------------- the matrix core kernels ----
typedef float ka_v16 __attribute__((ext_vector_type(16)));
typedef float ka_f4 __attribute__((ext_vector_type(4)));
typedef float ka_f2 __attribute__((ext_vector_type(2)));
typedef _Float16 ka_h8 __attribute__((ext_vector_type(8)));
typedef __fp16 ka_p4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void ka_lds_t;
typedef __attribute__((address_space(3))) ka_p4 ka_lds_p4;

constexpr int KA_COLS = 32;      // columns of a tile
constexpr int KA_KEYS = 32;      // keys of a tile
constexpr float KA_LOG2E = 1.44269504088896340736f;
// fp16 weights are held times 2^10, so that those down to 2^-24 of the largest are normal
// numbers; the sum is scaled alike.
constexpr float KA_LIFT = 10.f;
constexpr int KA_Q_EXP = 12;     // fp32 queries over an fp16 cache: the column's largest is 2^12 .. 2^13

// Geometry of a cache row and of its image in LDS: rows of RB bytes in 16-byte
// slots, slot s of row r holding chunk s ^ swz(r), so that 16 consecutive rows'
// reads of one chunk fall into different banks.
template <typename KT, int D>
struct Ka {
    static constexpr bool F16 = sizeof(KT) == 2;
    static constexpr int NT = D / 32;                  // O^T tiles
    static constexpr int RB = D * (int)sizeof(KT), SL = RB / 16;
    static constexpr int RPI = 64 / SL;                // rows of one copy instruction
    static constexpr int NI = KA_KEYS / RPI;           // copies of a tile of K (or V)
    static constexpr int TILE = KA_KEYS * RB;          // bytes
    static constexpr int QC = F16 ? D / 16 : D / 8;    // operand groups of a score
    static constexpr int OP = D + 4;                   // LDS pitch of a column's output (floats)
    __device__ static int swz(int r) { return RB == 128 ? (r >> 1) & 7 : r & 15; }
    __device__ static int slot(int r, int chunk) { return r * RB + ((chunk ^ swz(r)) << 4); }
    // dimension that register e of O^T tile n holds in half h
    __device__ static int dim(int n, int e, int h) {
        const int i = 8 * (e >> 2) + 4 * h + (e & 3);
        return F16 ? 32 * n + i : NT * i + n;
    }
};

// A column's query as operands, and the factor of its scores (base 2).
template <typename KT, int D, int XP>
struct KaQ {
    ka_h8 h[XP][Ka<KT, D>::QC];
    float cs;
};
template <int D>
struct KaQ<float, D, 1> {
    ka_f4 f[D / 8];
    float cs;
};

// q of (row, head), this lane's half of every group; zeros for a column without a row.
template <typename KT, int D, int XP>
__device__ __forceinline__ void ka_load_q(const KaArgs& a, int row, int head, bool live, int h, KaQ<KT, D, XP>& q) {
    constexpr int QC = Ka<KT, D>::QC;
    const int64_t at = (live ? row * a.q_stride + (int64_t)head * D : 0);
    q.cs = a.scale * KA_LOG2E;
    if constexpr (!Ka<KT, D>::F16) {
#pragma unroll
        for (int c = 0; c < QC; c++) {
            const int64_t e0 = at + 8 * c + 4 * h;
            if (a.q16) {
#pragma unroll
                for (int e = 0; e < 4; e++) q.f[c][e] = (float)((const _Float16*)a.q)[e0 + e];
            } else {
                q.f[c] = *(const ka_f4*)((const float*)a.q + e0);
            }
            if (!live) q.f[c] = ka_f4{0.f, 0.f, 0.f, 0.f};
        }
    } else if constexpr (XP == 1) {
#pragma unroll
        for (int c = 0; c < QC; c++) {
            q.h[0][c] = *(const ka_h8*)((const _Float16*)a.q + at + 16 * c + 8 * h);
            if (!live) q.h[0][c] = ka_h8{0, 0, 0, 0, 0, 0, 0, 0};
        }
    } else {
        float x[QC][8], most = 0.f;
        bool odd = false;
#pragma unroll
        for (int c = 0; c < QC; c++) {
            load8<float>((const float*)a.q + at + 16 * c + 8 * h, x[c]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (!live) x[c][e] = 0.f;
                most = fmaxf(most, fabsf(x[c][e]));
                odd |= !(fabsf(x[c][e]) <= FLT_MAX);
            }
        }
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        odd = odd || __shfl_xor((int)odd, 32, 64);
        int ex = 0;
        if (most > 0.f && !odd) frexpf(most, &ex);     // most = 2^ex * [0.5, 1)
        ex = KA_Q_EXP + 1 - ex;
#pragma unroll
        for (int c = 0; c < QC; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = ldexpf(x[c][e], ex);
                const _Float16 hi = (_Float16)v;
                q.h[0][c][e] = hi;
                q.h[XP - 1][c][e] = (_Float16)(v - (float)hi);
            }
        q.cs = odd ? NAN : ldexpf(q.cs, -ex);
    }
}

// S^T of one tile of 32 keys; kt: K's rows in LDS.
template <typename KT, int D, int XP>
__device__ __forceinline__ ka_v16 ka_scores(const char* kt, const KaQ<KT, D, XP>& q, int lane) {
    using T = Ka<KT, D>;
    const int key = lane & 31, h = lane >> 5;
    ka_v16 s;
#pragma unroll
    for (int e = 0; e < 16; e++) s[e] = 0.f;
    if constexpr (T::F16) {
#pragma unroll
        for (int c = 0; c < T::QC; c++) {
            const ka_h8 k = *(const ka_h8*)(kt + T::slot(key, 2 * c + h));
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q.h[0][c], s, 0, 0, 0);
            if constexpr (XP == 2) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q.h[XP - 1][c], s, 0, 0, 0);
        }
    } else {
        // 4 chains: half the rounding of one
        ka_v16 sum[4];
#pragma unroll
        for (int ch = 0; ch < 4; ch++)
#pragma unroll
            for (int e = 0; e < 16; e++) sum[ch][e] = 0.f;
#pragma unroll
        for (int c = 0; c < T::QC; c++) {
            const ka_f4 k = *(const ka_f4*)(kt + T::slot(key, 2 * c + h));
#pragma unroll
            for (int e = 0; e < 4; e++)
                sum[c % 4] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q.f[c][e], sum[c % 4], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = (sum[0][e] + sum[1][e]) + (sum[2][e] + sum[3][e]);
    }
    return s;
}

// A lane's 8 values of V^T (O^T tile n, key group kc of 16): one dimension, the
// keys of S^T's registers 8 kc .. 8 kc + 7.
template <int D>
__device__ __forceinline__ ka_h8 ka_vt(const char* vt, int n, int kc, int lane) {
    using T = Ka<_Float16, D>;
    const int i = lane & 15, g = lane >> 4, h = g >> 1;
    ka_h8 v;
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const int row = 16 * kc + 8 * b + 4 * h + (i >> 2), chunk = 4 * n + 2 * (g & 1) + ((i >> 1) & 1);
        const ka_p4 r = __builtin_amdgcn_ds_read_tr16_b64_v4f16((ka_lds_p4*)(vt + T::slot(row, chunk) + 8 * (i & 1)));
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * b + e] = (_Float16)r[e];
    }
    return v;
}

// Whether any of a tile's 32 rows of V holds inf or NaN.
template <typename KT, int D>
__device__ __forceinline__ bool ka_odd(const char* vt, int lane) {
    bool odd = false;
#pragma unroll 4
    for (int u = lane; u < Ka<KT, D>::TILE / 16; u += 64) {
        const uint4 x = *(const uint4*)(vt + 16 * u);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (sizeof(KT) == 2) odd |= (w[e] & 0x7c00u) == 0x7c00u || (w[e] & 0x7c000000u) == 0x7c000000u;
            else odd |= (w[e] & 0x7f800000u) == 0x7f800000u;
        }
    }
    return __any(odd);
}

// A column's running softmax: (max, sum) in base 2, O^T.
template <typename KT, int D>
struct KaAcc {
    float m, l;
    ka_v16 o[Ka<KT, D>::NT];
    __device__ void clear() {
        m = -FLT_MAX;
        l = 0.f;
#pragma unroll
        for (int n = 0; n < Ka<KT, D>::NT; n++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[n][e] = 0.f;
    }
};

// Scores -> weights (in s), and the running maximum and sum. The tile's keys
// from t0; edge (wave-uniform): some column does not see all of them.
template <typename KT, int D>
__device__ __forceinline__ void ka_softmax(KaAcc<KT, D>& x, ka_v16& s, float cs, int t0, int limit, bool edge, int h) {
    constexpr float lift = Ka<KT, D>::F16 ? KA_LIFT : 0.f;
    float top = -INFINITY;
    if (edge) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const bool seen = t0 + 8 * (e >> 2) + 4 * h + (e & 3) < limit;
            s[e] = seen ? s[e] * cs : -INFINITY;
            top = fmaxf(top, s[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            s[e] *= cs;
            top = fmaxf(top, s[e]);
        }
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float m = fmaxf(x.m, top);
    if (__any(m != x.m)) {
        const float corr = __builtin_amdgcn_exp2f(x.m - m);
        x.l *= corr;
#pragma unroll
        for (int n = 0; n < Ka<KT, D>::NT; n++)
#pragma unroll
            for (int e = 0; e < 16; e++) x.o[n][e] *= corr;
        x.m = m;
    }
    const float base = m - lift;
    float sum[16];
#pragma unroll
    for (int e = 0; e < 16; e++) {
        s[e] = __builtin_amdgcn_exp2f(s[e] - base);     // -inf: 0 (the maximum is finite, or the scores are no numbers)
        sum[e] = s[e];
    }
#pragma unroll
    for (int n = 8; n >= 1; n >>= 1)
#pragma unroll
        for (int e = 0; e < n; e++) sum[e] += sum[e + n];
    x.l += sum[0];
}

// O^T += V^T P^T over one tile. `odd`: V holds inf or NaN and some column does not
// see all keys: 0 * inf would make those columns NaN, so inf and NaN are taken out of
// the product and added where a column sees them (their weights are positive).
template <typename KT, int D, int XP>
__device__ __forceinline__ void ka_values(KaAcc<KT, D>& x, const ka_v16& p, const char* vt, int lane, bool odd, int t0,
                                          int limit) {
    using T = Ka<KT, D>;
    const int h = lane >> 5;
    typedef typename std::conditional<T::NT == 4, ka_f4, ka_f2>::type V;
    auto row = [&](int e) {                // fp32: dimensions NT i .. of the key of register e
        const int r = 8 * (e >> 2) + 4 * h + (e & 3), i = lane & 31;
        if constexpr (T::NT == 4) return *(const V*)(vt + T::slot(r, i));
        else return *(const V*)(vt + T::slot(r, i >> 1) + 8 * (i & 1));
    };
    auto product = [&](auto finite) {
        if constexpr (T::F16) {
#pragma unroll
            for (int kc = 0; kc < 2; kc++) {
                ka_h8 w[XP];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const _Float16 hi = (_Float16)p[8 * kc + e];
                    w[0][e] = hi;
                    if constexpr (XP == 2) w[XP - 1][e] = (_Float16)(p[8 * kc + e] - (float)hi);
                }
#pragma unroll
                for (int n = 0; n < T::NT; n++) {
                    ka_h8 v = ka_vt<D>(vt, n, kc, lane);
                    if constexpr (!decltype(finite)::value) {
#pragma unroll
                        for (int e = 0; e < 8; e++) v[e] = fabsf((float)v[e]) <= 65504.f ? v[e] : (_Float16)0;
                    }
                    x.o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w[0], x.o[n], 0, 0, 0);
                    if constexpr (XP == 2) x.o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w[XP - 1], x.o[n], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                V v = row(e);
#pragma unroll
                for (int n = 0; n < T::NT; n++) {
                    if constexpr (!decltype(finite)::value) v[n] = fabsf(v[n]) <= FLT_MAX ? v[n] : 0.f;
                    x.o[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[n], p[e], x.o[n], 0, 0, 0);
                }
            }
        }
    };
    if (!odd) {
        product(std::true_type{});
        return;
    }
    product(std::false_type{});
    // how many +inf, -inf and NaN each (dimension, column) sees
#pragma unroll
    for (int n = 0; n < T::NT; n++) {
#pragma unroll 1
        for (int kind = 0; kind < 3; kind++) {
            const float what = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
            ka_v16 c;
#pragma unroll
            for (int e = 0; e < 16; e++) c[e] = 0.f;
            auto is = [&](float f) { return kind == 2 ? f != f : f == what; };
            auto sees = [&](int e) { return t0 + 8 * (e >> 2) + 4 * h + (e & 3) < limit; };
            if constexpr (T::F16) {
#pragma unroll 1
                for (int kc = 0; kc < 2; kc++) {
                    const ka_h8 v = ka_vt<D>(vt, n, kc, lane);
                    ka_h8 k, w;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        k[e] = is((float)v[e]) ? (_Float16)1 : (_Float16)0;
                        w[e] = sees(8 * kc + e) ? (_Float16)1 : (_Float16)0;
                    }
                    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, w, c, 0, 0, 0);
                }
            } else {
#pragma unroll 1
                for (int e = 0; e < 16; e++)
                    c = __builtin_amdgcn_mfma_f32_32x32x2f32(is(row(e)[n]) ? 1.f : 0.f, sees(e) ? 1.f : 0.f, c, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (c[e] > 0.5f) x.o[n][e] += what;
        }
    }
}

// ---- one item by 4 waves: 32 columns, every 4th tile of the keys each, from a
// piece of LDS of the wave's own (one tile of K, one of V). The next K tile is
// copied during this one's softmax and product with V, the next V tile during the
// next scores. No barriers: a wave waits for its own copies.
template <int N>
__device__ __forceinline__ void ka_wait_copies() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (0xF << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void ka_wait_reads() {     // the wave's LDS reads are done: copies may overwrite them
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);               // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

struct KaKeys {
    const int32_t* row;      // the table row that the keys are read through
    int g, k0, k1;           // kv head, keys
};

template <typename KT, int D, int XP>
__device__ __forceinline__ void ka_walk(const KaArgs& a, const KaKeys& keys, char* mine, int w, int lane, int limit,
                                        int least, const KaQ<KT, D, XP>& q, KaAcc<KT, D>& x, bool& bad) {
    using T = Ka<KT, D>;
    const pio_kv_cache& c = a.c;
    const int h = lane >> 5, lg = kv_log2(c.page_size), mask = c.page_size - 1, per_page = c.n_kv_heads * c.page_size;
    const char* kb = (const char*)c.kv + ((int64_t)(2 * a.layer) * c.n_pages * per_page + (int64_t)keys.g * c.page_size) * T::RB;
    const char* vb = kb + (int64_t)c.n_pages * per_page * T::RB;
    char *kt = mine, *vt = mine + T::TILE;
    const int tiles = (keys.k1 - keys.k0 + KA_KEYS - 1) / KA_KEYS;
    // cache row of this lane's key of tile j (keys behind the last one re-read it)
    auto key_row = [&](int j) -> uint32_t {
        const int t = min(keys.k0 + min(j, tiles - 1) * KA_KEYS + (lane & 31), keys.k1 - 1);
        int page = keys.row[t >> lg];
        if (page < 0 || page >= c.n_pages) {
            bad = true;
            page = 0;
        }
        return (uint32_t)page * (uint32_t)per_page + (uint32_t)(t & mask);
    };
    int64_t off[T::NI];
    auto offsets = [&](uint32_t row) {
#pragma unroll
        for (int i = 0; i < T::NI; i++) {
            const int r = T::RPI * i + lane / T::SL;
            off[i] = (int64_t)(uint32_t)__shfl((int)row, r, 64) * T::RB + (((lane % T::SL) ^ T::swz(r)) << 4);
        }
    };
    auto copy = [&](const char* from, char* to) {
#pragma unroll
        for (int i = 0; i < T::NI; i++)
            __builtin_amdgcn_global_load_lds((const void*)(from + off[i]), (ka_lds_t*)(to + i * 1024), 16, 0, 0);
    };
    if (w >= tiles) return;
    uint32_t next = key_row(w);
    offsets(next);
    next = key_row(w + 4);
    copy(kb, kt);
    copy(vb, vt);
    for (int j = w; j < tiles; j += 4) {
        const int t0 = keys.k0 + j * KA_KEYS;
        const bool more = j + 4 < tiles, edge = t0 + KA_KEYS > least;
        ka_wait_copies<T::NI>();
        ka_v16 s = ka_scores<KT, D, XP>(kt, q, lane);
        ka_wait_reads();
        if (more) {
            offsets(next);
            copy(kb, kt);
            next = key_row(j + 8);
        }
        ka_softmax<KT, D>(x, s, q.cs, t0, limit, edge, h);
        if (more) ka_wait_copies<T::NI + 1>();
        else ka_wait_copies<0>();
        const bool odd = edge && ka_odd<KT, D>(vt, lane);
        ka_values<KT, D, XP>(x, s, vt, lane, odd, t0, limit);
        ka_wait_reads();
        if (more) copy(vb, vt);
    }
}

// A lane's part of an accumulated column, times f, into LDS (column's row at `to`).
template <typename KT, int D>
__device__ __forceinline__ void ka_spill(const KaAcc<KT, D>& x, float f, float* to, int h) {
    using T = Ka<KT, D>;
    if constexpr (T::F16) {
#pragma unroll
        for (int n = 0; n < T::NT; n++)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *(ka_f4*)(to + T::dim(n, e, h)) = ka_f4{x.o[n][e] * f, x.o[n][e + 1] * f, x.o[n][e + 2] * f, x.o[n][e + 3] * f};
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++)
#pragma unroll
            for (int n = 0; n < T::NT; n++) to[T::dim(n, e, h)] = x.o[n][e] * f;
    }
}

// 4 consecutive dimensions from d of column (row, head): an item's part of it, or
// the result.
__device__ __forceinline__ void ka_put(const KaArgs& a, int D, int slot, int row, int head, int d, ka_f4 v, float m, float l) {
    const int64_t at = (int64_t)slot * a.rows * a.H + (int64_t)row * a.H + head;
    *(ka_f4*)(a.part_o + at * D + d) = v;
    if (d == 0) *(ka_f2*)(a.part_ml + 2 * at) = ka_f2{m, l};
}
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

// Keys of tail split z of a request: from `from` to `len`, in runs of whole rounds
// of 4 tiles; how many runs there are.
__host__ __device__ __forceinline__ int ka_tail_runs(int from, int len, int splits, int& keys) {
    constexpr int ROUND = 4 * KA_KEYS;
    if (len <= from) {
        keys = 0;
        return 0;
    }
    const int rounds = (len - from + ROUND - 1) / ROUND;
    const int per = (rounds + splits - 1) / splits;
    keys = per * ROUND;
    return (rounds + per - 1) / per;
}

// Rows in LDS that a tile of columns has: limit (keys that the row sees) and
// whether a request has the row.
template <int N>
struct KaRows {
    int limit[N];
};

// The limits of rows first .. first + N - 1 of the batch, by the whole workgroup.
template <int N>
__device__ __forceinline__ void ka_limits(const KaArgs& a, int first, KaRows<N>& r) {
    for (int i = threadIdx.x; i < N; i += blockDim.x) r.limit[i] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
        int r0, r1;
        ka_rows(a, i, r0, r1);
        const int lo = max(r0, first), hi = min(r1, first + N);
        if (lo >= hi) continue;
        const int L = kv_seq_len(a.c, a.seq[i]);
        if (L < 0) continue;
        for (int row = lo; row < hi; row++) r.limit[row - first] = max(L - (r1 - row) + 1, 0);
    }
    __syncthreads();
}

__device__ __forceinline__ int ka_wave_min(int v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return v;
}

// Workgroup items. GROUPS groups of 4 waves; WIDE: the prefix is taken by 8 waves
// together (128 columns, below), else by groups of 4 as the tails are.
template <typename KT, int D, int GROUPS>
constexpr size_t ka_group_bytes() {
    using T = Ka<KT, D>;
    return std::max<size_t>(4 * 2 * T::TILE, (size_t)4 * KA_COLS * T::OP * 4);
}

constexpr int KA_WIDE_MIN = 64;      // columns from which on
constexpr int KA_WIDE_COLS = 128, KA_WIDE_KEYS = 64, KA_STAGES = 4, KA_WIDE_PAGES = 4096;
template <int D>
constexpr size_t ka_wide_bytes() {
    return std::max<size_t>({(size_t)KA_STAGES * 2 * KA_WIDE_KEYS * D * 2, (size_t)KA_WIDE_COLS * (D + 4) * 4,
                             2 * ka_group_bytes<_Float16, D, 2>()});
}

// A group's columns joined over its 4 waves and written. first_limit: keys that row
// row0 sees (fewer than one: none; each row behind it sees one more).
template <typename KT, int D>
__device__ __forceinline__ void ka_join(const KaArgs& a, KaAcc<KT, D>& x, char* lds, float (*ml)[KA_COLS][2], int w, int lane,
                                        bool bad, int slot, int row0, int g, int c0, int ncols, bool live,
                                        int first_limit = 1) {
    using T = Ka<KT, D>;
    const int col = lane & 31, h = lane >> 5;
    x.l += __shfl_xor(x.l, 32, 64);
    if (__any(bad)) x.l = NAN;
    if (h == 0) {
        ml[w][col][0] = x.m;
        ml[w][col][1] = x.l;
    }
    __syncthreads();
    float mx = ml[0][col][0];
#pragma unroll
    for (int i = 1; i < 4; i++) mx = fmaxf(mx, ml[i][col][0]);
    ka_spill<KT, D>(x, __builtin_amdgcn_exp2f(x.m - mx), (float*)lds + (w * KA_COLS + col) * T::OP, h);
    __syncthreads();
    if (live)
        for (int i = w * 64 + lane; i < KA_COLS * (D / 4); i += 256) {
            const int c = i / (D / 4), d = (i % (D / 4)) * 4;
            if (c0 + c >= ncols) break;
            float m = ml[0][c][0], l = 0.f;
#pragma unroll
            for (int k = 1; k < 4; k++) m = fmaxf(m, ml[k][c][0]);
            ka_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v += *(const ka_f4*)((const float*)lds + (k * KA_COLS + c) * T::OP + d);
                l += ml[k][c][1] * __builtin_amdgcn_exp2f(ml[k][c][0] - m);
            }
            const int row = row0 + (c0 + c) / a.G, head = g * a.G + (c0 + c) % a.G;
            if (a.direct) {
                v = v / l;
                if (first_limit + row - row0 <= 0 && l == 0.f) v = ka_f4{0.f, 0.f, 0.f, 0.f};
                ka_out(a, D, row, head, d, v);
            }
            else ka_put(a, D, slot, row, head, d, v, m, l);
        }
}

// The prefix item of 8 waves: 128 columns, 4 tiles of 32 by waves w % 4, the two
// halves of every 64 keys by waves w / 4. K and V of 64 keys are one of KA_STAGES
// stages in LDS that all waves copy together.
template <int D, int XP>
__device__ __forceinline__ void ka_wide(const KaArgs& a, char* lds, int* pages, float (*ml)[KA_COLS][2], KaRows<128>& rows,
                                        int g, int split, int ct) {
    typedef _Float16 KT;
    using T = Ka<KT, D>;
    const pio_kv_cache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), cg = w & 3, kg = w >> 2;
    const int col = lane & 31, h = lane >> 5;
    const int lg = kv_log2(c.page_size), mask = c.page_size - 1, per_page = c.n_kv_heads * c.page_size;
    const int k0 = split * a.pre_keys, k1 = min(k0 + a.pre_keys, a.shared);
    const int ncols = a.rows * a.G, c0 = ct * KA_WIDE_COLS + cg * KA_COLS, first = ct * KA_WIDE_COLS / a.G;
    bool bad = a.seq[0] < 0 || a.seq[0] >= c.max_seqs;
    const int32_t* trow = c.table + (int64_t)(bad ? 0 : a.seq[0]) * c.max_pages;
    const int p0 = k0 >> lg, np = ((k1 - 1) >> lg) - p0 + 1;
    for (int i = tid; i < np; i += 512) {
        int page = trow[p0 + i];
        if (page < 0 || page >= c.n_pages) {
            bad = true;
            page = 0;
        }
        pages[i] = page;
    }
    ka_limits(a, first, rows);
    const bool has = c0 + col < ncols;
    const int row = has ? (c0 + col) / a.G : 0, head = g * a.G + (has ? (c0 + col) % a.G : 0);
    int limit = has ? rows.limit[row - first] : -1;
    limit = limit < 0 ? k1 : min(limit, k1);
    const int least = ka_wave_min(limit);
    KaQ<KT, D, XP> q;
    ka_load_q<KT, D, XP>(a, row, head, has, h, q);
    KaAcc<KT, D> x;
    x.clear();

    const char* kb = (const char*)c.kv + ((int64_t)(2 * a.layer) * c.n_pages * per_page + (int64_t)g * c.page_size) * T::RB;
    const char* vb = kb + (int64_t)c.n_pages * per_page * T::RB;
    constexpr int STAGE = 2 * KA_WIDE_KEYS * T::RB, PW = 8 / T::RPI;    // copies of a wave: PW of K, PW of V
    // stage s: its rows 8 w .. 8 w + 7 (keys behind the last one re-read it)
    auto copy = [&](int s) {
        char* to = lds + (s % KA_STAGES) * STAGE + 8 * w * T::RB;
#pragma unroll
        for (int i = 0; i < PW; i++) {
            const int r = 8 * w + T::RPI * i + lane / T::SL, t = min(k0 + s * KA_WIDE_KEYS + r, k1 - 1);
            const uint32_t at = (uint32_t)pages[(t >> lg) - p0] * (uint32_t)per_page + (uint32_t)(t & mask);
            const int64_t off = (int64_t)at * T::RB + (((lane % T::SL) ^ T::swz(r)) << 4);
            __builtin_amdgcn_global_load_lds((const void*)(kb + off), (ka_lds_t*)(to + i * 1024), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const void*)(vb + off), (ka_lds_t*)(to + KA_WIDE_KEYS * T::RB + i * 1024), 16, 0, 0);
        }
    };
    const int stages = (k1 - k0 + KA_WIDE_KEYS - 1) / KA_WIDE_KEYS;
    ka_wait_copies<0>();               // q is here: the waits below count copies alone
#pragma unroll
    for (int s = 0; s < KA_STAGES - 1; s++) copy(s);
    for (int s = 0; s < stages; s++) {
        stage_barrier<(KA_STAGES - 2) * 2 * PW>();
        // into the stage that every wave has read before this barrier; past the end the last key again
        copy(s + KA_STAGES - 1);
        const char* kt = lds + (s % KA_STAGES) * STAGE + kg * T::TILE;
        const char* vt = kt + KA_WIDE_KEYS * T::RB;
        const int t0 = k0 + s * KA_WIDE_KEYS + kg * KA_KEYS;
        const bool edge = t0 + KA_KEYS > least;
        ka_v16 sc = ka_scores<KT, D, XP>(kt, q, lane);
        ka_softmax<KT, D>(x, sc, q.cs, t0, limit, edge, h);
        const bool odd = edge && ka_odd<KT, D>(vt, lane);
        ka_values<KT, D, XP>(x, sc, vt, lane, odd, t0, limit);
    }
    // the halves of the keys meet in LDS
    x.l += __shfl_xor(x.l, 32, 64);
    if (h == 0) {
        ml[w][col][0] = x.m;
        ml[w][col][1] = x.l;
    }
    const bool any_bad = __syncthreads_or(bad);        // and every copy has landed, every stage is read
    if (any_bad && tid == 0) atomicOr(c.work, KV_BAD);
    const float mx = fmaxf(ml[cg][col][0], ml[cg + 4][col][0]), f = __builtin_amdgcn_exp2f(x.m - mx);
    float* ob = (float*)lds + (cg * KA_COLS + col) * T::OP;
    if (kg) ka_spill<KT, D>(x, f, ob, h);
    __syncthreads();
    if (!kg) {
#pragma unroll
        for (int n = 0; n < T::NT; n++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                ka_f4* at = (ka_f4*)(ob + T::dim(n, e, h));
                *at += ka_f4{x.o[n][e] * f, x.o[n][e + 1] * f, x.o[n][e + 2] * f, x.o[n][e + 3] * f};
            }
    }
    __syncthreads();
    for (int i = tid; i < KA_WIDE_COLS * (D / 4); i += 512) {
        const int cc = i / (D / 4), d = (i % (D / 4)) * 4, at = ct * KA_WIDE_COLS + cc;
        if (at >= ncols) break;
        const float m0 = ml[cc >> 5][cc & 31][0], m1 = ml[4 + (cc >> 5)][cc & 31][0], m = fmaxf(m0, m1);
        float l = ml[cc >> 5][cc & 31][1] * __builtin_amdgcn_exp2f(m0 - m) +
                  ml[4 + (cc >> 5)][cc & 31][1] * __builtin_amdgcn_exp2f(m1 - m);
        if (any_bad) l = NAN;
        ka_put(a, D, split, at / a.G, g * a.G + at % a.G, d, *(const ka_f4*)((const float*)lds + cc * T::OP + d), m, l);
    }
}

// Workgroups: the prefix's items, then the tails'. WIDE: 8 waves, prefix items of
// all of them and tail items of 4; else 4 waves, items of 4.
template <typename KT, int D, int XP, bool WIDE>
__global__ __launch_bounds__(WIDE ? 512 : 256, sizeof(KT) == 4 ? 1 : 2) void ka_kernel(KaArgs a) {
    constexpr int GROUPS = WIDE ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) char ka_lds[];
    __shared__ float ml[4 * GROUPS][KA_COLS][2];
    __shared__ KaRows<WIDE ? 128 : KA_COLS> rows;
    const pio_kv_cache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, w8 = __builtin_amdgcn_readfirstlane(tid >> 6), w = w8 & 3, grp = w8 >> 2;
    const int col = lane & 31, h = lane >> 5, Hk = c.n_kv_heads;
    if ((int)blockIdx.x < a.pre_items) {
        // the column tiles of a (kv head, run of keys) on one XCD, next to each other: they read the same K and V
        const int x = blockIdx.x & 7, y = blockIdx.x >> 3, ct = y % a.pre_tiles, unit = (y / a.pre_tiles) * 8 + x;
        if (unit >= Hk * a.pre_splits) return;
        const int g = unit % Hk, split = unit / Hk;
        if constexpr (WIDE) {
            ka_wide<D, XP>(a, ka_lds, (int*)(ka_lds + ka_wide_bytes<D>()), ml, rows, g, split, ct);
        } else {
            const int ncols = a.rows * a.G, c0 = ct * KA_COLS, first = c0 / a.G;
            bool bad = a.seq[0] < 0 || a.seq[0] >= c.max_seqs;
            KaKeys keys{c.table + (int64_t)(bad ? 0 : a.seq[0]) * c.max_pages, g, split * a.pre_keys, 0};
            keys.k1 = min(keys.k0 + a.pre_keys, a.shared);
            ka_limits(a, first, rows);
            const bool has = c0 + col < ncols;
            const int row = has ? (c0 + col) / a.G : 0, head = g * a.G + (has ? (c0 + col) % a.G : 0);
            int limit = has ? rows.limit[row - first] : -1;
            limit = limit < 0 ? keys.k1 : min(limit, keys.k1);
            KaQ<KT, D, XP> q;
            ka_load_q<KT, D, XP>(a, row, head, has, h, q);
            KaAcc<KT, D> acc;
            acc.clear();
            ka_walk<KT, D, XP>(a, keys, ka_lds + w * 2 * Ka<KT, D>::TILE, w, lane, limit, ka_wave_min(limit), q, acc, bad);
            if (__any(bad) && lane == 0) atomicOr(c.work, KV_BAD);
            ka_join<KT, D>(a, acc, ka_lds, ml, w, lane, bad, split, 0, g, c0, ncols, true);
        }
        return;
    }
    // tails: (request, kv head, column tile, run), two neighbours per workgroup of 8 waves
    int item = ((int)blockIdx.x - a.pre_items) * GROUPS + grp;
    const int z = item % a.tail_splits;
    item /= a.tail_splits;
    const int ct0 = item % a.tail_tiles;
    item /= a.tail_tiles;
    const int g = item % Hk, i = item / Hk;
    int r0 = 0, r1 = 0, L = -1, s = -1, keys_per = 0, runs = 0;
    if (i < a.n) {
        ka_rows(a, i, r0, r1);
        s = a.seq[i];
        L = kv_seq_len(c, s);
        runs = ka_tail_runs(a.shared, L, a.tail_splits, keys_per);
    }
    char* lds = ka_lds + grp * ka_group_bytes<KT, D, GROUPS>();
    float (*gml)[KA_COLS][2] = ml + 4 * grp;
    const int ncols = max(r1 - r0, 0) * a.G;
    // columns beyond the tiles of the grid (a request of more rows than announced): more rounds.
    // Both groups of a workgroup make as many, for the barriers.
    const bool live = i < a.n && (a.direct || z < runs);
    int rounds = live ? (ncols + KA_COLS - 1) / KA_COLS - ct0 : 0;
    rounds = rounds > 0 ? (rounds + a.tail_tiles - 1) / a.tail_tiles : 0;
    if constexpr (GROUPS == 2) {
        __shared__ int most[2];
        if ((tid & 255) == 0) most[grp] = rounds;
        __syncthreads();
        rounds = max(most[0], most[1]);
    }
    for (int r = 0; r < rounds; r++) {
        const int c0 = (ct0 + r * a.tail_tiles) * KA_COLS;
        const bool on = live && c0 < ncols;
        bool bad = L < 0;
        KaAcc<KT, D> acc;
        acc.clear();
        if (on && z < runs) {
            const bool has = c0 + col < ncols;
            const int row = has ? r0 + (c0 + col) / a.G : r0, head = g * a.G + (has ? (c0 + col) % a.G : 0);
            KaKeys keys{c.table + (int64_t)s * c.max_pages, g, a.shared + z * keys_per, 0};
            keys.k1 = min(keys.k0 + keys_per, L);
            const int limit = has ? min(L - (r1 - row) + 1, keys.k1) : keys.k1;
            KaQ<KT, D, XP> q;
            ka_load_q<KT, D, XP>(a, row, head, has, h, q);
            ka_walk<KT, D, XP>(a, keys, lds + w * 2 * Ka<KT, D>::TILE, w, lane, limit, ka_wave_min(limit), q, acc, bad);
        }
        if (on && __any(bad) && lane == 0) atomicOr(c.work, KV_BAD);
        if (r) __syncthreads();        // the last round's output is out of LDS
        ka_join<KT, D>(a, acc, lds, gml, w, lane, bad, a.pre_splits + z, r0, g, c0, ncols, on,
                        L - (r1 - r0) + 1);
    }
}

// A column's items joined, one workgroup per column; D / 4 lanes have its dimensions,
// the groups of them take every such item.
template <int D>
__global__ __launch_bounds__(256) void ka_merge_kernel(KaArgs a) {
    constexpr int TPC = D / 4, Z = 256 / TPC;
    __shared__ __attribute__((aligned(16))) float so[Z][D];
    __shared__ float sml[Z][2];
    __shared__ int req, behind;
    const pio_kv_cache& c = a.c;
    const int tid = threadIdx.x, zg = tid / TPC, d = (tid % TPC) * 4, row = blockIdx.x / a.H, head = blockIdx.x - row * a.H;
    if (tid == 0) req = -1;
    __syncthreads();
    for (int i = tid; i < a.n; i += 256) {
        int r0, r1;
        ka_rows(a, i, r0, r1);
        if (row >= r0 && row < r1) {
            req = i;
            behind = r1 - row;
        }
    }
    __syncthreads();
    if (req < 0) return;               // behind the last request
    const int s = a.seq[req], L = kv_seq_len(c, s);
    const bool bad = L < 0 || (a.shared > 0 && kv_seq_len(c, a.seq[0]) < 0);
    int keys;
    const int runs = bad ? 0 : ka_tail_runs(a.shared, L, a.tail_splits, keys), parts = bad ? 0 : a.pre_splits + runs;
    const int64_t step = (int64_t)a.rows * a.H, at = (int64_t)blockIdx.x;
    float m = -FLT_MAX, l = 0.f;
    ka_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int z = zg; z < parts; z += Z) {
        const ka_f2 ml = *(const ka_f2*)(a.part_ml + 2 * (at + z * step));
        const ka_f4 o = *(const ka_f4*)(a.part_o + (at + z * step) * D + d);
        const float nm = fmaxf(m, ml[0]), f = __builtin_amdgcn_exp2f(m - nm), fz = __builtin_amdgcn_exp2f(ml[0] - nm);
        l = l * f + ml[1] * fz;
        v = v * f + o * fz;
        m = nm;
    }
    *(ka_f4*)&so[zg][d] = v;
    if (d == 0) {
        sml[zg][0] = m;
        sml[zg][1] = l;
    }
    __syncthreads();
    if (zg) return;
    for (int z = 1; z < Z; z++) m = fmaxf(m, sml[z][0]);
    l = 0.f;
    v = ka_f4{0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < Z; z++) {
        const float f = __builtin_amdgcn_exp2f(sml[z][0] - m);
        l += sml[z][1] * f;
        v += *(const ka_f4*)&so[z][d] * f;
    }
    v = v / l;
    if (L - behind + 1 <= 0) v = ka_f4{0.f, 0.f, 0.f, 0.f};     // sees no key
    if (bad) v = ka_f4{NAN, NAN, NAN, NAN};
    ka_out(a, D, row, head, d, v);
    if (bad && tid == 0) atomicOr(c.work, KV_BAD);
}

template <typename KT, int D, int XP, bool WIDE>
static int ka_launch(const KaArgs& a, hipStream_t st) {
    constexpr int GROUPS = WIDE ? 2 : 1;
    size_t lds = ka_group_bytes<KT, D, GROUPS>();
    if constexpr (WIDE) lds = ka_wide_bytes<D>() + KA_WIDE_PAGES * sizeof(int);
    const int64_t tails = (int64_t)a.n * a.c.n_kv_heads * a.tail_tiles * a.tail_splits;
    PIO_TRY((allow_lds<ka_kernel<KT, D, XP, WIDE>>(lds)));
    ka_kernel<KT, D, XP, WIDE><<<(unsigned)(a.pre_items + (tails + GROUPS - 1) / GROUPS), 256 * GROUPS, lds, st>>>(a);
    PIO_LAUNCHED();
    if (!a.direct) {
        ka_merge_kernel<D><<<a.rows * a.H, 256, 0, st>>>(a);
        PIO_LAUNCHED();
    }
    return PIO_OK;
}

template <int D>
static int ka_route(const KaArgs& a, bool wide, hipStream_t st) {
    if (a.c.kv_dtype == PIO_F32) return ka_launch<float, D, 1, false>(a, st);
    if (a.q16) return wide ? ka_launch<_Float16, D, 1, true>(a, st) : ka_launch<_Float16, D, 1, false>(a, st);
    return wide ? ka_launch<_Float16, D, 2, true>(a, st) : ka_launch<_Float16, D, 2, false>(a, st);
}

// Items for the matrix core kernels.
static int ka_matrix(KaArgs& a, int max_rows, hipStream_t st) {
    const int Hk = a.c.n_kv_heads, cus = 256;
    const bool f16 = a.c.kv_dtype == PIO_F16;
    const int64_t cols = (int64_t)a.rows * a.G;
    const bool wide = f16 && a.shared > 0 && cols > KA_WIDE_MIN;
    if (a.shared > 0) {
        // prefix: as many items as the device holds at once, each of at least a few tiles of keys
        const int width = wide ? KA_WIDE_COLS : KA_COLS, round = wide ? KA_WIDE_KEYS : 4 * KA_KEYS;
        const int at_once = wide || !f16 ? cus : 2 * cus;
        a.pre_tiles = ceil_div(cols, width);
        int64_t splits = std::max<int64_t>(1, at_once / std::max<int64_t>(1, (int64_t)Hk * a.pre_tiles));
        splits = std::min<int64_t>(splits, ceil_div(a.shared, 4 * KA_KEYS));
        int keys = ceil_div(ceil_div(a.shared, splits), round) * round;
        if (wide) keys = (int)std::min<int64_t>(keys, (int64_t)(KA_WIDE_PAGES - 1) * a.c.page_size / round * round);
        a.pre_keys = keys;
        a.pre_splits = ceil_div(a.shared, keys);
        const int64_t items = (int64_t)ceil_div((int64_t)Hk * a.pre_splits, 8) * 8 * a.pre_tiles;
        PIO_REQUIRE(items <= INT_MAX / 2, "pio_kv_attention: too many rows over %d shared tokens", a.shared);
        a.pre_items = (int)items;
    }
    a.tail_tiles = ceil_div((int64_t)std::min(max_rows, a.rows) * a.G, KA_COLS);
    const int64_t items = (int64_t)a.n * Hk * a.tail_tiles;
    PIO_REQUIRE(items <= INT_MAX / 64, "pio_kv_attention: %d requests of %d rows are too many", a.n, max_rows);
    const int64_t longest = std::max<int64_t>((int64_t)a.c.max_pages * a.c.page_size - a.shared, 1);
    a.tail_splits = (int)std::max<int64_t>(1, std::min<int64_t>({4 * cus / items, 32, ceil_div(longest, 4 * KA_KEYS)}));
    a.direct = a.shared == 0 && a.tail_splits == 1;
    Scratch ws;
    if (!a.direct) {
        const size_t parts = (size_t)(a.pre_splits + a.tail_splits) * a.rows * a.H;
        PIO_TRY(ws.get(parts * (a.c.head_dim + 2) * sizeof(float), st));
        a.part_o = (float*)ws.ptr;
        a.part_ml = a.part_o + parts * a.c.head_dim;
    }
    return a.c.head_dim == 128 ? ka_route<128>(a, wide, st) : ka_route<64>(a, wide, st);
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
    if (c->head_dim == 128 || c->head_dim == 64) return ka_matrix(a, max_rows, st);
    if (c->kv_dtype == PIO_F32) ka_simple_kernel<float><<<rows * n_heads, KA_THREADS, 0, st>>>(a);
    else ka_simple_kernel<_Float16><<<rows * n_heads, KA_THREADS, 0, st>>>(a);
    PIO_LAUNCHED();
    return PIO_OK;
}
