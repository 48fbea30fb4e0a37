// Causal attention of a batch over the paged cache (kv_pages.hip):
//   out[r, h] = sum_t softmax_t(q[r, h] . k[t] * scale) v[t].
//
// The keys fall in two parts: the prefix that all sequences have in common, whose
// columns (a column is one (query, head) pair) are those of the whole batch, and
// the tails, one per sequence. Both are cut into items of a few columns and a run
// of keys, each item's (max, sum, weighted sum) goes to a workspace, and a last
// launch joins a column's items.
//
// Scores and weighted sums are contractions on the matrix cores, formed
// transposed, S^T = K Q^T and O^T = V^T P^T, as in attention.hip: a column is held
// by lanes c and c + 32, its softmax is arithmetic inside them, and the
// accumulator registers of S^T are, after the exp, operand registers of O^T.
//   fp16 cache: v_mfma_f32_16x16x32_f16 or 32x32x16. K is read from LDS as operands, V
//     through the transposing LDS read (a lane gets one dimension of 4 keys).
//     fp16 queries: one part of q, weights rounded to fp16 (their sum is not).
//     fp32 queries: q and the weights as two fp16 parts each, 22 bits, q scaled
//     to a fixed exponent per column first (exact).
//   fp32 cache: v_mfma_f32_16x16x4_f32.
// K and V come by direct global -> LDS copies: page ids only change addresses,
// and any mix of pages in a tile costs the same.
#include "gemm_core.hpp"
#include "kv_attention.hpp"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace pio {

// Head dimensions other than 64 and 128. One workgroup per (row, head): 256 keys at a time,
// a thread for each key's score, then a thread for each dimension of the weighted sum, bound
// by the waits for a row of K and for KA_DEEP values. 32 sequences of 2,040 to 2,700 tokens, 16 heads of
// 256: 210 us (one value at a time, K 16 bytes at a time: 860).
constexpr int KA_DEEP = 16;
template <typename KT>
__global__ __launch_bounds__(KA_THREADS) void ka_simple_kernel(KaArgs a) {
    __shared__ float qs[256], ps[KA_THREADS], red[4];
    __shared__ int64_t vrow[KA_THREADS];       // where a key's value is, -1: nowhere
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
    // the same in every thread, always; of seq[0] only the table row counts, and only where tokens are shared
    int bad = L < 0 || (a.shared > 0 && (s0 < 0 || s0 >= c.max_seqs));
    const int64_t head = (int64_t)c.page_size * D, page_e = head * c.n_kv_heads;
    const KT* kb = (const KT*)c.kv + (int64_t)(2 * a.layer) * c.n_pages * page_e + g * head;
    const KT* vb = kb + (int64_t)c.n_pages * page_e;
    float m = -FLT_MAX, l = 0.f, o = 0.f;
    for (int t0 = 0; t0 < limit && !bad; t0 += KA_THREADS) {
        const int t = t0 + tid;
        float sc = -INFINITY;
        int64_t vr = -1;
        int wrong = 0;
        if (t < limit) {
            const int page = c.table[(int64_t)(t < a.shared ? s0 : s) * c.max_pages + (t >> lg)];
            if (page < 0 || page >= c.n_pages) {
                wrong = 1;
            } else {
                const int64_t at = page * page_e + (int64_t)(t & (c.page_size - 1)) * D;
                float d = 0.f;
                for (int e0 = 0; e0 < D; e0 += 32) {           // whole lines of a row at once
                    float x[4][8];
#pragma unroll
                    for (int i = 0; i < 4; i++) load8<KT>(kb + at + min(e0 + 8 * i, D - 8), x[i]);
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (e0 + 8 * i < D) d = fmaf(x[i][j], qs[e0 + 8 * i + j], d);
                }
                sc = d * a.scale;
                vr = at;
            }
        }
        vrow[tid] = vr;
        float mt = wave_max(sc);
        if ((tid & 63) == 0) red[tid >> 6] = mt;
        __syncthreads();
        mt = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        ps[tid] = vr >= 0 ? expf(sc - mt) : 0.f;
        const float corr = expf(m - mt);
        m = mt;
        o *= corr;
        l *= corr;
        __syncthreads();
        const int keys = min(KA_THREADS, limit - t0);
        for (int u0 = 0; u0 < keys; u0 += KA_DEEP) {      // (a key behind the last one has no row and weight 0)
            float x[KA_DEEP];
#pragma unroll
            for (int i = 0; i < KA_DEEP; i++) x[i] = (float)vb[max(vrow[u0 + i], (int64_t)0) + min(tid, D - 1)];
#pragma unroll
            for (int i = 0; i < KA_DEEP; i++) x[i] = vrow[u0 + i] >= 0 ? x[i] : 0.f;
#pragma unroll
            for (int i = 0; i < KA_DEEP; i++) {
                l += ps[u0 + i];
                o = fmaf(ps[u0 + i], x[i], o);
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

// ------------------------------------------------- the matrix core kernels ----
typedef __fp16 ka_p4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void ka_lds_t;
typedef __attribute__((address_space(3))) ka_p4 ka_lds_p4;

constexpr int KA_Q_EXP = 12;     // fp32 queries over an fp16 cache: the column's largest is 2^12 .. 2^13

// A tile of keys x COLS columns (16 or 32) on v_mfma_*_COLSxCOLS: lane l holds
// column l % COLS and is one of PL = 64 / COLS parts q = l / COLS of it.
//   S^T: accumulator e of part q is key COLS * (e / E) + sub(e % E, q)
//   O^T: NT tiles of COLS dimensions
// A row of the cache is RB bytes in 16-byte chunks. In LDS a tile is RB / 128 blocks of
// KEYS rows of 128 bytes (a copy instruction fills 8 of them: whole lines of 8 rows),
// where slot s of row r holds chunk s ^ swz(r), a permutation of the bits of r above the
// lowest: 16 consecutive rows' reads of one chunk (K) fall into different banks, and so do
// 4 or 8 rows' reads of 4 or 2 neighbouring chunks (V, transposed; the plain bits in order
// would put such rows on the same banks).
template <typename KT, int D, int COLS_>
struct Ka {
    static constexpr bool F16 = sizeof(KT) == 2;
    static constexpr int COLS = COLS_, PL = 64 / COLS;
    static constexpr int KEYS = F16 ? 32 : 16;         // keys of a tile: the depth of fp16's product with V
    static constexpr int E = COLS * COLS / 64;         // accumulators of one COLS x COLS tile
    static constexpr int ST = KEYS / COLS;             // S^T tiles
    static constexpr int NS = ST * E;                  // a lane's scores
    static constexpr int NT = D / COLS;
    static constexpr int RB = D * (int)sizeof(KT), CB = RB / 128;
    static constexpr int NB = KEYS / 8;                // groups of 8 rows: CB copies each of a tile of K (or V)
    static constexpr int NI = NB * CB;
    static constexpr int BLOCK = KEYS * 128, TILE = CB * BLOCK;    // bytes
    static constexpr int QC = RB / 16 / PL;            // operand chunks of a lane in a score
    static constexpr int OP = D + 4;                   // LDS pitch of a column's output (floats)
    typedef typename std::conditional<COLS == 32, ka_v16, ka_f4>::type Acc;
    __device__ static int swz(int r) { return (r << 1 & 4) | (r >> 1 & 2) | (r >> 3 & 1); }
    __device__ static int slot(int r, int chunk) { return (chunk >> 3) * BLOCK + r * 128 + (((chunk & 7) ^ swz(r)) << 4); }
    // where chunk c of a row lies beside the row's chunk 0 (c a multiple of what lanes add): XOR and offset
    static constexpr uint32_t flip(int c) { return (c & 7) << 4; }
    static constexpr uint32_t block(int c) { return (c >> 3) * BLOCK; }
    // row of a COLS x COLS accumulator tile that element e of part q is
    __device__ static int sub(int e, int q) { return COLS == 32 ? 8 * (e >> 2) + 4 * q + (e & 3) : 4 * q + e; }
    // key of score i of part q
    __device__ static int key(int i, int q) { return COLS * (i / E) + sub(i % E, q); }
    // dimension that element e of O^T tile n is in part q. fp32: a lane reads 16 bytes of
    // V at a time, dimensions 4 i .. 4 i + 3 of each 64, so a tile's row i is dimension 4 i + n % 4.
    __device__ static int dim(int n, int e, int q) {
        return F16 ? COLS * n + sub(e, q) : 4 * sub(e, q) + (n & 3) + 64 * (n >> 2);
    }
    __device__ static Acc mfma(ka_h8 a, ka_h8 b, Acc c) {
        if constexpr (COLS == 32) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    __device__ static Acc zero() {
        Acc c;
#pragma unroll
        for (int e = 0; e < E; e++) c[e] = 0.f;
        return c;
    }
};

// A column's query as operands (chunk PL c + q of its row), and the factor of its
// scores (base 2).
template <typename KT, int D, int COLS, int XP>
struct KaQ {
    ka_h8 h[XP][Ka<KT, D, COLS>::QC];
    float cs;
};
template <int D, int COLS>
struct KaQ<float, D, COLS, 1> {
    ka_f4 f[Ka<float, D, COLS>::QC];
    float cs;
};

// q of (row, head); zeros for a column without a row.
template <typename KT, int D, int COLS, int XP>
__device__ __forceinline__ void ka_load_q(const KaArgs& a, int row, int head, bool live, int part, KaQ<KT, D, COLS, XP>& q) {
    using T = Ka<KT, D, COLS>;
    const int64_t at = live ? row * a.q_stride + (int64_t)head * D : 0;
    // (a maximum of scores is one of their products with it; a masked score, -inf, times it is -inf)
    q.cs = fmaxf(fabsf(a.scale) * KA_LOG2E, FLT_MIN);
    const bool neg = a.scale < 0.f;
    if constexpr (!T::F16) {
#pragma unroll
        for (int c = 0; c < T::QC; c++) {
            const int64_t e0 = at + 4 * (T::PL * c + part);
            if (a.q16) {
#pragma unroll
                for (int e = 0; e < 4; e++) q.f[c][e] = (float)((const _Float16*)a.q)[e0 + e];
            } else {
                q.f[c] = *(const ka_f4*)((const float*)a.q + e0);
            }
            if (neg) q.f[c] = -q.f[c];
            if (!live) q.f[c] = ka_f4{0.f, 0.f, 0.f, 0.f};
        }
    } else if constexpr (XP == 1) {
#pragma unroll
        for (int c = 0; c < T::QC; c++) {
            q.h[0][c] = *(const ka_h8*)((const _Float16*)a.q + at + 8 * (T::PL * c + part));
            if (neg) q.h[0][c] = -q.h[0][c];
            if (!live) q.h[0][c] = ka_h8{0, 0, 0, 0, 0, 0, 0, 0};
        }
    } else {
        float x[T::QC][8], most = 0.f, odd = 0.f;
#pragma unroll
        for (int c = 0; c < T::QC; c++) load8<float>((const float*)a.q + at + 8 * (T::PL * c + part), x[c]);
#pragma unroll
        for (int c = 0; c < T::QC; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (!live) x[c][e] = 0.f;
                most = fmaxf(most, fabsf(x[c][e]));
                odd += x[c][e] * 0.f;                  // NaN if any is inf or NaN
            }
        most = ka_max<COLS>(most);
        odd = ka_max<COLS>(odd == 0.f ? 0.f : 1.f);
        int ex = 0;
        if (most > 0.f && most <= FLT_MAX) frexpf(most, &ex);     // most = 2^ex * [0.5, 1)
        ex = KA_Q_EXP + 1 - ex;
#pragma unroll
        for (int c = 0; c < T::QC; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = ldexpf(neg ? -x[c][e] : x[c][e], ex);
                const _Float16 hi = (_Float16)v;
                q.h[0][c][e] = hi;
                q.h[XP - 1][c][e] = (_Float16)(v - (float)hi);
            }
        q.cs = odd > 0.f ? NAN : fmaxf(ldexpf(q.cs, -ex), FLT_MIN);
    }
}

// Operand addresses. A lane's reads of a tile differ in bits that the swizzle
// XORs, so all are (x ^ constant) + base + constant, one instruction from one
// register; opaque in the loop, or the compiler would hold each in a register.
typedef __attribute__((address_space(3))) char ka_lds_c;
// (offsets from the LDS array's own name: with an address of unknown origin the
// compiler waits for every copy in flight before each read)
extern __shared__ __attribute__((aligned(256))) char ka_lds[];
template <typename V>
__device__ __forceinline__ V ka_read(uint32_t at) { return *(const __attribute__((address_space(3))) V*)((ka_lds_c*)ka_lds + at); }
__device__ __forceinline__ uint32_t ka_addr(const char* p) { return (uint32_t)(p - ka_lds); }
__device__ __forceinline__ uint32_t ka_opaque(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
// K: row lane % COLS, chunk part
template <typename KT, int D, int COLS>
__device__ __forceinline__ uint32_t ka_kx(int lane) { return Ka<KT, D, COLS>::slot(lane % COLS, lane / COLS); }
// V, fp16: 16 lanes read 16 dimensions of 4 keys, 8 bytes each; fp32: 4 dimensions of the part's first key
template <typename KT, int D, int COLS>
__device__ __forceinline__ uint32_t ka_vx(int lane) {
    using T = Ka<KT, D, COLS>;
    const int i = lane & 15, part = lane / COLS;
    if constexpr (T::F16) return T::slot(4 * part + (i >> 2), (COLS == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((i >> 1) & 1)) + 8 * (i & 1);
    else return T::slot(4 * part, i);
}

// S^T of one tile: K's operands (rows at kt), all reads in flight together, and the products.
template <typename KT, int D, int COLS>
struct KaKeysOf {
    using T = Ka<KT, D, COLS>;
    typedef typename std::conditional<T::F16, ka_h8, ka_f4>::type K;
    K k[T::ST][T::QC];
    __device__ __forceinline__ void read(uint32_t kt, uint32_t kx) {
        kx = ka_opaque(kx);
#pragma unroll
        for (int st = 0; st < T::ST; st++)
#pragma unroll
            for (int i = 0; i < T::QC; i++)
                k[st][i] = ka_read<K>((kx ^ T::flip(T::PL * i)) + kt + T::block(T::PL * i) + st * COLS * 128);
    }
};
template <typename KT, int D, int COLS, int XP>
__device__ __forceinline__ void ka_scores(const KaKeysOf<KT, D, COLS>& k, const KaQ<KT, D, COLS, XP>& q,
                                          float (&s)[Ka<KT, D, COLS>::NS]) {
    using T = Ka<KT, D, COLS>;
#pragma unroll
    for (int st = 0; st < T::ST; st++) {
        if constexpr (T::F16) {
            typename T::Acc c = T::zero();
#pragma unroll
            for (int i = 0; i < T::QC; i++) {
                c = T::mfma(k.k[st][i], q.h[0][i], c);
                if constexpr (XP == 2) c = T::mfma(k.k[st][i], q.h[XP - 1][i], c);
            }
#pragma unroll
            for (int e = 0; e < T::E; e++) s[st * T::E + e] = c[e];
        } else {
            ka_f4 c[4];                // 4 chains: half the rounding of one, and the MFMAs need not wait for each other
#pragma unroll
            for (int ch = 0; ch < 4; ch++) c[ch] = T::zero();
#pragma unroll
            for (int i = 0; i < T::QC; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) c[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.k[st][i][e], q.f[i][e], c[e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] = (c[0][e] + c[1][e]) + (c[2][e] + c[3][e]);
        }
    }
}

// Pairs of transposed reads, OFF bytes apart, from each address, and the wait for them in
// one piece: the compiler cannot tell what a transposed read does not alias, and would wait
// for every copy in flight before the first (a round trip to memory in every tile).
template <int OFF>
__device__ __forceinline__ void ka_read_tr(const uint32_t (&a)[4], ka_p4 (&r)[4][2]) {
    asm volatile("ds_read_b64_tr_b16 %0, %8\n ds_read_b64_tr_b16 %1, %8 offset:%12\n"
                 "ds_read_b64_tr_b16 %2, %9\n ds_read_b64_tr_b16 %3, %9 offset:%12\n"
                 "ds_read_b64_tr_b16 %4, %10\n ds_read_b64_tr_b16 %5, %10 offset:%12\n"
                 "ds_read_b64_tr_b16 %6, %11\n ds_read_b64_tr_b16 %7, %11 offset:%12\n"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[2][0]), "=&v"(r[2][1]),
                   "=&v"(r[3][0]), "=&v"(r[3][1])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF));
}
template <int OFF>
__device__ __forceinline__ void ka_read_tr(const uint32_t (&a)[8], ka_p4 (&r)[8][2]) {
    asm volatile("ds_read_b64_tr_b16 %0, %16\n ds_read_b64_tr_b16 %1, %16 offset:%24\n"
                 "ds_read_b64_tr_b16 %2, %17\n ds_read_b64_tr_b16 %3, %17 offset:%24\n"
                 "ds_read_b64_tr_b16 %4, %18\n ds_read_b64_tr_b16 %5, %18 offset:%24\n"
                 "ds_read_b64_tr_b16 %6, %19\n ds_read_b64_tr_b16 %7, %19 offset:%24\n"
                 "ds_read_b64_tr_b16 %8, %20\n ds_read_b64_tr_b16 %9, %20 offset:%24\n"
                 "ds_read_b64_tr_b16 %10, %21\n ds_read_b64_tr_b16 %11, %21 offset:%24\n"
                 "ds_read_b64_tr_b16 %12, %22\n ds_read_b64_tr_b16 %13, %22 offset:%24\n"
                 "ds_read_b64_tr_b16 %14, %23\n ds_read_b64_tr_b16 %15, %23 offset:%24\n"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[2][0]), "=&v"(r[2][1]),
                   "=&v"(r[3][0]), "=&v"(r[3][1]), "=&v"(r[4][0]), "=&v"(r[4][1]), "=&v"(r[5][0]), "=&v"(r[5][1]),
                   "=&v"(r[6][0]), "=&v"(r[6][1]), "=&v"(r[7][0]), "=&v"(r[7][1])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "n"(OFF));
}

// V^T of one tile as operands (rows at vt): of O^T tile n and key group kc, a lane's 8
// values of one dimension, the keys of scores 8 kc .. 8 kc + 7.
template <int D, int COLS>
struct KaValuesOf {
    using T = Ka<_Float16, D, COLS>;
    static constexpr int KC = T::NS / 8;
    ka_h8 v[T::NT][KC];
    __device__ __forceinline__ void read(uint32_t vt, uint32_t vx) {
        vx = ka_opaque(vx);
        // 16 lanes read 16 dimensions of 4 keys. 32 columns: an operand's second 4 keys are 8 rows on, with another
        // swizzle, the second key group 16; 16 columns: the second 4 keys 16 rows on
        constexpr int B = COLS == 32 ? 2 : 1;
        uint32_t a[T::NT * B];
        ka_p4 r[T::NT * B][2];
#pragma unroll
        for (int n = 0; n < T::NT; n++)
#pragma unroll
            for (int b = 0; b < B; b++)
                a[n * B + b] = (vx ^ (T::flip(COLS / 8 * n) ^ (b << 4))) + vt + T::block(COLS / 8 * n) + 8 * b * 128;
#pragma unroll
        for (int i = 0; i < T::NT * B; i++) a[i] += (uint32_t)(uintptr_t)(ka_lds_c*)ka_lds;
        ka_read_tr<16 * 128>(a, r);
#pragma unroll
        for (int n = 0; n < T::NT; n++)
#pragma unroll
            for (int kc = 0; kc < KC; kc++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[n][kc][e] = (_Float16)(B == 2 ? r[2 * n][kc] : r[n][0])[e];
                    v[n][kc][4 + e] = (_Float16)(B == 2 ? r[2 * n + 1][kc] : r[n][1])[e];
                }
    }
};

// A column's running softmax: (reference, sum) in base 2, O^T.
template <typename KT, int D, int COLS>
struct KaAcc {
    float m, l;
    typename Ka<KT, D, COLS>::Acc o[Ka<KT, D, COLS>::NT];
    __device__ void clear() {
        m = -FLT_MAX;
        l = 0.f;
#pragma unroll
        for (int n = 0; n < Ka<KT, D, COLS>::NT; n++) o[n] = Ka<KT, D, COLS>::zero();
    }
};

// Scores -> weights (in s), and the running reference and sum, in steps. The tile's
// keys from t0; edge (wave-uniform): some column does not see all of them.
//   1. what a column does not see is -inf; its maximum
template <typename KT, int D, int COLS>
__device__ __forceinline__ void ka_mask(int t0, int limit, int part, float (&s)[Ka<KT, D, COLS>::NS]) {
    using T = Ka<KT, D, COLS>;
    const int left = ka_opaque(limit - t0 - T::key(0, part));
#pragma unroll
    for (int e = 0; e < T::NS; e++) s[e] = T::key(e, 0) < left ? s[e] : -INFINITY;
}
template <typename KT, int D, int COLS>
__device__ __forceinline__ float ka_top(const float (&s)[Ka<KT, D, COLS>::NS], float cs, int t0, int limit) {
    float top = s[0];
#pragma unroll
    for (int e = 1; e < Ka<KT, D, COLS>::NS; e++) top = fmaxf(top, s[e]);
    return ka_max<COLS>(fmaxf(top * cs, t0 < limit ? KA_SEEN : -FLT_MAX));
}
//   2. the reference, where the maximum has grown enough
template <typename KT, int D, int COLS>
__device__ __forceinline__ void ka_follow(KaAcc<KT, D, COLS>& x, float top) {
    using T = Ka<KT, D, COLS>;
    if (__any(top > x.m + KA_SLACK)) {
        const float m = fmaxf(x.m, top), corr = __builtin_amdgcn_exp2f(x.m - m);
        x.l *= corr;
#pragma unroll
        for (int n = 0; n < T::NT; n++)
#pragma unroll
            for (int e = 0; e < T::E; e++) x.o[n][e] *= corr;
        x.m = m;
    }
}
//   3. the weights
template <typename KT, int D, int COLS>
__device__ __forceinline__ void ka_weights(KaAcc<KT, D, COLS>& x, float (&s)[Ka<KT, D, COLS>::NS], float cs) {
    using T = Ka<KT, D, COLS>;
    const float base = (T::F16 ? KA_LIFT : 0.f) - x.m;
    float sum[T::NS];
#pragma unroll
    for (int e = 0; e < T::NS; e++) {
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], cs, base));
        sum[e] = s[e];
    }
#pragma unroll
    for (int n = T::NS / 2; n >= 1; n >>= 1)
#pragma unroll
        for (int e = 0; e < n; e++) sum[e] += sum[e + n];
    x.l += sum[0];
}

// fp16 weights as operands, in XP parts.
template <int D, int COLS, int XP>
struct KaWeights {
    static constexpr int KC = KaValuesOf<D, COLS>::KC;
    ka_h8 w[KC][XP];
    __device__ __forceinline__ void pack(const float (&p)[8 * KC]) {
#pragma unroll
        for (int kc = 0; kc < KC; kc++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const _Float16 hi = (_Float16)p[8 * kc + e];
                w[kc][0][e] = hi;
                if constexpr (XP == 2) w[kc][XP - 1][e] = (_Float16)(p[8 * kc + e] - (float)hi);
            }
    }
    // computed where this stands: the compiler would sink it behind the next branch
    __device__ __forceinline__ void here() {
#pragma unroll
        for (int kc = 0; kc < KC; kc++)
#pragma unroll
            for (int i = 0; i < XP; i++) asm volatile("" : "+v"(w[kc][i]));
    }
};

// O^T += V^T P^T over one tile. In a tile that some column does not see all of, a value
// of inf or NaN would make that column NaN, 0 * inf: such values are left out (ka_finite,
// for fp16; it returns whether there were any, in every lane), and ka_mend adds them to
// the columns that see them.
template <int D, int COLS>
__device__ __forceinline__ bool ka_finite(KaValuesOf<D, COLS>& vs) {
    using T = Ka<_Float16, D, COLS>;
    constexpr int KC = KaValuesOf<D, COLS>::KC;
    ka_h8 z = {0, 0, 0, 0, 0, 0, 0, 0};        // stays 0, but for inf and NaN
#pragma unroll
    for (int n = 0; n < T::NT; n++)
#pragma unroll
        for (int kc = 0; kc < KC; kc++) z = vs.v[n][kc] * (_Float16)0 + z;
    bool any = false;
#pragma unroll
    for (int e = 0; e < 8; e++) any |= z[e] != z[e];
    if (!__any(any)) return false;
#pragma unroll
    for (int n = 0; n < T::NT; n++)
#pragma unroll
        for (int kc = 0; kc < KC; kc++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const _Float16 v = vs.v[n][kc][e];
                vs.v[n][kc][e] = v * (_Float16)0 == (_Float16)0 ? v : (_Float16)0;
            }
    return true;
}
template <int D, int COLS, int XP>
__device__ __forceinline__ void ka_product(KaAcc<_Float16, D, COLS>& x, const KaWeights<D, COLS, XP>& w,
                                           const KaValuesOf<D, COLS>& vs) {
    using T = Ka<_Float16, D, COLS>;
#pragma unroll
    for (int kc = 0; kc < KaValuesOf<D, COLS>::KC; kc++)
#pragma unroll
        for (int n = 0; n < T::NT; n++)
#pragma unroll
            for (int i = 0; i < XP; i++) x.o[n] = T::mfma(vs.v[n][kc], w.w[kc][i], x.o[n]);
}
template <typename KT, int D, int COLS, int XP>
__device__ __forceinline__ bool ka_values(KaAcc<KT, D, COLS>& x, const float (&p)[Ka<KT, D, COLS>::NS], uint32_t vt,
                                          uint32_t vx, bool edge) {
    using T = Ka<KT, D, COLS>;
    bool odd = false;
    if constexpr (T::F16) {
        KaValuesOf<D, COLS> vs;
        vs.read(vt, vx);
        if (edge) odd = ka_finite<D, COLS>(vs);
        KaWeights<D, COLS, XP> w;
        w.pack(p);
        ka_product<D, COLS, XP>(x, w, vs);
    } else {
        vx = ka_opaque(vx);
        ka_f4 v[T::NS][T::NT / 4];             // 4 dimensions of the key of each score
#pragma unroll
        for (int e = 0; e < T::NS; e++)
#pragma unroll
            for (int half = 0; half < T::NT / 4; half++)
                v[e][half] = ka_read<ka_f4>((vx ^ ((e & 2) << 5)) + vt + T::block(16 * half) + e * 128);
        if (edge) {
            ka_f4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < T::NS; e++)
#pragma unroll
                for (int half = 0; half < T::NT / 4; half++) z = v[e][half] * 0.f + z;
            odd = __any(!((z[0] + z[1]) + (z[2] + z[3]) == 0.f));
            if (odd) {
#pragma unroll
                for (int e = 0; e < T::NS; e++)
#pragma unroll
                    for (int half = 0; half < T::NT / 4; half++)
#pragma unroll
                        for (int n = 0; n < 4; n++) v[e][half][n] = fabsf(v[e][half][n]) <= FLT_MAX ? v[e][half][n] : 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < T::NS; e++)
#pragma unroll
            for (int n = 0; n < T::NT; n++)
                x.o[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e][n >> 2][n & 3], p[e], x.o[n], 0, 0, 0);
    }
    return odd;
}

// A lane's part of an accumulated column, times f, into LDS (column's row at `to`),
// or added to what is there.
template <typename KT, int D, int COLS, bool ADD>
__device__ __forceinline__ void ka_spill(const KaAcc<KT, D, COLS>& x, float f, float* to, int part) {
    using T = Ka<KT, D, COLS>;
#pragma unroll
    for (int n = 0; n < T::NT; n += T::F16 ? 1 : 4)
#pragma unroll
        for (int e = 0; e < T::E; e += T::F16 ? 4 : 1) {
            ka_f4 v;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = (T::F16 ? x.o[n][e + j] : x.o[n + j][e]) * f;
            ka_f4* at = (ka_f4*)(to + T::dim(n, e, part));
            *at = ADD ? *at + v : v;
        }
}

// Where a layer's K of kv head g begins (V: a plane behind it).
template <int RB>
__device__ __forceinline__ const char* ka_base(const KaArgs& a, int g) {
    const pio_kv_cache& c = a.c;
    return (const char*)c.kv + (((int64_t)2 * a.layer * c.n_pages * c.n_kv_heads + g) * c.page_size) * RB;
}
template <int RB>
__device__ __forceinline__ int64_t ka_plane(const KaArgs& a) {
    return (int64_t)a.c.n_pages * a.c.n_kv_heads * a.c.page_size * RB;
}

// inf and NaN values that ka_values left out, added to 4 dimensions from d of column
// `col` (of the item) with limit `limit`, out of the keys from `from` on.
template <typename KT, int D>
__device__ __forceinline__ void ka_mend(const KaArgs& a, const KaItem& it, int from, int limit, int d, ka_f4& v) {
    const pio_kv_cache& c = a.c;
    constexpr int RB = D * (int)sizeof(KT);
    const int lg = kv_log2(c.page_size);
    const KT* vb = (const KT*)(ka_base<RB>(a, it.g) + ka_plane<RB>(a));
    for (int t = max(from, it.k0); t < min(limit, it.k1); t++) {
        const int page = it.table[t >> lg];
        if (page < 0 || page >= c.n_pages) continue;
        const KT* r = vb + ((int64_t)page * c.n_kv_heads * c.page_size + (t & (c.page_size - 1))) * D + d;
        for (int e = 0; e < 4; e++)
            if (!(fabsf((float)r[e]) <= FLT_MAX)) v[e] += (float)r[e];
    }
}
// ---- narrow items: 4 waves, 16 columns, every 4th tile of the keys each, from a
// piece of LDS of the wave's own (one tile of K, one of V). The next K tile is
// copied during this one's softmax and product with V, the next V tile during the
// next scores. No barriers: a wave waits for its own copies.
//   16 columns and not 32: few queries to a request leave the rest of a tile empty, and the
// 16 x 16 products read K and V at the same rate. Two workgroups to a CU (64 KB of LDS each at
// fp16 x 128). Long tails are bound by HBM: 8 sequences of 20,000 tokens (8 kv heads x 128,
// fp16) 24.4 us, 4.1 TB/s; short ones by an item's chain of waits (its requests, a page, K, the
// join), some 12,000 clocks: 32 sequences behind 2,039 tokens 15.3 us, 2.1 TB/s.
constexpr int KA_COLS = 16, KA_WAVES = 4;

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

template <typename KT, int D>
struct KaWalk {
    using T = Ka<KT, D, KA_COLS>;
    const char *kb, *vb;
    char *kt, *vt;
    int tiles, per_page, lg, mask;
    int page, key;                         // this lane's key of the next tile, and its page's id, unchecked
    int64_t off[T::NB];
    int bad_at = INT_MAX;                  // first key of this lane in a page outside the cache
    bool odd = false;

    // (keys behind the last one re-read it)
    __device__ void look_up(const KaItem& it, int j, int lane) {
        key = min(it.k0 + min(j, tiles - 1) * T::KEYS + lane % T::KEYS, it.k1 - 1);
        page = it.table[key >> lg];
    }
    // Where this lane's 16 bytes of each 8 rows are: rows lane / 8 of them.
    __device__ void offsets(const KaArgs& a, int lane) {
        const bool ok = page >= 0 && page < a.c.n_pages;
        bad_at = ok ? bad_at : min(bad_at, key);
        const uint32_t row = (uint32_t)(ok ? page : 0) * (uint32_t)per_page + (uint32_t)(key & mask);
        int r[T::NB];
#pragma unroll
        for (int i = 0; i < T::NB; i++) r[i] = __shfl((int)row, 8 * i + lane / 8, 64);
#pragma unroll
        for (int i = 0; i < T::NB; i++)
            off[i] = (int64_t)(uint32_t)r[i] * T::RB + (((lane & 7) ^ T::swz(8 * i + lane / 8)) << 4);
    }
    __device__ void copy(const char* from, char* to) {
#pragma unroll
        for (int i = 0; i < T::NB; i++)
#pragma unroll
            for (int cb = 0; cb < T::CB; cb++)
                __builtin_amdgcn_global_load_lds((const void*)(from + off[i] + 128 * cb),
                                                 (ka_lds_t*)(to + cb * T::BLOCK + i * 1024), 16, 0, 0);
    }
    // The first tile's copies, if the wave has one.
    __device__ void begin(const KaArgs& a, const KaItem& it, char* mine, int w, int lane) {
        lg = kv_log2(a.c.page_size);
        mask = a.c.page_size - 1;
        per_page = a.c.n_kv_heads * a.c.page_size;
        kb = ka_base<T::RB>(a, it.g);
        vb = kb + ka_plane<T::RB>(a);
        kt = mine;
        vt = mine + T::TILE;
        tiles = (it.k1 - it.k0 + T::KEYS - 1) / T::KEYS;
        if (w >= tiles) return;
        look_up(it, w, lane);
        offsets(a, lane);
        look_up(it, w + KA_WAVES, lane);
        copy(kb, kt);
        copy(vb, vt);
    }
    template <int XP>
    __device__ void run(const KaArgs& a, const KaItem& it, int w, int lane, int limit, int row, int head, bool has,
                        KaAcc<KT, D, KA_COLS>& x) {
        if (w >= tiles) return;
        const int part = lane / KA_COLS;
        KaQ<KT, D, KA_COLS, XP> q;
        ka_load_q<KT, D, KA_COLS, XP>(a, row, head, has, part, q);
        const int least = ka_wave_min(limit);
        const uint32_t kx = ka_kx<KT, D, KA_COLS>(lane), vx = ka_vx<KT, D, KA_COLS>(lane);
        ka_wait_copies<0>();               // the query too: below only copies and one page id are counted
        for (int j = w; j < tiles; j += KA_WAVES) {
            const int t0 = it.k0 + j * T::KEYS;
            const bool more = j + KA_WAVES < tiles, edge = t0 + T::KEYS > least;
            ka_wait_copies<T::NI>();
            float s[T::NS];
            KaKeysOf<KT, D, KA_COLS> k;
            k.read(ka_addr(kt), kx);
            ka_scores<KT, D, KA_COLS, XP>(k, q, s);
            ka_wait_reads();
            if (more) {
                offsets(a, lane);
                copy(kb, kt);
                look_up(it, j + 2 * KA_WAVES, lane);      // (used in the next round: not waited for here)
            }
            if (edge) ka_mask<KT, D, KA_COLS>(t0, limit, part, s);
            ka_follow<KT, D, KA_COLS>(x, ka_top<KT, D, KA_COLS>(s, q.cs, t0, limit));
            ka_weights<KT, D, KA_COLS>(x, s, q.cs);
            if (more) ka_wait_copies<T::NI + 1>();
            else ka_wait_copies<0>();
            odd |= ka_values<KT, D, KA_COLS, XP>(x, s, ka_addr(vt), vx, edge);
            ka_wait_reads();
            if (more) copy(vb, vt);
        }
    }
};

template <typename KT, int D>
constexpr size_t ka_narrow_bytes() {
    using T = Ka<KT, D, KA_COLS>;
    return std::max<size_t>(KA_WAVES * 2 * T::TILE, (size_t)KA_WAVES * KA_COLS * T::OP * 4);
}

// An item's 16 columns from c0 joined over its waves and written.
template <typename KT, int D>
__device__ __forceinline__ void ka_join(const KaArgs& a, const KaItem& it, KaAcc<KT, D, KA_COLS>& x, char* lds,
                                        float (*ml)[KA_COLS][2], int w, int lane, bool bad, bool odd, int c0,
                                        const int* limits) {
    using T = Ka<KT, D, KA_COLS>;
    const int col = lane % KA_COLS, part = lane / KA_COLS;
    x.l += __shfl_xor(x.l, 32, 64);
    x.l += __shfl_xor(x.l, 16, 64);
    if (bad) x.l = NAN;
    if (part == 0) {
        ml[w][col][0] = x.m;
        ml[w][col][1] = x.l;
    }
    odd = __syncthreads_or(odd);           // and every wave is done with its tiles
    float mx = ml[0][col][0];
#pragma unroll
    for (int i = 1; i < KA_WAVES; i++) mx = fmaxf(mx, ml[i][col][0]);
    ka_spill<KT, D, KA_COLS, false>(x, __builtin_amdgcn_exp2f(x.m - mx), (float*)lds + (w * KA_COLS + col) * T::OP, part);
    __syncthreads();
    for (int i = w * 64 + lane; i < min(KA_COLS, it.ncols - c0) * (D / 4); i += 64 * KA_WAVES) {
        const int c = i / (D / 4), d = (i % (D / 4)) * 4;
        float m = ml[0][c][0], l = 0.f;
#pragma unroll
        for (int k = 1; k < KA_WAVES; k++) m = fmaxf(m, ml[k][c][0]);
        ka_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KA_WAVES; k++) {
            v += *(const ka_f4*)((const float*)lds + (k * KA_COLS + c) * T::OP + d);
            l += ml[k][c][1] * __builtin_amdgcn_exp2f(ml[k][c][0] - m);
        }
        if (odd) {
            const int first = ka_div(a, c0);
            ka_mend<KT, D>(a, it, limits ? it.k0 : it.first_limit + first - T::KEYS, ka_limit(it, limits, first, ka_div(a, c0 + c)), d, v);
        }
        ka_emit(a, D, it, c0 + c, d, v, m, l);
    }
}

// A narrow item; limits: of a prefix's rows, from c0 / G.
template <typename KT, int D, int XP>
__device__ __forceinline__ void ka_narrow(const KaArgs& a, const KaItem& it, float (*ml)[KA_COLS][2], int* limits, int c0,
                                          int w, int lane) {
    using T = Ka<KT, D, KA_COLS>;
    KaAcc<KT, D, KA_COLS> acc;
    acc.clear();
    KaWalk<KT, D> walk;
    walk.begin(a, it, ka_lds + w * 2 * T::TILE, w, lane);
    if (limits) ka_limits(a, ka_div(a, c0), limits, KA_COLS);     // under the first copies' way
    const int col = c0 + lane % KA_COLS;
    const bool has = col < it.ncols;
    const int r = has ? ka_div(a, col) : 0, head = it.g * a.G + (has ? col - r * a.G : 0);
    const int limit = has ? ka_limit(it, limits, ka_div(a, c0), r) : it.k1;
    walk.template run<XP>(a, it, w, lane, limit, it.row0 + r, head, has, acc);
    // a page outside the cache: NaN for the columns that see its keys
    bool bad = it.bad, told = it.bad;
    if (__any(walk.bad_at != INT_MAX)) {
        const int first_bad = ka_wave_min(walk.bad_at);
        bad |= limit > first_bad;
        told |= has && (limits ? limits[r - ka_div(a, c0)] : it.first_limit + r) > first_bad;    // (a row without a request: -1)
    }
    if (told) atomicOr(a.c.work, KV_BAD);
    ka_join<KT, D>(a, it, acc, ka_lds, ml, w, lane, bad, walk.odd, c0, limits);
}

// ---- wide items: 8 waves, 128 columns: 4 tiles of 32 by waves w % 4, the halves of every
// 64 keys by waves w / 4. K and V of 64 keys are one of KA_STAGES stages in LDS that the
// waves copy together, so that they cross from L2 once for 128 columns. Bound by the waves'
// own work between two barriers, 2,700 clocks a stage: the matrix cores have 1,024 of it, the
// VALU 1,600, LDS 1,300. 512 columns over 32,000 tokens (4 kv heads x 128): 53 us, 630 TFLOP/s,
// 10 of it an item's first and last 20,000 clocks; 4 x as many columns 700 TFLOP/s. Tried
// and no faster: 4 waves of 64 columns with all registers of a SIMD each (the accumulators move
// between register files), the second half's waves half a stage behind the first's, products
// and exponentials interleaved by hand.
constexpr int KA_WIDE_COLS = 128, KA_WIDE_KEYS = 64, KA_STAGES = 4, KA_WIDE_PAGES = 4096;
template <int D>
constexpr size_t ka_wide_bytes() {
    return std::max<size_t>((size_t)KA_STAGES * 2 * KA_WIDE_KEYS * D * 2, (size_t)KA_WIDE_COLS * (D + 4) * 4);
}

template <int D>
constexpr size_t ka_wide_lds() {
    return ka_wide_bytes<D>() + KA_WIDE_PAGES * sizeof(int);
}

template <int D, int XP>
__device__ __forceinline__ void ka_wide(const KaArgs& a, const KaItem& it, char* lds, int* pages,
                                        float (*ml)[32][2], int* limits, int base) {
    typedef _Float16 KT;
    using T = Ka<KT, D, 32>;
    const pio_kv_cache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), cg = w & 3, kg = w >> 2;
    const int col = lane & 31, h = lane >> 5;
    const int lg = kv_log2(c.page_size), mask = c.page_size - 1, per_page = c.n_kv_heads * c.page_size;
    const int first = ka_div(a, base), cc = base + cg * 32 + col;
    const bool has = cc < it.ncols;
    const int r = has ? ka_div(a, cc) : 0, head = it.g * a.G + (has ? cc - r * a.G : 0);
    KaQ<KT, D, 32, XP> q;
    KaAcc<KT, D, 32> x;
    x.clear();
    int limit = it.k1, least = it.k1;
    int bad_at = it.bad ? INT_MIN : INT_MAX;       // first key in a page outside the cache
    bool odd = false;
    const uint32_t kx = ka_kx<KT, D, 32>(lane), vx = ka_vx<KT, D, 32>(lane);

    const char* kb = ka_base<T::RB>(a, it.g);
    const char* vb = kb + ka_plane<T::RB>(a);
    constexpr int STAGE = 2 * KA_WIDE_KEYS * T::RB, PW = T::CB;        // copies of a wave: PW of K, PW of V
    const int chunk = (KA_WIDE_PAGES - 1) * c.page_size / KA_WIDE_KEYS * KA_WIDE_KEYS;
    for (int k0 = it.k0; k0 < it.k1; k0 += chunk) {    // as many keys as page ids fit
        const int k1 = min(it.k1 - k0, chunk) + k0, p0 = k0 >> lg, np = ((k1 - 1) >> lg) - p0 + 1;
        int page = tid < np ? it.table[p0 + tid] : 0;
        if (k0 != it.k0) __syncthreads();
        // under its way; limits: of the rows from `first` (prefix), else by first_limit
        else if (limits) ka_limits(a, first, limits, KA_WIDE_COLS);
        for (int i = tid; i < np; i += 512) {
            if (i != tid) page = it.table[p0 + i];
            if (page < 0 || page >= c.n_pages) {
                bad_at = min(bad_at, max(k0, (p0 + i) << lg));
                page = 0;
            }
            pages[i] = page;
        }
        __syncthreads();
        // stage s: its rows 8 w .. 8 w + 7 (keys behind the last one re-read it), those of tile w / 4
        auto place = [&](int s) {
            const int t = min(k0 + s * KA_WIDE_KEYS + 8 * w + lane / 8, k1 - 1);
            return (uint32_t)pages[(t >> lg) - p0] * (uint32_t)per_page + (uint32_t)(t & mask);
        };
        auto copy = [&](int s, uint32_t at, int kind) {        // K (0) or V (1)
            const char* from = (kind ? vb : kb) + (int64_t)at * T::RB + (((lane & 7) ^ T::swz(8 * cg + lane / 8)) << 4);
            char* to = lds + (s % KA_STAGES) * STAGE + kind * KA_WIDE_KEYS * T::RB + kg * T::TILE + cg * 1024;
#pragma unroll
            for (int cb = 0; cb < T::CB; cb++)
                __builtin_amdgcn_global_load_lds((const void*)(from + 128 * cb), (ka_lds_t*)(to + cb * T::BLOCK), 16, 0, 0);
        };
        const int stages = (k1 - k0 + KA_WIDE_KEYS - 1) / KA_WIDE_KEYS;
        ka_wait_copies<0>();
#pragma unroll
        for (int s = 0; s < KA_STAGES - 1; s++) {
            copy(s, place(s), 0);
            copy(s, place(s), 1);
        }
        // The scores run one stage ahead of the softmax: their products fill the matrix cores
        // while the exponentials fill the VALU. (A workgroup's waves pass the barriers together,
        // and so do not cover each other.) Two parts of 128 dimensions leave no registers for it.
        constexpr bool AHEAD = XP == 1 || D < 128;
        uint32_t at = place(3);
        if constexpr (AHEAD) copy(3, at, 0);
        if (k0 == it.k0) {
            if (has) limit = ka_limit(it, limits, first, r);
            least = ka_wave_min(limit);
            ka_load_q<KT, D, 32, XP>(a, it.row0 + r, head, has, h, q);
            ka_wait_copies<0>();           // q is here: the waits below count copies alone
        }
        const int end = min(limit, k1);    // (a chunk's end is not the item's: keys behind it come with the next chunk)
        auto tile = [&](int s) { return ka_addr(lds + (s % KA_STAGES) * STAGE + kg * T::TILE); };
        auto first_key = [&](int s) { return k0 + s * KA_WIDE_KEYS + kg * T::KEYS; };
        auto edge = [&](int s) { return first_key(s) + T::KEYS > min(least, k1); };
        KaKeysOf<KT, D, 32> k;
        KaValuesOf<D, 32> v;
        KaWeights<D, 32, XP> wt;
        float sc[T::NS], top;
        auto masked_top = [&](int s) {
            if (edge(s)) ka_mask<KT, D, 32>(first_key(s), end, h, sc);
            top = ka_top<KT, D, 32>(sc, q.cs, first_key(s), end);
        };
        if constexpr (AHEAD) {
            // K of stage s + 2 is read into registers beside the products of stage s with V, so that LDS
            // and the matrix cores work at one time. So K's places are free two stages before V's.
            uint32_t at1 = place(4), at2 = place(5);
            stage_barrier<0>();
            k.read(tile(0), kx);
            ka_scores<KT, D, 32, XP>(k, q, sc);
            masked_top(0);
            k.read(tile(1), kx);
            stage_barrier<0>();
            copy(4, at1, 0);
            for (int s = 0; s < stages; s++) {
                // K of stage s + 2 and V of stage s have landed; read by all: K up to s + 1, V up to s - 1
                stage_barrier<4 * PW>();
                copy(s + 5, at2, 0);               // (past the end the last key again)
                copy(s + 3, at, 1);
                ka_follow<KT, D, 32>(x, top);
                const uint32_t vt = tile(s) + KA_WIDE_KEYS * T::RB;
                v.read(vt, vx);
                if (edge(s)) odd |= ka_finite<D, 32>(v);
                float next[T::NS];
                ka_weights<KT, D, 32>(x, sc, q.cs);
                wt.pack(sc);
                ka_scores<KT, D, 32, XP>(k, q, next);
#pragma unroll
                for (int i = 0; i < T::QC * XP; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                   // a product
                    __builtin_amdgcn_sched_group_barrier(0x402, 64 / (T::QC * XP), 0);   // its share of the VALU's work
                }
                wt.here();
#pragma unroll
                for (int e = 0; e < T::NS; e++) sc[e] = next[e];
                k.read(tile(s + 2), kx);
                ka_product<D, 32, XP>(x, wt, v);
                at = at1;
                at1 = at2;
                at2 = place(s + 6);
                masked_top(s + 1);
            }
        } else {
            for (int s = 0; s < stages; s++) {
                stage_barrier<(KA_STAGES - 2) * 2 * PW>();
                k.read(tile(s), kx);
                // into the stage that every wave has read before this barrier
                copy(s + 3, at, 0);
                copy(s + 3, at, 1);
                ka_scores<KT, D, 32, XP>(k, q, sc);
                masked_top(s);
                ka_follow<KT, D, 32>(x, top);
                ka_weights<KT, D, 32>(x, sc, q.cs);
                odd |= ka_values<KT, D, 32, XP>(x, sc, tile(s) + KA_WIDE_KEYS * T::RB, vx, edge(s));
                at = place(s + 4);
            }
        }
    }
    ka_wait_copies<0>();                   // those past the end too: the stages are overwritten
    // the halves of the keys meet in LDS
    x.l += __shfl_xor(x.l, 32, 64);
    if (h == 0) {
        ml[w][col][0] = x.m;
        ml[w][col][1] = x.l;
    }
    const bool any_bad = __syncthreads_or(bad_at != INT_MAX);      // and every stage is read
    odd = __syncthreads_or(odd);
    if (any_bad) {                         // NaN for the columns that see it
        if (tid == 0) pages[0] = INT_MAX;
        __syncthreads();
        atomicMin(pages, bad_at);
        __syncthreads();
        bad_at = pages[0];
        if (tid < min(KA_WIDE_COLS, it.ncols - base)) {
            const int row = ka_div(a, base + tid);
            if ((limits ? limits[row - first] : it.first_limit + row) > bad_at) atomicOr(c.work, KV_BAD);   // (a row without a request: -1)
        }
    }
    const float f = __builtin_amdgcn_exp2f(x.m - fmaxf(ml[cg][col][0], ml[cg + 4][col][0]));
    float* ob = (float*)lds + (cg * 32 + col) * T::OP;
    if (kg) ka_spill<KT, D, 32, false>(x, f, ob, h);
    __syncthreads();
    if (!kg) ka_spill<KT, D, 32, true>(x, f, ob, h);
    __syncthreads();
    const int out = min(KA_WIDE_COLS, it.ncols - base) * (D / 4);
    auto emit = [&](int i, bool mend) {
        const int cc = i / (D / 4), d = (i % (D / 4)) * 4;
        const float m0 = ml[cc >> 5][cc & 31][0], m1 = ml[4 + (cc >> 5)][cc & 31][0], m = fmaxf(m0, m1);
        float l = ml[cc >> 5][cc & 31][1] * __builtin_amdgcn_exp2f(m0 - m) +
                  ml[4 + (cc >> 5)][cc & 31][1] * __builtin_amdgcn_exp2f(m1 - m);
        if (any_bad && ka_limit(it, limits, first, ka_div(a, base + cc)) > bad_at) l = NAN;
        ka_f4 v = *(const ka_f4*)((const float*)lds + cc * T::OP + d);
        if (mend)
            ka_mend<KT, D>(a, it, limits ? it.k0 : it.first_limit + first - T::KEYS, ka_limit(it, limits, first, ka_div(a, base + cc)), d, v);
        ka_emit(a, D, it, base + cc, d, v, m, l);
    };
    if (odd) {
        for (int i = tid; i < out; i += 512) emit(i, true);
    } else {
#pragma unroll 4
        for (int i = tid; i < out; i += 512) emit(i, false);
    }
}

// The prefix's items, then the tails'.
//   WIDE 0: narrow items, workgroups of 4 waves
//   WIDE 1: wide items of the prefix alone, workgroups of 8 waves
//   WIDE 2: wide items, workgroups of 8 waves
template <typename KT, int D, int XP, int WIDE>
__global__ __launch_bounds__(WIDE ? 512 : 256, 2) void ka_kernel(KaArgs a) {
    constexpr int WAVES = WIDE ? 8 : KA_WAVES;
    __shared__ float ml[WIDE ? 8 * 32 * 2 : 4 * KA_COLS * 2];
    __shared__ int limits[WIDE ? KA_WIDE_COLS : KA_COLS];
    __shared__ KaRun found;
    __shared__ int red[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    float (*gml)[KA_COLS][2] = (float (*)[KA_COLS][2])ml;
    KaItem it;
    int ct;
    if (WIDE == 1 || (int)blockIdx.x < a.pre_items) {
        if (!ka_prefix(a, it, ct)) return;
        if constexpr (WIDE)
            ka_wide<D, XP>(a, it, ka_lds, (int*)(ka_lds + ka_wide_bytes<D>()), (float (*)[32][2])ml, limits, ct * KA_WIDE_COLS);
        else
            ka_narrow<KT, D, XP>(a, it, gml, limits, ct * KA_COLS, w, lane);
    } else {
        constexpr int COLS = WIDE == 2 ? KA_WIDE_COLS : KA_COLS;
        const int item = (int)blockIdx.x - a.pre_items, unit = item / a.c.n_kv_heads, g = item - unit * a.c.n_kv_heads;
        ka_runs(a, unit, found, red, COLS);
        const KaRun r = found;
        ct = r.ct;
        if (!ka_tail(a, it, r, g)) return;
        if (!a.direct && g == 0 && ct == 0 && r.z == 0)
            for (int i = tid; i < r.r1 - r.r0; i += 64 * WAVES) a.part_n[r.r0 + i] = it.direct ? 0 : r.runs;
        // columns beyond the tiles of the grid (a request of more rows than announced): more rounds
        for (int c0 = ct * COLS; c0 < it.ncols; c0 += r.tiles * COLS) {
            if constexpr (WIDE == 2)
                ka_wide<D, XP>(a, it, ka_lds, (int*)(ka_lds + ka_wide_bytes<D>()), (float (*)[32][2])ml, nullptr, c0);
            else
                ka_narrow<KT, D, XP>(a, it, gml, nullptr, c0, w, lane);
            __syncthreads();               // its output is out of LDS
        }
    }
}

template <typename KT, int D, int XP, int WIDE>
static int ka_launch(const KaArgs& a, hipStream_t st) {
    size_t lds = ka_narrow_bytes<KT, D>();
    if constexpr (WIDE) lds = ka_wide_lds<D>();
    PIO_TRY((allow_lds<ka_kernel<KT, D, XP, WIDE>>(lds)));
    ka_kernel<KT, D, XP, WIDE><<<a.pre_items + (WIDE == 1 ? 0 : a.tail_items), WIDE ? 512 : 256, lds, st>>>(a);
    PIO_LAUNCHED();
    if constexpr (WIDE == 1) {
        // the tails on their own: narrow workgroups beside wide ones would be one to a CU
        KaArgs t = a;
        t.pre_items = 0;
        return ka_launch<KT, D, XP, 0>(t, st);
    }
    if (!a.direct) {
        constexpr int GRP = 1024 / D;
        const int cols = a.rows * a.H;
        if (cols <= 2048) ka_merge_kernel<D, 8><<<ceil_div(cols, GRP / 8), 256, 0, st>>>(a);
        else ka_merge_kernel<D, 1><<<ceil_div(cols, GRP), 256, 0, st>>>(a);
        PIO_LAUNCHED();
    }
    return PIO_OK;
}

template <int D, int XP>
static int ka_route16(const KaArgs& a, int wide, hipStream_t st) {
    return wide == 2 ? ka_launch<_Float16, D, XP, 2>(a, st)
           : wide    ? ka_launch<_Float16, D, XP, 1>(a, st)
                     : ka_launch<_Float16, D, XP, 0>(a, st);
}
template <int D>
static int ka_route(const KaArgs& a, int wide, hipStream_t st) {
    if (a.c.kv_dtype == PIO_F32) return ka_launch<float, D, 1, 0>(a, st);
    return a.q16 ? ka_route16<D, 1>(a, wide, st) : ka_route16<D, 2>(a, wide, st);
}

// Workgroups of the tails' kernel that a CU holds.
template <typename KT, int D, int XP, int WIDE>
static int ka_held_by(int& held) {
    static std::atomic<int> known{0};
    held = known.load(std::memory_order_relaxed);
    if (held) return PIO_OK;
    const size_t lds = WIDE ? ka_wide_lds<D>() : ka_narrow_bytes<KT, D>();
    PIO_TRY((allow_lds<ka_kernel<KT, D, XP, WIDE>>(lds)));
    PIO_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&held, ka_kernel<KT, D, XP, WIDE>, WIDE ? 512 : 256, lds));
    held = std::max(held, 1);
    known.store(held, std::memory_order_relaxed);
    return PIO_OK;
}
template <int D>
static int ka_held(const KaArgs& a, bool wide, int& held) {
    if (a.c.kv_dtype == PIO_F32) return ka_held_by<float, D, 1, 0>(held);
    if (wide) return a.q16 ? ka_held_by<_Float16, D, 1, 2>(held) : ka_held_by<_Float16, D, 2, 2>(held);
    return a.q16 ? ka_held_by<_Float16, D, 1, 0>(held) : ka_held_by<_Float16, D, 2, 0>(held);
}

// An item costs its rounds of keys and this many more (its requests, pages, first copies; its
// join and output): 12,000 clocks beside 3,400 of a round.
constexpr float KA_FIXED = 3.5f;

// Items for the matrix core kernels.
static int ka_matrix(KaArgs& a, int max_rows, hipStream_t st) {
    const int Hk = a.c.n_kv_heads, cus = 256;
    const bool f16 = a.c.kv_dtype == PIO_F16;
    const int64_t cols = (int64_t)a.rows * a.G, tail_cols = (int64_t)std::min(max_rows, a.rows) * a.G;
    // A wide kernel for the prefix reads it once for 128 columns, but comes on top of the tails', some
    // 10 us. fp16 queries, 512 columns x 4 kv heads x 128 dimensions over 4,000 tokens 36 us (narrow 28),
    // over 8,000 39 (39), over 16,000 45 (58), over 32,000 64 (94); 128 x 8 x 64 over 16,000 30 (24), over
    // 32,000 36 (37). fp32 queries, whose wide kernel spills registers, even out at more than this: 512
    // x 4 x 128 over 8,000 49 (42), over 16,000 64 (64), over 32,000 93 (108).
    const bool long_prefix = cols > 64 && (double)cols * Hk * a.c.head_dim * a.shared >= 0x1.8p30;
    // Wide items for tails of more than 32 columns, which pays where there is much to read for many of them:
    // 8 heads to each of 4 kv heads of 128, fp16 queries, a prompt of 1,000 tokens 37 us (narrow 67), 48
    // windows of 8 behind 8,000 tokens 99 (121), of 5 behind 2,000 41 (52), 16 windows of 5 over 3,000 own
    // tokens 41 (44); and costs up to twice as much where there is little (the tails' lengths are not known
    // here): 16 windows of 16 over 300 own tokens 23 (16), one of 8 over 4,000 19 (13); fp32 queries 35 (18),
    // 25 (14), the prompt 56 (77), the windows behind 8,000 144 (161).
    const int wide = !f16 ? 0 : tail_cols > 32 ? 2 : long_prefix ? 1 : 0;
    a.tail_tiles = ceil_div(tail_cols, wide == 2 ? KA_WIDE_COLS : KA_COLS);
    // Items of one run to a request: all requests have max_rows rows, or one the most of them and each of
    // the others at worst one tile that is not full.
    PIO_REQUIRE((int64_t)a.n * Hk <= 1 << 22, "pio_kv_attention: %d requests are too many", a.n);
    const int64_t items = std::min((int64_t)a.n * a.tail_tiles, cols / (wide == 2 ? KA_WIDE_COLS : KA_COLS) + a.n) * Hk;
    // Runs. The lengths of the tails are not known here: a short prefix gets a quarter of the device,
    // a longer one up to all of it in runs of 8 rounds or more, and the tails are cut for what is there
    // by the kernel (ka_runs). 32 sequences behind 2,039 tokens 17 us, where both are cut to
    // fill the device on their own 24 us.
    int held = 1;
    PIO_TRY(a.c.head_dim == 128 ? ka_held<128>(a, wide == 2, held) : ka_held<64>(a, wide == 2, held));
    a.slots = cus * held;
    const int64_t units = (int64_t)Hk * a.tail_tiles;
    a.tail_runs = (int)std::max<int64_t>(1, (wide == 2 ? cus / 2 : 2 * cus) / units);
    const int64_t longest = std::max<int64_t>((int64_t)a.c.max_pages * a.c.page_size - a.shared, 1);
    // At most 32 to a request: one of 100,000 tokens over 4 kv heads of 128 takes 38 us (with 128 runs 41),
    // over one kv head 34 (20). And no more than 256 MB of partial results hold, as many rows fill the
    // device without; one there is whatever its size, and the prefix's runs come on top: rows x heads x
    // (D + 2) x 4 bytes for each.
    const int64_t part = (int64_t)a.rows * a.H * (a.c.head_dim + 2) * 4;
    a.max_runs = (int)std::min<int64_t>({a.tail_runs, 32, ceil_div(longest, KA_ROUND), std::max<int64_t>(1, (256 << 20) / part)});
    a.direct = a.shared == 0 && a.max_runs == 1;
    a.tail_items = (int)(items + (a.max_runs == 1 ? 0 : (int64_t)a.tail_runs * units));
    if (a.shared > 0) {
        a.pre_tiles = ceil_div(cols, wide ? KA_WIDE_COLS : KA_COLS);
        const int64_t pre_units = (int64_t)Hk * a.pre_tiles, rounds = ceil_div(a.shared, KA_ROUND), at_once = wide ? cus : 2 * cus;
        const int64_t most = at_once / pre_units;
        const int64_t splits = std::max<int64_t>({1, most / 4, wide == 1 ? most : std::min(rounds / 8, most)});
        a.pre_keys = (int)ceil_div(rounds, std::min(splits, rounds)) * KA_ROUND;
        a.pre_splits = ceil_div(a.shared, a.pre_keys);
        if (wide != 1) a.pre_work = (float)pre_units * (a.pre_splits * a.fixed + rounds);
        const int64_t pre = (int64_t)ceil_div((int64_t)Hk * a.pre_splits, 8) * 8 * a.pre_tiles;
        PIO_REQUIRE(pre <= 1 << 22, "pio_kv_attention: too many rows over %d shared tokens", a.shared);
        a.pre_items = (int)pre;
    }
    // (a grid has fewer than 2^32 threads)
    PIO_REQUIRE(((int64_t)a.pre_items + a.tail_items) * (wide ? 512 : 256) < (int64_t)1 << 32,
                "pio_kv_attention: %d requests and %d rows are too many", a.n, a.rows);
    Scratch ws;
    if (!a.direct) {
        const size_t parts = (size_t)(a.pre_splits + a.max_runs) * a.rows * a.H;
        PIO_TRY(ws.get(parts * (a.c.head_dim + 2) * sizeof(float) + a.rows * sizeof(int), st));
        a.part_o = (float*)ws.ptr;
        a.part_ml = a.part_o + parts * a.c.head_dim;
        a.part_n = (int*)(a.part_ml + 2 * parts);
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
    PIO_REQUIRE(out != q || q_stride == out_stride, "%s: out is q, at another stride", nm);
    // (a grid has fewer than 2^32 threads: the join's 8 columns to a workgroup, the simple kernel's one)
    const bool matrix = c->head_dim == 128 || c->head_dim == 64;
    PIO_REQUIRE((int64_t)rows * n_heads < (matrix ? 1 << 26 : 1 << 24), "%s: too many rows", nm);
    PIO_REQUIRE(std::isfinite(scale), "%s: scale %g", nm, (double)scale);
    KaArgs a{};
    a.fixed = KA_FIXED;
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
    a.g_magic = a.G > 1 ? (uint32_t)((1ull << 32) / a.G + 1) : 0;
    a.scale = scale;
    a.q16 = dtype == PIO_F16;
    hipStream_t st = pick_stream(stream);
    if (c->kv_dtype == PIO_MX4) return ka4_attention(a, max_rows, st);
    if (matrix) return ka_matrix(a, max_rows, st);
    if (c->kv_dtype == PIO_F32) ka_simple_kernel<float><<<rows * n_heads, KA_THREADS, 0, st>>>(a);
    else ka_simple_kernel<_Float16><<<rows * n_heads, KA_THREADS, 0, st>>>(a);
    PIO_LAUNCHED();
    return PIO_OK;
}
