// Causal attention of a batch over a paged cache of 4 bits (tensor_rocm.h: its layout):
//   out[r, h] = sum_t softmax_t(q[r, h] . k[t] * scale) v[t].
#include "kv_attention.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace pio {

// Head dimensions other than 64 and 128. One workgroup per (row, head): 256 keys at a time, a thread
// for each key's score, then a thread for each dimension of the weighted sum, KA4_DEEP values in flight; bound by the
// waits for them (where the matrix core kernels run, 128 dimensions: 40 sequences behind a prompt 273 us, there 15.6).
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

// ------------------------------------------------- the matrix core kernels ----
// Items (kv_attention.hpp) of 16 * NC columns by 4 waves; each wave takes every 4th tile of 32 keys on its own,
// K and V straight from memory into registers, the next tile under the way of this one's products. No LDS until
// the waves' sums meet.
//   S^T = K Q^T on v_mfma_scale_f32_16x16x128: 16 keys are one operand as they lie in memory, lane l the 16
//     bytes of key row l % 16 and dimensions 32 (l / 16) .. + 31, whose scale byte is the operand's own. Queries
//     are parts of 6 bits (e2m3), each of a scale of its own: a part holds 32 dimensions to within a 30th of the
//     largest, and the next part the rest. 6-bit operands run at the rate of 4-bit ones, twice that of 8 bits.
//     64 dimensions are half of an operand's depth: its halves are two parts of the query, the keys in both.
//   O^T = V^T P^T on v_mfma_f32_16x16x32_f16. Lane l reads the codes of 8 keys and dimensions D / 16 (l % 16) ..,
//     and widens each key's to fp16 under its scale, exactly: two keys' halves side by side are the operand, so
//     V is turned inside a lane. Row i of O^T tile n is dimension (D / 16) i + n.
// What it costs (2.4 GHz): an item's chain of waits (its request, page ids, K, the join) is 16,000 clocks, most of
// them loads on loads and code that is fetched for the first time; a tile of 32 keys and 32 columns of 128 dimensions, 34
// products (544 clocks) and 130 VALU instructions with fp16 queries, 1,100 clocks of a SIMD's issue, whatever the order:
// products and the VALU's work were measured to add up, also where two waves share the SIMD. Long tails are bound by
// memory: 3 sequences of 120,000 tokens (8 kv heads x 128, fp16) 70 us with their join, 5.6 TB/s; many columns by
// instructions: 78 rows of 32 heads over 24,000 tokens 49 us, 620 TFLOP/s. Tried and no faster (of 128 dimensions): the
// workgroup's waves on columns of their own around V widened once in LDS, K and V one more tile ahead, 3 waves to a SIMD
// of 16 columns, products and VALU interleaved by hand, wave priorities.
//   A lane's 8 scores are of the keys 4 q .. 4 q + 3 of either 16, q = l / 16, and those are the keys of its part of
//     the weights' operand; V's rows are read in that order.
typedef int ka4_i8 __attribute__((ext_vector_type(8)));
typedef uint32_t ka4_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t ka4_u6 __attribute__((ext_vector_type(6)));
typedef const __attribute__((address_space(1))) char* Ka4At;       // (global memory, as the compiler could not tell)
template <typename V>
__device__ __forceinline__ V ka4_get(Ka4At p) { return *(const __attribute__((address_space(1))) V*)p; }
typedef float ka4_v32 __attribute__((ext_vector_type(32)));
typedef _Float16 ka4_h2 __attribute__((ext_vector_type(2)));

constexpr int KA4_TILE = 32, KA4_WAVES = 4;

// X16: fp16 queries, 4 parts and weights in fp16; else 5 parts, and weights as two fp16 parts.
//   4 parts are within 2^-18 of the largest of 32 dimensions: what is a 128th of that or more keeps all 11 bits, and
// for what is smaller the loss of a block is a 20th of what rounding its largest to fp16 was. One dimension 30, 300,
// 3,000 times the others, 4,096 normal keys: 5e-6, 3e-5 and 2e-4 to 1e-3 of the output in the 2-norm, whose rounding is
// 2e-4 (3 parts: 2e-4, 5e-4 to 3e-3, 7e-3 to 3e-2; 5, as fp32 queries have: 2e-7, 7e-7, 4e-6, as fp32 products). 78
// rows behind 24,000 tokens 49.8 us (3 parts 47.6, 5 52.4), prompts of 509 and 111 rows 53.1 (50.6, 56.2); of 64
// dimensions, where an operand holds two parts, 24 windows of up to 6 in 32 columns 16.0 (15.8, 16.9).
//   Weights: rounding them costs normal inputs as much as rounding the output, 2.0e-4 each; a second part is a third of
// the products.
template <int D, bool X16>
struct Ka4 {
    static constexpr int PARTS = X16 ? 4 : 5, XP = X16 ? 1 : 2;
    static constexpr int QM = D == 128 ? PARTS : (PARTS + 1) / 2;      // products of a score
    static constexpr int NT = D / 16, RB = D / 2;                      // O^T tiles; bytes of a row's codes
    static constexpr int OP = D + 4;                                   // LDS pitch of a column's output (floats)
};

// The conversions between 32 floats (the even ones in a, the odd ones in b) and 6-bit codes write
// their result while they still read: the builtins do not say so, and the registers may overlap.
__device__ __forceinline__ ka4_u6 ka4_to6(const ka_v16& a, const ka_v16& b, float scale) {
    ka4_u6 r;
    asm("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3\n s_nop 1" : "=&v"(r) : "v"(a), "v"(b), "v"(scale));
    return r;
}
__device__ __forceinline__ ka4_v32 ka4_from6(const ka4_u6& c, float scale) {
    ka4_v32 r;
    asm("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2\n s_nop 1" : "=&v"(r) : "v"(c), "v"(scale));
    return r;
}

// A column's query times scale * log2(e), so that a score is the exponent of its weight as it comes: lane l has
// 32 dimensions of column l % 16.
template <int D, bool X16>
struct Ka4Q {
    ka4_u6 p[Ka4<D, X16>::QM];
    uint32_t e[(Ka4<D, X16>::QM + 3) / 4];         // four scales to a word
    __device__ __forceinline__ void scale(int m, int to) {
        e[m / 4] = (e[m / 4] & ~(255u << 8 * (m & 3))) | (uint32_t)to << 8 * (m & 3);
    }
};
// Its elements as they lie in memory, loaded ahead of the keys (waits for loads are in order).
template <bool X16>
struct Ka4Raw {
    uint4 u[X16 ? 4 : 8];
};
template <int D, bool X16>
__device__ __forceinline__ void ka4_raw_q(const KaArgs& a, int row, int head, bool live, int part, Ka4Raw<X16>& raw) {
    const int64_t at = (live ? row * a.q_stride + (int64_t)head * D : 0) + 32 * (D == 128 ? part : part & 1);
    const uint4* from = (const uint4*)((const char*)a.q + at * (X16 ? 2 : 4));
#pragma unroll
    for (int i = 0; i < (X16 ? 4 : 8); i++) raw.u[i] = from[i];
}
template <int D, bool X16>
__device__ __forceinline__ void ka4_set_q(const KaArgs& a, const Ka4Raw<X16>& raw, bool live, int part, Ka4Q<D, X16>& q) {
    using T = Ka4<D, X16>;
    const int half = D == 128 ? 0 : part >> 1;         // 64 dimensions: which parts this half of the operand has
    const float scale = a.scale * KA_LOG2E;
    ka_v16 xa, xb;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        float x;
        if constexpr (X16) x = (float)__builtin_bit_cast(ka_h8, raw.u[i / 8])[i % 8];
        else x = __builtin_bit_cast(ka_f4, raw.u[i / 4])[i % 4];
        x *= scale;
        most = max(most, __float_as_uint(x) & 0x7fffffffu);
        (i & 1 ? xb : xa)[i / 2] = x;
    }
    const bool odd = most >= 0x7f800000u;              // inf or NaN: a NaN scale makes the column's scores NaN
    if (!live || odd) {
        most = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) xa[i] = xb[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < (T::QM + 3) / 4; i++) q.e[i] = 0;
    // the least power of two (a byte of exponent) that the largest is below 7.5 of, with what rounds up to 8; a
    // part's rest is at most a quarter of its step's unit, or an eighth from the second part on: 4 and 5 bits
    const int first = (int)((most + 0x100000u) >> 23) - 2;
#pragma unroll
    for (int p = 0; p < T::PARTS; p++) {
        int e = max(first - (p ? 5 * p - 1 : 0), 1);
        const float unit = __uint_as_float((uint32_t)e << 23);
        const ka4_u6 c = ka4_to6(xa, xb, unit);
        if (live && odd) e = KV_MX4_NAN;
        if constexpr (D == 128) {
            q.p[p] = c;
            q.scale(p, e);
        } else if (p % 2 == 0) {
            q.p[p / 2] = c;
            q.scale(p / 2, e);
            if (half && p == T::PARTS - 1) q.p[p / 2] = ka4_u6{0, 0, 0, 0, 0, 0};
        } else if (half) {
            q.p[p / 2] = c;
            q.scale(p / 2, e);
        }
        if (p + 1 < T::PARTS) {
            const ka4_v32 y = ka4_from6(c, unit);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                xa[i] -= y[2 * i];
                xb[i] -= y[2 * i + 1];
            }
        }
    }
}

// A column's running softmax. `ref`: minus its reference, plus KA_LIFT, in all elements: the products of a score
// start there, and give the exponent of its weight. l: the sum of the weights, which the matrix cores add up too
// (of the rounded weights, as O^T is), in all elements.
template <int D>
struct Ka4Acc {
    ka_f4 ref, l, o[D / 16];
    // The reference; -FLT_MAX: saw no key (the largest weight of a tile is never lost in l).
    __device__ __forceinline__ float m() const { return l[0] == 0.f ? -FLT_MAX : -ref[0]; }
    __device__ void clear() {
        ref = l = ka_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < D / 16; n++) o[n] = ka_f4{0.f, 0.f, 0.f, 0.f};
    }
};

// A lane's share of a tile's keys, and of its values.
struct Ka4K {
    ka4_u4 k[2];
    int ks[2];
};
struct Ka4V {
    uint32_t v[8], vs[2];
};

// Sums over the lanes up to each.
__device__ __forceinline__ int ka4_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);      // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);      // row_bcast 15, into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);      // row_bcast 31, into rows 2 and 3
    return x;
}

// The least of the wave's.
__device__ __forceinline__ int ka4_least(int x) {
    auto with = [&](auto ctrl, auto rows) {
        x = min(x, __builtin_amdgcn_update_dpp(INT_MAX, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    };
    with(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});      // as above
    with(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    with(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    with(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    with(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
    with(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
    return __builtin_amdgcn_readlane(x, 63);
}

// A wave's tiles, every KA4_WAVES-th. The scores run one tile ahead of the softmax, in one piece of code without
// branches: their products fill the matrix cores while the VALU forms the weights and widens the values. K is
// loaded two tiles ahead, V one, by turns into two sets of registers.
// ONCE: no other column tile reads these keys (a request of more rows than announced does so itself).
template <int D, bool X16, int NC, bool ONCE>
struct Ka4Walk {
    using T = Ka4<D, X16>;
    const char* kb;
    int64_t plane;                                 // from K to V
    uint32_t page_b;
    uint32_t ko, kso, vo, vso;                     // this lane's offsets from a half tile's codes, and scales
    int first, count, lo, hi, lg, mask;            // first key, tiles of this wave; first and last page of the table row
    // Of the next 32 tiles to be loaded, lane l has half l % 2 of the l / 2-th (pages of 16 keys or more: a half has
    // one; outside the item's keys, the nearest): where its codes begin, and the page of the 32 behind
    uint64_t base;
    int id;
    int bad_at = INT_MAX;                          // first key in a page outside the cache
    bool odd = false;
    Ka4At kc[2], vc[2];                            // halves of the next tiles of K and V to be loaded: their codes,
    int kd[2], vd[2];                              // and how far behind those their scales
    Ka4K k0, k1;
    Ka4V v0, v1;

    __device__ __forceinline__ int half_of(int i, int lane) const {
        return first + min(i + (lane >> 1), count - 1) * (KA4_WAVES * KA4_TILE) + 16 * (lane & 1);
    }
    __device__ __forceinline__ void look_up(const KaItem& it, int i, int lane) {
        id = it.table[min(max(half_of(i, lane) >> lg, lo), hi)];
    }
    // The next tile's place: its lanes' words as scalars.
    __device__ __forceinline__ void place(const KaArgs& a, const KaItem& it, int i, int lane) {
        if ((i & 31) == 0) {
            const int t = half_of(i, lane);
            const bool ok = (unsigned)id < (unsigned)a.c.n_pages;
            if (__any(!ok))
                bad_at = min(bad_at, ka4_least(ok ? INT_MAX : max(min(max(t, it.k0), it.k1 - 1) & -16, it.k0)));
            base = (uint64_t)(uintptr_t)kb + (uint64_t)(ok ? (uint32_t)id : 0u) * page_b + (t & mask) * T::RB;
            if (i + 32 < count) look_up(it, i + 32, lane);
        }
        const int t = first + min(i, count - 1) * (KA4_WAVES * KA4_TILE);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int l = 2 * (i & 31) + h;
            kc[h] = (Ka4At)(uintptr_t)((uint32_t)__builtin_amdgcn_readlane((int)base, l) |
                                             (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(base >> 32), l) << 32);
            vc[h] = kc[h] + plane;
            kd[h] = vd[h] = (T::RB << lg) - ((t + 16 * h) & mask) * (T::RB - 1);
        }
    }
    // (opaque where they are used: a load is then one instruction, of scalars and an offset)
    __device__ __forceinline__ static uint32_t here(uint32_t offset) {
        asm volatile("" : "+v"(offset));
        return offset;
    }
    __device__ __forceinline__ void load_k(Ka4K& to) {
        const uint32_t o = here(ko);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            // (past the caches where the keys are read once: 3 sequences of 120,000 tokens 70.3 us, through them 76.8, 32 of
            // 16,000 54.7 and 58.8, where no cache holds them before the call; where the memory-side cache does, the same 137
            // MB again and again, 43.6 and 41.2. V's rows, whose lines two loads share, are not. Where several tiles read the
            // keys: 24 windows of up to 6 over 16,000 tokens, 3 tiles each, 26.6 past the caches, 25.2 through them)
            if constexpr (ONCE)
                to.k[h] = __builtin_nontemporal_load((const __attribute__((address_space(1))) ka4_u4*)(kc[h] + o));
            else
                to.k[h] = ka4_get<ka4_u4>(kc[h] + o);
            to.ks[h] = ka4_get<uint8_t>(kc[h] + here(kso + kd[h]));
        }
    }
    __device__ __forceinline__ void load_v(Ka4V& to) {
        const uint32_t o = here(vo);
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (D == 128) to.v[4 * h + i] = ka4_get<uint32_t>(vc[h] + o + i * T::RB);
                else to.v[4 * h + i] = ka4_get<uint16_t>(vc[h] + o + i * T::RB);
            }
            to.vs[h] = ka4_get<uint32_t>(vc[h] + here(vso + vd[h]));
        }
    }
    // The first tiles' loads, if the wave has any.
    __device__ __forceinline__ void begin(const KaArgs& a, const KaItem& it, int w, int lane) {
        const pio_kv_cache& c = a.c;
        lg = kv_log2(c.page_size);
        mask = c.page_size - 1;
        const int64_t head = (int64_t)c.page_size * (D / 32 * 17);
        page_b = (uint32_t)(head * c.n_kv_heads);
        plane = (int64_t)c.n_pages * page_b;
        kb = (const char*)c.kv + 2 * a.layer * plane + it.g * head;
        first = (it.k0 & -KA4_TILE) + w * KA4_TILE;
        lo = it.k0 >> lg;
        hi = max(it.k1 - 1, 0) >> lg;
        count = it.k1 > first ? (it.k1 - first + KA4_WAVES * KA4_TILE - 1) / (KA4_WAVES * KA4_TILE) : 0;
        if (it.k1 <= it.k0) count = 0;
        if (count == 0) return;
        look_up(it, 0, lane);
        const uint32_t r = lane & 15, part = lane >> 4, kblock = D == 128 ? part : part & 1;
        ko = r * T::RB + 16 * kblock;
        kso = (kblock << lg) + r;
        vo = 4 * part * T::RB + D / 32 * r;
        vso = ((D / 16 * r >> 5) << lg) + 4 * part;
        place(a, it, 0, lane);
        load_k(k0);
        load_v(v0);
        place(a, it, 1, lane);
        load_k(k1);
    }

    // Scores of 16 NC columns, exponents of weights.
    __device__ __forceinline__ void scores(const Ka4K& k, const Ka4Q<D, X16> (&q)[NC], const Ka4Acc<D> (&x)[NC],
                                           float (&s)[NC][8]) {
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const ka4_i8 kt = {(int)k.k[t][0], (int)k.k[t][1], (int)k.k[t][2], (int)k.k[t][3], 0, 0, 0, 0};
                ka_f4 acc = x[c].ref;
#pragma unroll
                for (int m = T::QM - 1; m >= 0; m--) {             // the small parts first
                    const ka4_u6& p = q[c].p[m];
                    const ka4_i8 qm = {(int)p[0], (int)p[1], (int)p[2], (int)p[3], (int)p[4], (int)p[5], 0, 0};
                    const int at = (int)q[c].e[m / 4];             // (which byte of it is in the instruction)
                    if ((m & 3) == 0) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kt, qm, acc, 4, 2, 0, k.ks[t], 0, at);
                    if ((m & 3) == 1) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kt, qm, acc, 4, 2, 0, k.ks[t], 1, at);
                    if ((m & 3) == 2) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kt, qm, acc, 4, 2, 0, k.ks[t], 2, at);
                    if ((m & 3) == 3) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kt, qm, acc, 4, 2, 0, k.ks[t], 3, at);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) s[c][4 * t + e] = acc[e];
            }
    }
    // Keys of a lane's scores (from 4 part on), and the rows of its values.
    static constexpr int key(int i) { return 16 * (i / 4) + i % 4; }
    // What a column does not see, and the references. They are the wave's first tile's maxima (a column that sees no
    // key there sees none at all), and follow where a score has grown past them.
    __device__ __forceinline__ void settle(const KaItem& it, int t0, int part, bool edge, bool begin,
                                           const int (&limit)[NC], Ka4Acc<D> (&x)[NC], float (&s)[NC][8]) {
        if (edge) {
            int key0 = t0 + 4 * part;
            asm volatile("" : "+v"(key0));         // (a branch: as selects in every tile the masks cost 40 instructions)
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    s[c][i] = key0 + key(i) < limit[c] && key0 + key(i) >= it.k0 ? s[c][i] : -INFINITY;
        }
        float top[NC], most;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            top[c] = s[c][0];
#pragma unroll
            for (int i = 1; i < 8; i++) top[c] = fmaxf(top[c], s[c][i]);
            most = c ? fmaxf(most, top[c]) : top[c];
        }
        if (!begin && !__any(most > KA_LIFT + KA_SLACK)) return;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const float t = ka_max<16>(top[c]);
            const bool sees = t > KA_SEEN;
            const float by = begin ? (sees ? KA_LIFT - t : 0.f) : fminf(KA_LIFT - fmaxf(t, KA_LIFT), 0.f);
            x[c].ref += by;
            if (!begin) {
                const float corr = __builtin_amdgcn_exp2f(by);
                x[c].l *= corr;
#pragma unroll
                for (int n = 0; n < T::NT; n++) x[c].o[n] *= corr;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) s[c][i] += by;
        }
    }
    // O^T and l of one tile, of the scores s; their place then has the next tile's.
    __device__ __forceinline__ void products(const Ka4K& k, const Ka4V& v, const Ka4Q<D, X16> (&q)[NC], Ka4Acc<D> (&x)[NC],
                                             float (&s)[NC][8]) {
        const _Float16 one = (_Float16)1.f;
        const ka_h8 ones = {one, one, one, one, one, one, one, one};
        float next[NC][8];
        scores(k, q, x, next);
        ka_h8 wt[NC][T::XP];
#pragma unroll
        for (int c = 0; c < NC; c++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float w = __builtin_amdgcn_exp2f(s[c][i]);
                const _Float16 hi = (_Float16)w;
                wt[c][0][i] = hi;
                if constexpr (T::XP == 2) wt[c][T::XP - 1][i] = (_Float16)(w - (float)hi);
            }
#pragma unroll
            for (int p = 0; p < T::XP; p++) x[c].l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, wt[c][p], x[c].l, 0, 0, 0);
        }
        // (the conversions look at a scale's exponent alone: what else a shift leaves in the word does not matter)
        float unit[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t word = v.vs[i / 4];
            unit[i] = __uint_as_float((i & 3) == 3 ? word >> 1 : word << (23 - 8 * (i & 3)));
        }
        auto pair = [&](auto byte) {
            constexpr int B = decltype(byte)::value;
            ka_h8 a0, a1;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const ka4_h2 y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v.v[i], unit[i], B);
                a0[i] = y[0];
                a1[i] = y[1];
            }
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int p = 0; p < T::XP; p++) {
                    x[c].o[2 * B] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, wt[c][p], x[c].o[2 * B], 0, 0, 0);
                    x[c].o[2 * B + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, wt[c][p], x[c].o[2 * B + 1], 0, 0, 0);
                }
        };
        pair(std::integral_constant<int, 0>{});
        pair(std::integral_constant<int, 1>{});
        if constexpr (D == 128) {
            pair(std::integral_constant<int, 2>{});
            pair(std::integral_constant<int, 3>{});
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) s[c][i] = next[c][i];
    }
    __device__ __forceinline__ void run(const KaArgs& a, const KaItem& it, int lane, const Ka4Q<D, X16> (&q)[NC],
                                        const int (&limit)[NC], Ka4Acc<D> (&x)[NC]) {
        if (count == 0) return;
        const int part = lane >> 4;
        int least = limit[0];
#pragma unroll
        for (int c = 1; c < NC; c++) least = min(least, limit[c]);
        least = ka4_least(least);
        auto begins = [&](int i) { return first + i * (KA4_WAVES * KA4_TILE); };
        const int whole = least >= first ? (least - first) / (KA4_WAVES * KA4_TILE) + (((least - first) & (KA4_WAVES * KA4_TILE - 1)) >= KA4_TILE) : 0;
        const int low = first < it.k0 ? 0 : -1;
        auto edge = [&](int i) { return i >= whole || i == low; };
        float s[NC][8];
        scores(k0, q, x, s);
        settle(it, begins(0), part, edge(0), true, limit, x, s);
        auto step = [&](int i, const Ka4K& k, Ka4K& kfree, Ka4V& v, Ka4V& vfree) {
            // (past the end the last tile again: under a branch the waits for loads could not count these)
            load_v(vfree);
            place(a, it, i + 2, lane);
            load_k(kfree);
            if (edge(i)) {
                // A value that some column does not see must not reach it, 0 * NaN: NaN blocks are left out (ka4_mend
                // adds them to the columns that see them), and whatever lies outside the item's keys
                int key0 = begins(i) + 4 * part;
                asm volatile("" : "+v"(key0));
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    uint32_t& word = v.vs[e / 4];
                    const uint32_t byte = word >> 8 * (e & 3) & 255u;
                    const bool in = key0 + key(e) >= it.k0 && key0 + key(e) < it.k1, wrong = byte > KV_MX4_MOST;
                    odd |= in && wrong;
                    if (!in || wrong) word &= ~(255u << 8 * (e & 3));
                }
            }
            products(k, v, q, x, s);               // (behind the last tile the scores of some tile again, unused)
            if (i + 1 < count) settle(it, begins(i + 1), part, edge(i + 1), false, limit, x, s);
        };
        for (int i = 0; i < count; i += 2) {
            step(i, k1, k0, v0, v1);
            if (i + 1 < count) step(i + 1, k0, k1, v1, v0);
        }
    }
};

// NaN value blocks that the walk left out, added to 4 dimensions from d of a column that sees the keys up to `limit`: they
// are in the item's first tile, where that begins before its keys, and from `edge` on, the first tile that some column
// does not see all of. (A NaN in the last token: a prompt's 509 rows over 12,000 tokens 140 us, 117 without it, 8,670 by all
// keys of a run.)
template <int D>
__device__ __forceinline__ void ka4_mend(const KaArgs& a, const KaItem& it, int edge, int limit, int d, ka_f4& v) {
    const pio_kv_cache& c = a.c;
    const int lg = kv_log2(c.page_size);
    const int64_t head = (int64_t)c.page_size * (D / 32 * 17), page_b = head * c.n_kv_heads;
    const uint8_t* vb = (const uint8_t*)c.kv + (int64_t)(2 * a.layer + 1) * c.n_pages * page_b + it.g * head +
                        c.page_size * (D / 2 + d / 32);
    auto look = [&](int from, int to) {
        for (int t = from; t < min(to, min(limit, it.k1)); t++) {
            const int page = it.table[t >> lg];
            if (page < 0 || page >= c.n_pages) continue;
            if (vb[page * page_b + (t & (c.page_size - 1))] > KV_MX4_MOST) v = ka_f4{NAN, NAN, NAN, NAN};
        }
    };
    if (it.k0 % KA4_TILE) look(it.k0, (it.k0 | (KA4_TILE - 1)) + 1);
    look(max(it.k0, edge), it.k1);
}

// An item's columns from c0 joined over its waves and written, 16 at a time.
template <int D, bool X16, int NC, bool ONCE>
__device__ __forceinline__ void ka4_item(const KaArgs& a, const KaItem& it, float* lds, float (*ml)[16][2], int* limits,
                                         int c0, int w, int lane) {
    using T = Ka4<D, X16>;
    Ka4Walk<D, X16, NC, ONCE> walk;
    const int first = ka_div(a, c0);
    Ka4Raw<X16> raw[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int col = c0 + 16 * c + (lane & 15);
        const bool has = col < it.ncols;
        const int r = has ? ka_div(a, col) : 0, head = it.g * a.G + (has ? col - r * a.G : 0);
        ka4_raw_q<D, X16>(a, it.row0 + r, head, has, lane >> 4, raw[c]);
    }
    walk.begin(a, it, w, lane);
    if (limits) ka_limits(a, first, limits, 16 * NC);      // under the first loads' way
    Ka4Q<D, X16> q[NC];
    Ka4Acc<D> x[NC];
    int limit[NC], sees[NC];                               // in this item; at all (-1: no such column or row)
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int col = c0 + 16 * c + (lane & 15);
        const bool has = col < it.ncols;
        const int r = has ? ka_div(a, col) : 0;
        limit[c] = has ? ka_limit(it, limits, first, r) : it.k1;
        sees[c] = !has ? -1 : limits ? limits[r - first] : it.first_limit + r;
        x[c].clear();
        ka4_set_q<D, X16>(a, raw[c], has, lane >> 4, q[c]);
    }
    walk.run(a, it, lane, q, limit, x);
    // a page outside the cache: NaN for the columns that see its keys
    const int bad_at = walk.bad_at;
    bool told = it.bad;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        told |= sees[c] > bad_at;
        if (it.bad || limit[c] > bad_at) x[c].l[0] = NAN;
    }
    if (told) atomicOr(a.c.work, KV_BAD);
    const bool odd = __syncthreads_or(walk.odd);
    int edge = 0;
    if (odd) {
        int least = limit[0];
#pragma unroll
        for (int c = 1; c < NC; c++) least = min(least, limit[c]);
        edge = max(ka4_least(least), 0) & -KA4_TILE;
    }
#pragma unroll
    for (int c = 0; c < NC; c++) {
        if (c && c0 + 16 * c >= it.ncols) break;
        if (c) __syncthreads();                            // the last columns are out of LDS
        const int col = lane & 15, part = lane >> 4;
        if (part == 0) {
            ml[w][col][0] = x[c].m();
            ml[w][col][1] = x[c].l[0];
        }
        __syncthreads();
        float mx = ml[0][col][0];
#pragma unroll
        for (int i = 1; i < KA4_WAVES; i++) mx = fmaxf(mx, ml[i][col][0]);
        const float f = __builtin_amdgcn_exp2f(x[c].m() - mx);
        float* to = lds + (w * 16 + col) * T::OP;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int n = 0; n < T::NT; n += 4) {
                ka_f4 v;
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = x[c].o[n + k][e] * f;
                *(ka_f4*)(to + T::NT * (4 * part + e) + n) = v;
            }
        __syncthreads();
        for (int i = w * 64 + lane; i < min(16, it.ncols - c0 - 16 * c) * (D / 4); i += 64 * KA4_WAVES) {
            const int cc = i / (D / 4), d = (i % (D / 4)) * 4, at = c0 + 16 * c + cc;
            float m = ml[0][cc][0], l = 0.f;
#pragma unroll
            for (int k = 1; k < KA4_WAVES; k++) m = fmaxf(m, ml[k][cc][0]);
            ka_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KA4_WAVES; k++) {
                v += *(const ka_f4*)(lds + (k * 16 + cc) * T::OP + d);
                l += ml[k][cc][1] * __builtin_amdgcn_exp2f(ml[k][cc][0] - m);
            }
            if (odd) ka4_mend<D>(a, it, edge, ka_limit(it, limits, first, ka_div(a, at)), d, v);
            ka_emit(a, D, it, at, d, v, m, l);
        }
    }
}

// ka_runs for up to 64 N requests, by each wave on its own: no LDS and no barriers, and what is found is the same
// for the wave's lanes as the compiler sees it. 1 sequence 8.9 us (by the workgroup 9.6), 40 behind a prompt 15.7
// (16.8), 200 of up to 300 tokens 31.8 (32.2); more would cost registers.
template <int N>
__device__ __forceinline__ void ka4_runs(const KaArgs& a, int unit, KaRun& found, int cols) {
    const int lane = threadIdx.x & 63;
    int r0[N], r1[N], s[N], L[N], n[N], sum = 0;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int i = min(lane + 64 * k, a.n - 1);
        ka_rows(a, i, r0[k], r1[k]);
        s[k] = a.seq[i];
    }
#pragma unroll
    for (int k = 0; k < N; k++) L[k] = kv_seq_len(a.c, s[k]);
#pragma unroll
    for (int k = 0; k < N; k++) {
        n[k] = L[k] <= a.shared ? 1 : (L[k] - a.shared + KA_ROUND - 1) / KA_ROUND;
        if (lane + 64 * k >= a.n || r1[k] <= r0[k]) n[k] = 0;
        sum += n[k];
    }
    const int total = __builtin_amdgcn_readlane(ka4_scan(sum), 63);
    const float units = a.c.n_kv_heads * a.tail_tiles;
    const float cut = fmaxf(fmaxf(1.f, (float)total / a.tail_runs),
                            fminf(a.fixed, ka_cut(total, units, a.pre_work + a.n * units * a.fixed, a.slots, a.fixed)));
    found.i = -1;
    int before = 0;
#pragma unroll
    for (int k = 0; k < N; k++) {
        int per = 1, runs = 0, tiles = 0;
        if (n[k] > 0) {
            tiles = min(a.tail_tiles, ((r1[k] - r0[k]) * a.G + cols - 1) / cols);
            runs = min(max(1, (int)(n[k] / cut + 0.5f)), a.max_runs);
            per = (n[k] + runs - 1) / runs;
            runs = (n[k] + per - 1) / per;
        }
        const int mine = runs * tiles, upto = before + ka4_scan(mine);
        const uint64_t hit = __ballot(unit >= upto - mine && unit < upto);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            found.i = l + 64 * k;
            found.runs = of(runs);
            found.per = of(per);
            found.tiles = of(tiles);
            found.r0 = of(r0[k]);
            found.r1 = of(r1[k]);
            found.s = of(s[k]);
            found.L = of(L[k]);
            const int at = unit - of(upto - mine);
            found.z = at / found.tiles;
            found.ct = at - found.z * found.tiles;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
}

// Workgroups to a CU, by registers: 168 hold 16 columns of fp16 queries of 64 dimensions (60 sequences of up to 492 tokens,
// 16 heads of their own, 15.0 us, two to a CU 17.2), the others take 187 to 256.
__host__ __device__ constexpr int ka4_held(int D, bool x16, int nc) { return D == 64 && x16 && nc == 1 ? 3 : 2; }

// The prefix's items, then the tails'.
template <int D, bool X16, int NC, bool ONCE>
__global__ __launch_bounds__(256, ka4_held(D, X16, NC)) void ka4_kernel(KaArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[KA4_WAVES * 16 * Ka4<D, X16>::OP];
    __shared__ float ml[KA4_WAVES][16][2];
    __shared__ int limits[16 * NC];
    __shared__ KaRun found;
    __shared__ int red[KA4_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int COLS = 16 * NC;
    KaItem it;
    int ct;
    if ((int)blockIdx.x < a.pre_items) {
        if (ka_prefix(a, it, ct)) ka4_item<D, X16, NC, false>(a, it, lds, ml, limits, ct * COLS, w, lane);
        return;
    }
    const int item = (int)blockIdx.x - a.pre_items, unit = item / a.c.n_kv_heads, g = item - unit * a.c.n_kv_heads;
    KaRun r;
    if (a.n <= 64) {
        ka4_runs<1>(a, unit, r, COLS);
    } else if (a.n <= 256) {
        ka4_runs<4>(a, unit, r, COLS);
    } else {
        ka_runs(a, unit, found, red, COLS);
        auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
        r = KaRun{same(found.i), same(found.z), same(found.runs), same(found.per), same(found.ct), same(found.tiles),
                  same(found.r0), same(found.r1), same(found.s), same(found.L)};
    }
    if (!ka_tail(a, it, r, g)) return;
    if (!a.direct && g == 0 && r.ct == 0 && r.z == 0)
        for (int i = tid; i < r.r1 - r.r0; i += 64 * KA4_WAVES) a.part_n[r.r0 + i] = it.direct ? 0 : r.runs;
    // columns beyond the tiles of the grid (a request of more rows than announced): more rounds
    for (int c0 = r.ct * COLS; c0 < it.ncols; c0 += r.tiles * COLS) {
        // (opaque: else the addresses that the lane alone decides are formed ahead of the loop, and 32 columns of 128
        // have no registers for them: their reloads put the first loads in a row, two prompts 57 us, so 55)
        int own = lane;
        if constexpr (NC > 1) asm volatile("" : "+v"(own));
        ka4_item<D, X16, NC, ONCE>(a, it, lds, ml, nullptr, c0, w, own);
        __syncthreads();                                   // its output is out of LDS
    }
}

template <int D, bool X16, int NC, bool ONCE>
static int ka4_launch(const KaArgs& a, hipStream_t st) {
    ka4_kernel<D, X16, NC, ONCE><<<a.pre_items + a.tail_items, 256, 0, st>>>(a);
    PIO_LAUNCHED();
    return PIO_OK;
}
template <int D, bool X16>
static int ka4_width(const KaArgs& a, int nc, hipStream_t st) {
    if (nc > 1) return ka4_launch<D, X16, 2, false>(a, st);
    return a.tail_tiles == 1 ? ka4_launch<D, X16, 1, true>(a, st) : ka4_launch<D, X16, 1, false>(a, st);
}
template <int D>
static int ka4_route(const KaArgs& a, int nc, hipStream_t st) {
    return a.q16 ? ka4_width<D, true>(a, nc, st) : ka4_width<D, false>(a, nc, st);
}
template <int D>
static int ka4_join(const KaArgs& a, hipStream_t st) {
    constexpr int GRP = 1024 / D;
    const int cols = a.rows * a.H;
    if (cols <= 2048) ka_merge_kernel<D, 8><<<ceil_div(cols, GRP / 8), 256, 0, st>>>(a);
    else ka_merge_kernel<D, 1><<<ceil_div(cols, GRP), 256, 0, st>>>(a);
    PIO_LAUNCHED();
    return PIO_OK;
}

// An item costs its rounds of keys and this many more. A small figure cuts long rows into more runs than pay for their
// join: 32 sequences of up to 16,000 tokens 19.8 us with 4, 17.2 with 6, 17.0 with 8, and 96 of them 43.5 us with any of
// these; with 2, 40 sequences behind a prompt 16.3 us against 15.6.
constexpr float KA4_FIXED = 6.f;
// Rounds of a run at least, as a table row's pages allow: below, what the waves save is less than what the join costs.
// 1 sequence of 301 tokens 8.9 us, in runs of a round 10.1; of 200 8.2 and 10.0, of 500 10.7 and 10.2.
constexpr int KA4_LEAST = 4;
// Keys of a prefix's run at most (below).
constexpr int KA4_RUN = 8192;

// Rounds of a request's own tokens, which the host does not know: taken for all where the width of the items is chosen.
constexpr int KA4_TAIL = 8;

// How the columns are cut into items of `width`, and the rounds of 16 columns that the device takes for them: as long as an
// item, and as all of them over its `places`. A round of 32 columns is `round` of 16.
struct Ka4Cut {
    int64_t tail_tiles, items;                     // column tiles of a request at most; items of one run to a request
    int64_t pre_tiles, pre_splits, pre_keys;
    float cost;
};
static Ka4Cut ka4_cut(const KaArgs& a, int64_t tail_cols, int64_t part, int width, float round, int places) {
    Ka4Cut k{};
    const int64_t Hk = a.c.n_kv_heads, cols = (int64_t)a.rows * a.G;
    const float tail = a.fixed + round * KA4_TAIL;
    k.tail_tiles = (tail_cols + width - 1) / width;
    k.items = std::min(a.n * k.tail_tiles, cols / width + a.n) * Hk;
    k.cost = std::max(tail, k.items * tail / places);
    if (a.shared == 0) return k;
    k.pre_tiles = (cols + width - 1) / width;
    const int64_t units = Hk * k.pre_tiles, rounds = (a.shared + KA_ROUND - 1) / KA_ROUND, most = a.slots / units;
    // As many runs as fill the device, a quarter of that where the prefix is short (the tails need some of it), and
    // none longer than KA4_RUN keys where several column tiles read them: an XCD's workgroups then stay within what
    // its L2 holds (and no more of these than 256 MB of partial results hold). 78 rows of 32 heads on 4 over 96,000 tokens
    // 178 us, 240 in longer runs, 171 in runs of 6,144; over 48,000 78, 78 and 90.
    const int64_t splits = std::max<int64_t>({1, most / 4, std::min(rounds / 8, most),
                                              k.pre_tiles > 1 ? std::min<int64_t>((a.shared + KA4_RUN - 1) / KA4_RUN, (256 << 20) / part) : 1});
    const int64_t each = std::min(splits, rounds), run = (rounds + each - 1) / each;
    k.pre_keys = run * KA_ROUND;
    k.pre_splits = (a.shared + k.pre_keys - 1) / k.pre_keys;
    const float pre = a.fixed + round * run;
    k.cost = std::max({pre, tail, (units * k.pre_splits * pre + k.items * tail) / places});
    return k;
}

// Items for the matrix core kernels.
static int ka4_matrix(KaArgs& a, int max_rows, hipStream_t st) {
    const int Hk = a.c.n_kv_heads, cus = 256;
    const int64_t tail_cols = (int64_t)std::min(max_rows, a.rows) * a.G;
    const int64_t part = (int64_t)a.rows * a.H * (a.c.head_dim + 2) * 4;
    a.fixed = KA4_FIXED;
    a.slots = 2 * cus;                             // two workgroups to a CU
    PIO_REQUIRE((int64_t)a.n * Hk <= 1 << 22, "pio_kv_attention: %d requests are too many", a.n);
    // Items of 32 columns widen V once for both their tiles and halve what crosses from L2, items of 16 are twice as
    // many: 32 where their cost is the lower (where a request has 16 columns at most, half of them would be empty). Over
    // 4,000 random shapes of 17 columns a request and more, up to 60,000 shared tokens and tails of 20,000, which were not
    // used to choose this, what is taken costs 1.1 % more than the better of both (fp16 of 64 dimensions 2.1 %; one in 20
    // costs 9 to 17 %), always 16 columns 5 to 10 %, always 32 12 to 14 %. fp16 queries, 8 heads to each of 4 kv heads of
    // 128, 40 windows of up to 3 (78 rows): behind 48,000 tokens 78.6 us (16 columns: 105.0), 24,000 49.7 (84.4), 12,000
    // 47.9 (46.0), 6,000 34.8 (29.2), 2,000 19.9 (17.7); prompts of 509 and 111 rows over 4,090 and 1,065 tokens, 4 heads to
    // each of 8, 53.3 (64.5), of 2,000 tokens 113 (158). Of 64 dimensions, 7 heads to each of 2, 24 windows of up to 3 12.6
    // (32 columns: 14.9), 6 14.9 (16.3), 12 19.9 (17.9). fp32, those 40 windows behind 48,000 109 (16 columns: 130), 24,000
    // 68.2 (99.8), 12,000 60.8 (55.1), 2,000 25.2 (23.9), those prompts 66.4 (75.2).
    // What the cost does not see is how the tails fit beside the prefix's items.
    Ka4Cut cut = ka4_cut(a, tail_cols, part, 16, 1.f, cus * ka4_held(a.c.head_dim, a.q16, 1));
    int nc = 1;
    if (tail_cols > 16) {
        const Ka4Cut wide = ka4_cut(a, tail_cols, part, 32, a.q16 ? 1.3f : 1.45f,
                                    cus * ka4_held(a.c.head_dim, a.q16, 2));
        if (wide.cost < cut.cost) {
            cut = wide;
            nc = 2;
        }
    }
    a.tail_tiles = (int)cut.tail_tiles;
    const int64_t units = (int64_t)Hk * a.tail_tiles;
    a.tail_runs = (int)std::max<int64_t>(1, a.slots / units);
    const int64_t longest = std::max<int64_t>((int64_t)a.c.max_pages * a.c.page_size - a.shared, 1);
    a.max_runs = (int)std::min<int64_t>({a.tail_runs, 64, ceil_div(longest, KA4_LEAST * KA_ROUND), std::max<int64_t>(1, (256 << 20) / part)});
    a.direct = a.shared == 0 && a.max_runs == 1;
    a.tail_items = (int)(cut.items + (a.max_runs == 1 ? 0 : (int64_t)a.tail_runs * units));
    if (a.shared > 0) {
        const int64_t pre_units = Hk * cut.pre_tiles;
        a.pre_tiles = (int)cut.pre_tiles;
        a.pre_keys = (int)cut.pre_keys;
        a.pre_splits = (int)cut.pre_splits;
        a.pre_work = (float)pre_units * (a.pre_splits * a.fixed + ceil_div(a.shared, KA_ROUND));
        const int64_t pre = (int64_t)ceil_div((int64_t)Hk * a.pre_splits, 8) * 8 * a.pre_tiles;
        PIO_REQUIRE(pre <= 1 << 22, "pio_kv_attention: too many rows over %d shared tokens", a.shared);
        a.pre_items = (int)pre;
    }
    // (a grid has fewer than 2^32 threads)
    PIO_REQUIRE(((int64_t)a.pre_items + a.tail_items) * 256 < (int64_t)1 << 32,
                "pio_kv_attention: %d requests and %d rows are too many", a.n, a.rows);
    Scratch ws;
    if (!a.direct) {
        const size_t parts = (size_t)(a.pre_splits + a.max_runs) * a.rows * a.H;
        PIO_TRY(ws.get(parts * (a.c.head_dim + 2) * sizeof(float) + a.rows * sizeof(int), st));
        a.part_o = (float*)ws.ptr;
        a.part_ml = a.part_o + parts * a.c.head_dim;
        a.part_n = (int*)(a.part_ml + 2 * parts);
    }
    PIO_TRY(a.c.head_dim == 128 ? ka4_route<128>(a, nc, st) : ka4_route<64>(a, nc, st));
    if (a.direct) return PIO_OK;
    return a.c.head_dim == 128 ? ka4_join<128>(a, st) : ka4_join<64>(a, st);
}

int ka4_attention(KaArgs& a, int max_rows, hipStream_t st) {
    if (a.c.head_dim == 128 || a.c.head_dim == 64) return ka4_matrix(a, max_rows, st);
    PIO_REQUIRE((int64_t)a.rows * a.H < 1 << 24, "pio_kv_attention: too many rows");
    ka4_simple_kernel<<<a.rows * a.H, KA_THREADS, 0, st>>>(a);
    PIO_LAUNCHED();
    return PIO_OK;
}

}  // namespace pio
