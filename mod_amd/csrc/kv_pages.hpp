// Internals of the paged key / value cache (kv_pages.hip) that its attention
// (kv_attention.hip) uses.
#pragma once

#include "pio_common.hpp"

namespace pio {

// Bits of the status word work[0].
enum : int { KV_BAD = 1, KV_FULL = 2 };

// Checks the struct itself; `what` names the entry point.
int kv_check(const pio_kv_cache* c, const char* what);

// A cache of 4 bits as an element type (tensor_rocm.h: its layout). 8 values are a word.
struct KvMx4 {};
constexpr int KV_MX4_LEAST = 104, KV_MX4_MOST = 140, KV_MX4_NAN = 255;     // scale bytes

// Bytes of a token of one kv head.
__host__ __device__ __forceinline__ int kv_token_bytes(const pio_kv_cache& c) {
    return c.kv_dtype == PIO_MX4 ? c.head_dim / 32 * 17 : c.head_dim * (c.kv_dtype == PIO_F32 ? 4 : 2);
}

// 8 values of a block of 32 whose scale byte is `scale`.
__device__ __forceinline__ void kv_mx4_widen(uint32_t codes, int scale, float (&x)[8]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const float s = __uint_as_float((uint32_t)scale << 23);      // (255, infinite, gives NaN)
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1),
             c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1], x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
}
// The scale byte of 32 values, from the bits of the largest magnitude among them: the least exponent e with
// max < 7 * 2^e (a mantissa from 1.75 on carries), or NaN.
__device__ __forceinline__ int kv_mx4_scale(uint32_t most) {
    if (most >= 0x7f800000u) return KV_MX4_NAN;
    return min(max((int)((most + 0x200000u) >> 23) - 2, KV_MX4_LEAST), KV_MX4_MOST);
}
// 8 values as codes under a scale byte (zeros under NaN); the conversion rounds to nearest, ties to even, and saturates.
__device__ __forceinline__ uint32_t kv_mx4_codes(const float (&x)[8], int scale) {
    const float s = __uint_as_float((uint32_t)scale << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
    return scale == KV_MX4_NAN ? 0 : w;
}

// A sequence's length, or -1 for a sequence outside the cache or a length that
// its table row cannot have.
__device__ __forceinline__ int kv_seq_len(const pio_kv_cache& c, int s) {
    if (s < 0 || s >= c.max_seqs) return -1;
    const int n = c.lens[s];
    return n <= c.max_pages * c.page_size ? max(n, -1) : -1;
}
__device__ __forceinline__ int kv_log2(int p) { return 31 - __clz(p); }

}  // namespace pio
