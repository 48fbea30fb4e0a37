// Internals of the paged key / value cache (kv_pages.hip) that its attention
// (kv_attention.hip) uses.
#pragma once

#include "pio_common.hpp"

namespace pio {

// Bits of the status word work[0].
enum : int { KV_BAD = 1, KV_FULL = 2 };

// Checks the struct itself; `what` names the entry point.
int kv_check(const pio_kv_cache* c, const char* what);

// A sequence's length, or -1 for a sequence outside the cache or a length that
// its table row cannot have.
__device__ __forceinline__ int kv_seq_len(const pio_kv_cache& c, int s) {
    if (s < 0 || s >= c.max_seqs) return -1;
    const int n = c.lens[s];
    return n <= c.max_pages * c.page_size ? max(n, -1) : -1;
}
__device__ __forceinline__ int kv_log2(int p) { return 31 - __clz(p); }

}  // namespace pio
