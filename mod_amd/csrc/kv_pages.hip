// Pages of a key / value cache that many sequences share: reserve, write, fork,
// drop, compact (tensor_rocm.h). Tables, lengths and page counts live on the
// device and are changed there, so a step needs no host round trip and can be
// captured.
//
// The calls that hand out or move pages are a plan and its execution: one
// workgroup checks the requests, walks the page counts and leaves pairs
// (from, to, rows) in `work`; then the whole device copies. Fork and drop touch
// no page and run as one workgroup per request.
#include "kv_pages.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <type_traits>

namespace pio {

constexpr int KV_PLAN = 1024;          // threads of a planning workgroup
constexpr int KV_COPY = 256;
constexpr int KV_SCAN = 16;            // page counts per thread and step of a plan's walk

// ---- work: [0] status bits, [1] pairs of the plan, then
//   mark [max_seqs]        request that names a sequence
//   pairs [n_pages][3]     (from, to, rows of each head)
//   remap [n_pages]        free pages (reserve) / new page of each old one (compact)
//   held_up [max_seqs]     1: the last reserve that names a sequence was refused
// A step's calls follow each other without the host, so those behind a refused reserve have
// to find out on the device: its tokens are not there to be written or dropped.
constexpr int KV_HEAD = 16;
static inline size_t kv_work_ints(const pio_kv_cache& c) {
    return KV_HEAD + 2 * (size_t)c.max_seqs + 4 * (size_t)c.n_pages;
}
struct KvWork {
    int *status, *pairs_n, *mark, *pairs, *remap, *held_up;
};
__host__ __device__ __forceinline__ KvWork kv_work(const pio_kv_cache& c) {
    KvWork w;
    w.status = c.work;
    w.pairs_n = c.work + 1;
    w.mark = c.work + KV_HEAD;
    w.pairs = w.mark + c.max_seqs;
    w.remap = w.pairs + 3 * (int64_t)c.n_pages;
    w.held_up = w.remap + c.n_pages;
    return w;
}

int kv_check(const pio_kv_cache* c, const char* what) {
    PIO_REQUIRE(c, "%s: null cache", what);
    PIO_REQUIRE(c->kv && c->table && c->lens && c->refs && c->work, "%s: null pointer in the cache", what);
    PIO_REQUIRE(c->kv_dtype == PIO_F32 || c->kv_dtype == PIO_F16 || c->kv_dtype == PIO_MX4,
                "%s: cache dtype %d (fp32, fp16 or 4 bits)", what, c->kv_dtype);
    PIO_REQUIRE(c->n_layers > 0 && c->n_kv_heads > 0 && c->n_pages > 0 && c->max_seqs > 0 && c->max_pages > 0,
                "%s: empty cache dimension", what);
    PIO_REQUIRE(c->head_dim >= 8 && c->head_dim <= 256 && c->head_dim % 8 == 0,
                "%s: head_dim %d (a multiple of 8 up to 256)", what, c->head_dim);
    PIO_REQUIRE(c->page_size >= 1 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0,
                "%s: page_size %d (a power of two up to 1024)", what, c->page_size);
    PIO_REQUIRE(c->kv_dtype != PIO_MX4 || (c->head_dim % 32 == 0 && c->page_size >= 16),
                "%s: 4 bits, head_dim %d, page_size %d (a multiple of 32, from 16)", what, c->head_dim, c->page_size);
    // positions, and the pages or rounds of keys that 1024 requests need, are counted in 32 bits
    PIO_REQUIRE((int64_t)c->max_pages * c->page_size <= 1 << 28, "%s: table rows of over 2^28 positions", what);
    PIO_REQUIRE(c->n_pages <= 1 << 20 && c->max_seqs <= 1 << 20 && c->max_pages <= 1 << 20,
                "%s: over 2^20 pages, sequences or pages of a sequence", what);
    PIO_REQUIRE((int64_t)c->n_kv_heads * c->head_dim <= 1 << 20, "%s: n_kv_heads x head_dim over 2^20", what);
    PIO_REQUIRE(aligned16(c->kv), "%s: kv is not 16-byte aligned", what);
    for (const int32_t* p : {c->table, c->lens, c->refs, c->work})
        PIO_REQUIRE(((uintptr_t)p & 3u) == 0, "%s: int32 array not 4-byte aligned", what);
    return PIO_OK;
}

static int kv_requests(const pio_kv_cache* c, const void* a, const void* b, int n, const char* what) {
    PIO_TRY(kv_check(c, what));
    PIO_REQUIRE(n >= 0 && n <= PIO_KV_MAX_REQUESTS && n <= c->max_seqs, "%s: %d requests (0..%d)", what, n,
                std::min(PIO_KV_MAX_REQUESTS, c->max_seqs));
    PIO_REQUIRE(n == 0 || (a && b), "%s: null request list", what);
    PIO_REQUIRE(((uintptr_t)a & 3u) == 0 && ((uintptr_t)b & 3u) == 0, "%s: request list not 4-byte aligned", what);
    return PIO_OK;
}

__device__ __forceinline__ bool kv_seq_ok(const pio_kv_cache& c, int s) { return s >= 0 && s < c.max_seqs; }
// Pages that n positions take (n may be INT_MAX).
__device__ __forceinline__ int kv_pages_of(int n, int lg) { return (int)(((int64_t)n + (1 << lg) - 1) >> lg); }
// Exclusive scan over the workgroup's threads; `total` gets the sum. `red` has
// a word per wave.
__device__ __forceinline__ int kv_scan(int v, int* red, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();                   // the last call's readers are done with red
    if (lane == 63) red[w] = x;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); i++) {
        const int r = red[i];
        if (i < w) before += r;
        all += r;
    }
    total = all;
    return before + x - v;
}

// Page counts of SCAN consecutive pages from p0 (-1 behind the last page).
template <int SCAN>
__device__ __forceinline__ void kv_load_refs(const pio_kv_cache& c, int64_t p0, int (&r)[SCAN]) {
#pragma unroll
    for (int i = 0; i < SCAN; i++) r[i] = p0 + i < c.n_pages ? c.refs[p0 + i] : -1;
}

// ------------------------------------------------------------------ init ----
__global__ __launch_bounds__(KV_COPY) void kv_init_kernel(pio_kv_cache c) {
    const int64_t cells = (int64_t)c.max_seqs * c.max_pages;
    const int64_t at = (int64_t)blockIdx.x * KV_COPY + threadIdx.x, step = (int64_t)gridDim.x * KV_COPY;
    for (int64_t i = at; i < cells; i += step) c.table[i] = -1;
    for (int64_t i = at; i < c.max_seqs; i += step) {
        c.lens[i] = 0;
        kv_work(c).held_up[i] = 0;
    }
    for (int64_t i = at; i < c.n_pages; i += step) c.refs[i] = 0;
    if (at < 2) c.work[at] = 0;
}
// What was refused is known (pio_kv_status).
__global__ __launch_bounds__(KV_COPY) void kv_settle_kernel(pio_kv_cache c) {
    const KvWork w = kv_work(c);
    const int at = blockIdx.x * KV_COPY + threadIdx.x;
    if (at == 0) *w.status = 0;
    for (int i = at; i < c.max_seqs; i += gridDim.x * KV_COPY) w.held_up[i] = 0;
}

// --------------------------------------------------------------- reserve ----
// One workgroup: a chain of waits, for the requests, their lengths, their last pages
// and those pages' counts; the counts that free pages are found by are loaded first.
// SCAN pages to a thread and step: 1 where one step then holds all pages, as its code is
// the shorter (a plan over 1024 pages or fewer runs each instruction once).
// off[i]: pages that the requests before i take; held[i]: pages that request i's
// sequence has, doubled, plus one if its last is copied.
constexpr int KV_LIST = 2048;          // free pages listed in LDS (in remap, if more are needed)
template <int SCAN>
__global__ __launch_bounds__(KV_PLAN) void kv_reserve_plan_kernel(pio_kv_cache c, const int32_t* __restrict__ seq,
                                                                 const int32_t* __restrict__ count, int n) {
    __shared__ int off[PIO_KV_MAX_REQUESTS], held[PIO_KV_MAX_REQUESTS], list[KV_LIST], red[KV_PLAN / 64], bad, pairs;
    const KvWork w = kv_work(c);
    const int tid = threadIdx.x, lg = kv_log2(c.page_size);
    int r[SCAN];
    kv_load_refs<SCAN>(c, (int64_t)tid * SCAN, r);
    if (tid == 0) bad = pairs = 0;
    for (int i = tid; i < n; i += KV_PLAN)
        if (kv_seq_ok(c, seq[i])) w.mark[seq[i]] = i;
    __syncthreads();
    int total = 0;
    for (int i0 = 0; i0 < n; i0 += KV_PLAN) {
        const int i = i0 + tid;
        int need = 0, wrong = 0;
        if (i < n) {
            const int s = seq[i], k = count[i];
            int L = -1;
            if (kv_seq_ok(c, s)) {
                const int named = w.mark[s];
                L = kv_seq_len(c, s);
                if (named != i) L = -1;
            }
            if (L < 0 || k < 0) {
                wrong = KV_BAD;
            } else if ((int64_t)L + k > (int64_t)c.max_pages * c.page_size) {
                wrong = KV_FULL;
            } else {
                const int h = kv_pages_of(L, lg);
                int copy = 0;
                if (k > 0 && (L & (c.page_size - 1))) {
                    const int last = c.table[(int64_t)s * c.max_pages + h - 1];
                    if (last < 0 || last >= c.n_pages) wrong = KV_BAD;
                    else copy = c.refs[last] > 1;
                }
                need = copy + kv_pages_of(L + k, lg) - h;
                if (need > c.n_pages) wrong = KV_FULL, need = 0;
                held[i] = 2 * h + copy;
            }
        }
        if (wrong) atomicOr(&bad, wrong);
        int sum;
        const int before = kv_scan(need, red, sum);
        // more than every page there is: no need to count on
        if (i < n) off[i] = total + before;
        total = min(total + sum, c.n_pages + 1);
    }
    __syncthreads();
    // the lowest free pages, as many as are needed
    int found = 0;
    if (!bad && total <= c.n_pages) {
        for (int64_t p0 = 0; p0 < c.n_pages && found < total; p0 += KV_PLAN * SCAN) {
            int free = 0, sum;
            if (p0) kv_load_refs<SCAN>(c, p0 + (int64_t)tid * SCAN, r);
#pragma unroll
            for (int j = 0; j < SCAN; j++) free += r[j] == 0;
            int at = found + kv_scan(free, red, sum);
#pragma unroll
            for (int j = 0; j < SCAN; j++)
                if (r[j] == 0) {
                    const int page = (int)(p0 + (int64_t)tid * SCAN + j);
                    if (at < total) {
                        if (total <= KV_LIST) list[at] = page;
                        else w.remap[at] = page;
                    }
                    at++;
                }
            found += sum;
        }
    }
    if (bad || found < total) {
        for (int i = tid; i < n; i += KV_PLAN)
            if (kv_seq_ok(c, seq[i])) w.held_up[seq[i]] = 1;
        if (tid == 0) {
            *w.pairs_n = 0;
            atomicOr(w.status, bad ? bad : KV_FULL);
        }
        return;
    }
    __syncthreads();
    // page k of all goes to the request whose pages begin at or before k
    for (int k = tid; k < total; k += KV_PLAN) {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (off[mid] <= k) lo = mid;
            else hi = mid - 1;
        }
        const int s = seq[lo], h = held[lo] >> 1, copy = held[lo] & 1, j = k - off[lo];
        const int page = total <= KV_LIST ? list[k] : w.remap[k];
        int32_t* row = c.table + (int64_t)s * c.max_pages;
        c.refs[page] = 1;
        if (copy && j == 0) {
            const int last = row[h - 1], at = 3 * atomicAdd(&pairs, 1);
            w.pairs[at] = last;
            w.pairs[at + 1] = page;
            w.pairs[at + 2] = c.lens[s] & (c.page_size - 1);
            atomicAdd(&c.refs[last], -1);
            row[h - 1] = page;
        } else {
            row[h + j - copy] = page;
        }
    }
    __syncthreads();
    for (int i = tid; i < n; i += KV_PLAN) {
        c.lens[seq[i]] += count[i];
        w.held_up[seq[i]] = 0;
    }
    if (tid == 0) *w.pairs_n = pairs;
}

// ------------------------------------------------------------- page copy ----
// Pairs of the plan: the first rows of each head (of a cache of 4 bits, whose scales lie
// behind a page's codes, the whole page), in every layer's k and v; a workgroup
// takes a plane (layer, k or v) of a pair, n_kv_heads runs of rows * head_dim elements.
// tables: also rewrites the tables by remap and moves the pages' counts (compact).
//   Bytes bound it, from memory: 84 whole pages of 16 x 8 x 128 fp16 in 56 planes, half of
// them moved, 35 us, 4.3 TB/s; 5 rows of 16 of 64 pages 19 us. One load of a thread at a
// time: with 4 in flight before the first store, 4 KB apart, 42 and 31 us.
__global__ __launch_bounds__(KV_COPY) void kv_copy_kernel(pio_kv_cache c, int tables) {
    const KvWork w = kv_work(c);
    const int pairs = min(*w.pairs_n, c.n_pages), planes = 2 * c.n_layers, tid = threadIdx.x;
    const int token_b = kv_token_bytes(c);
    const int64_t head_b = (int64_t)c.page_size * token_b, page_b = head_b * c.n_kv_heads;
    const int pitch = (int)(head_b / 16);
    for (int pair = blockIdx.y; pair < pairs; pair += gridDim.y) {
        const int from = w.pairs[3 * pair], to = w.pairs[3 * pair + 1], rows = w.pairs[3 * pair + 2];
        // (a plan that something else wrote over may not lead out of the cache)
        if ((unsigned)from >= (unsigned)c.n_pages || (unsigned)to >= (unsigned)c.n_pages ||
            (unsigned)rows > (unsigned)c.page_size)
            continue;
        const int run = c.kv_dtype == PIO_MX4 ? pitch : rows * token_b / 16, all = run * c.n_kv_heads;
        const uint32_t magic = run > 1 ? 0xffffffffu / run + 1 : 0;     // u / run, or one more
        auto at = [&](int u) {
            if (run == pitch) return u;
            int h = magic ? (int)__umulhi((uint32_t)u, magic) : u;
            h -= h * run > u;
            return h * pitch + u - h * run;
        };
        for (int plane = blockIdx.x; plane < planes; plane += gridDim.x) {
            const uint4* src = (const uint4*)((const char*)c.kv + ((int64_t)plane * c.n_pages + from) * page_b);
            uint4* dst = (uint4*)((char*)c.kv + ((int64_t)plane * c.n_pages + to) * page_b);
#pragma unroll 1
            for (int u = tid; u < all; u += KV_COPY) dst[at(u)] = src[at(u)];
        }
        if (tables && blockIdx.x == 0 && tid == 0) {
            c.refs[to] = c.refs[from];
            c.refs[from] = 0;
        }
    }
    if (tables && pairs > 0) {
        const int64_t cells = (int64_t)c.max_seqs * c.max_pages, step = (int64_t)gridDim.x * gridDim.y * KV_COPY;
        for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * KV_COPY + tid; i < cells; i += step) {
            const int p = c.table[i];
            if (p >= 0 && p < c.n_pages) c.table[i] = w.remap[p];
        }
    }
}

static int kv_copy(const pio_kv_cache& c, int64_t most_pairs, bool tables, hipStream_t st) {
    // a workgroup to each plane of a pair, up to some rounds of the whole device
    const int planes = (int)std::min<int64_t>(2 * (int64_t)c.n_layers, 4096);
    const int64_t cells = tables ? ((int64_t)c.max_seqs * c.max_pages + KV_COPY - 1) / KV_COPY : 0;
    const int64_t most = std::max(most_pairs, std::min<int64_t>(2048, cells) / planes);
    const dim3 grid(planes, (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, 16384 / planes)));
    kv_copy_kernel<<<grid, KV_COPY, 0, st>>>(c, tables);
    PIO_LAUNCHED();
    return PIO_OK;
}

// --------------------------------------------------------------- compact ----
// The k-th free page below the number of pages in use takes the k-th page in use from
// there on. Up to KV_PLAN pages: a page to a thread, and live[k] the k-th in use.
__global__ __launch_bounds__(KV_PLAN) void kv_compact_few_kernel(pio_kv_cache c) {
    __shared__ int red[KV_PLAN / 64], live[KV_PLAN], below;
    const KvWork w = kv_work(c);
    const int p = threadIdx.x;
    int r[1], used;
    kv_load_refs<1>(c, p, r);
    const bool in_use = r[0] > 0;
    const int before = kv_scan(in_use, red, used);
    if (in_use) live[before] = p;
    if (p == min(used, KV_PLAN - 1)) below = before;       // in use below `used`
    __syncthreads();
    if (p < c.n_pages && !(in_use && p >= used)) w.remap[p] = p;
    if (p < used && !in_use) {
        const int k = p - before, from = live[below + k];
        w.pairs[3 * k] = from;
        w.pairs[3 * k + 1] = p;
        w.pairs[3 * k + 2] = c.page_size;
        w.remap[from] = p;
    }
    if (p == 0) *w.pairs_n = used == KV_PLAN ? 0 : used - below;
}
// Any number of pages, in steps.
__global__ __launch_bounds__(KV_PLAN) void kv_compact_plan_kernel(pio_kv_cache c) {
    __shared__ int red[KV_PLAN / 64];
    const KvWork w = kv_work(c);
    const int tid = threadIdx.x;
    constexpr int STEP = KV_PLAN * KV_SCAN;
    int used = 0, r[KV_SCAN];
    for (int64_t p0 = 0; p0 < c.n_pages; p0 += STEP) {
        int live = 0, sum;
        kv_load_refs<KV_SCAN>(c, p0 + (int64_t)tid * KV_SCAN, r);
#pragma unroll
        for (int j = 0; j < KV_SCAN; j++) live += r[j] > 0;
        kv_scan(live, red, sum);
        used += sum;
    }
    int holes = 0, movers = 0;
    for (int64_t p0 = 0; p0 < c.n_pages; p0 += STEP) {
        const int64_t base = p0 + (int64_t)tid * KV_SCAN;
        int hole = 0, mover = 0, sum;
        kv_load_refs<KV_SCAN>(c, base, r);
#pragma unroll
        for (int j = 0; j < KV_SCAN; j++) {
            hole += base + j < used && r[j] <= 0;
            mover += base + j >= used && r[j] > 0;
        }
        int h = holes + kv_scan(hole, red, sum);
        holes += sum;
        int m = movers + kv_scan(mover, red, sum);
        movers += sum;
#pragma unroll
        for (int j = 0; j < KV_SCAN; j++) {
            const int64_t p = base + j;
            if (p < used && r[j] <= 0) w.pairs[3 * h++ + 1] = (int)p;
            else if (p >= used && r[j] > 0) w.pairs[3 * m++] = (int)p;
            if (p < c.n_pages) w.remap[p] = (int)p;
        }
    }
    __syncthreads();
    // as many of one as of the other
    for (int k = tid; k < movers; k += KV_PLAN) {
        w.pairs[3 * k + 2] = c.page_size;
        w.remap[w.pairs[3 * k]] = w.pairs[3 * k + 1];
    }
    if (tid == 0) *w.pairs_n = movers;
}

// Rows of a cache of 4 bits share lines (two rows' codes, all of a page's scales), and each XCD has its own L2:
// neighbouring rows on one XCD, so that a line is read or written once. A grid's workgroups go round the XCDs.
__device__ __forceinline__ int kv_row_of(int block, int rows) {
    const int each = (rows + 7) >> 3, x = block & 7, full = rows & 7 ? rows & 7 : 8;     // the last XCDs have one fewer
    return x < full ? x * each + (block >> 3) : full * each + (x - full) * (each - 1) + (block >> 3);
}
// Quotients by a few fixed numbers: u / run, u < 2^31.
struct KvDiv {
    uint32_t run, magic;
    __device__ __forceinline__ explicit KvDiv(uint32_t run) : run(run), magic(run > 1 ? 0xffffffffu / run + 1 : 0) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t u) const {
        uint32_t q = magic ? __umulhi(u, magic) : u;           // or one more
        return q - (q * run > u);
    }
};
// Pieces of 8 elements of a row, [layer][k, v][head]: which one `u` is.
struct KvPiece {
    int l, kind, e, h, piece;          // e: of the row, piece: of the head
    __device__ __forceinline__ KvPiece(uint32_t u, const KvDiv& by_layer, const KvDiv& by_head) {
        l = (int)by_layer(u);
        const int in = (int)u - l * (int)by_layer.run, width = (int)by_layer.run / 2;
        kind = in >= width;
        e = in - kind * width;
        h = (int)by_head((uint32_t)e);
        piece = e - h * (int)by_head.run;
    }
};
constexpr int KV_FLIGHT = 4;           // pieces of a thread in flight
typedef uint32_t KvU4 __attribute__((ext_vector_type(4)));

// ----------------------------------------------------------------- write ----
// A workgroup takes one row through a few layers: it finds the row's request,
// then moves k and v in pieces of 8 elements. Bytes bound it: 336 rows of 28 layers,
// fp32 to fp16, 32 us, 3.5 TB/s; few rows, the chain of loads that says where a row goes
// and whether it may: 8 rows of one layer 4.3 us, 3.6 without its checks. In 4 bits the four
// threads of a block of 32 values share its largest magnitude; 3,941 rows of 28 layers of 8 x 128, fp16, 113 us,
// 5.1 TB/s (150 with loads through the caches).
template <typename XT, typename KT>
__global__ __launch_bounds__(KV_COPY) void kv_write_kernel(pio_kv_cache c, int layer, int layers,
                                                          const int32_t* __restrict__ seq,
                                                          const int32_t* __restrict__ row_start, int n,
                                                          const XT* __restrict__ k, const XT* __restrict__ v,
                                                          int64_t row_stride, int64_t layer_stride, int per_block) {
    __shared__ int found, named, where[2];     // the row's request, its sequence; page, row in it
    constexpr bool MX4 = std::is_same_v<KT, KvMx4>;
    const int row = MX4 ? kv_row_of(blockIdx.x, gridDim.x) : (int)blockIdx.x, tid = threadIdx.x, lg = kv_log2(c.page_size);
    if (tid == 0) found = where[0] = -1;
    __syncthreads();
    int s = -1, back = 0, first = -1;          // (first: what thread tid's first request with rows names)
    for (int i = tid; i < n; i += KV_COPY) {
        const int r0 = row_start[i], r1 = row_start[i + 1], si = seq[i];
        if (i == tid && r1 > r0) first = si;
        if (row < r0 || row >= r1) continue;
        found = i;
        named = s = si;
        back = r1 - row;
    }
    __syncthreads();
    const int req = found;
    if (req < 0) return;               // behind the last request
    const int width = c.n_kv_heads * c.head_dim / 8, per_head = c.head_dim / 8;
    const int l0 = blockIdx.y * per_block, l1 = min(layers, l0 + per_block);
    auto from = [&](int l, int u) {
        const int kind = u >= width;
        return (kind ? v : k) + l * layer_stride + row * row_stride + 8 * (u - kind * width);
    };
    float x[8];
    const KvDiv by_layer(2 * width), by_head(per_head);
    const int pieces = (l1 - l0) * 2 * width;
    Raw8<XT> raw[KV_FLIGHT];
    auto load = [&](int u0) {
#pragma unroll
        for (int i = 0; i < KV_FLIGHT; i++) {
            if (u0 + i * KV_COPY >= pieces) break;
            const KvPiece p(u0 + i * KV_COPY, by_layer, by_head);
            // (past the caches: they are not read again, the pages are)
            const KvU4* at = (const KvU4*)((p.kind ? v : k) + (l0 + p.l) * layer_stride + row * row_stride + 8 * p.e);
#pragma unroll
            for (int j = 0; j < (int)sizeof(XT) / 2; j++)
                raw[i].u[j] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(at + j));
        }
    };
    // under the way of the checks below
    if constexpr (MX4) load(tid);
    else if (tid < 2 * width) load8<XT>(from(l0, tid), x);
    if (tid == req % KV_COPY) {
        int page = -1, pos = -1;
        bool held_up = false;
        if (kv_seq_ok(c, s)) {
            held_up = kv_work(c).held_up[s];               // its tokens have no room: reported by the reserve
            pos = kv_seq_len(c, s) - back;
            if (pos >= 0) page = c.table[(int64_t)s * c.max_pages + (pos >> lg)];
        }
        // (a page that another table entry holds too is not this sequence's to change)
        if (held_up) {
        } else if (page < 0 || page >= c.n_pages || c.refs[page] > 1) {
            atomicOr(kv_work(c).status, KV_BAD);
        } else {
            where[0] = page;
            where[1] = pos & (c.page_size - 1);
        }
    }
    // a sequence that an earlier request with rows names is left to that one
    int twice = tid < req && first == named;
    for (int i = tid + KV_COPY; i < req; i += KV_COPY) twice |= seq[i] == named && row_start[i + 1] > row_start[i];
    if (__syncthreads_or(twice)) {
        if (tid == 0) atomicOr(kv_work(c).status, KV_BAD);
        return;
    }
    if (where[0] < 0) return;          // without room, or refused above
    if constexpr (MX4) {
        const int64_t head = (int64_t)c.page_size * kv_token_bytes(c), plane = head * c.n_kv_heads * c.n_pages;
        char* base = (char*)c.kv + head * c.n_kv_heads * where[0] + 2 * (layer + l0) * plane;
        for (int u0 = tid; u0 < pieces; u0 += KV_FLIGHT * KV_COPY) {
            if (u0 != tid) load(u0);
#pragma unroll
            for (int i = 0; i < KV_FLIGHT; i++) {
                const int u = u0 + i * KV_COPY;
                if (u >= pieces) break;                            // (all four threads of a block, or none)
                const KvPiece p(u, by_layer, by_head);
                raw8_widen<XT>(raw[i], x);
                uint32_t most = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(x[j]) & 0x7fffffffu);
                most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, DPP_XOR1, 0xF, 0xF, false));
                most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, DPP_XOR2, 0xF, 0xF, false));
                const int scale = kv_mx4_scale(most);
                char* to = base + (2 * p.l + p.kind) * plane + p.h * head;
                *(uint32_t*)(to + where[1] * (c.head_dim / 2) + 4 * p.piece) = kv_mx4_codes(x, scale);
                if ((p.piece & 3) == 0)
                    to[c.page_size * (c.head_dim / 2 + (p.piece >> 2)) + where[1]] = (char)scale;
            }
        }
    } else {
        const int64_t head = (int64_t)c.page_size * c.head_dim, plane = head * c.n_kv_heads * c.n_pages;
        KT* base = (KT*)c.kv + head * c.n_kv_heads * where[0] + (int64_t)where[1] * c.head_dim;
        for (int l = l0; l < l1; l++) {
            for (int u = tid; u < 2 * width; u += KV_COPY) {
                const int kind = u >= width, e = u - kind * width, h = e / per_head;
                if (l != l0 || u != tid) load8<XT>(from(l, u), x);
                KT* to = base + (2 * (layer + l) + kind) * plane + h * head + 8 * (e - h * per_head);
                __attribute__((aligned(16))) KT y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = from_f32<KT>(x[j]);   // to nearest, ties to even
#pragma unroll
                for (int j = 0; j < (int)sizeof(KT) / 2; j++) ((uint4*)to)[j] = ((const uint4*)y)[j];
            }
        }
    }
}

// ------------------------------------------------------------------ read ----
// The way back: a workgroup takes one row through a few layers, in pieces of 8 elements. Bytes bound it: 1,805 rows of
// 28 layers of 8 x 128 out of 4 bits to fp16 40 us, 6.5 TB/s (67 with stores through the caches; some pages are in the
// memory-side cache), out of fp16 to fp16 62, 6.6 TB/s, out of fp32 to fp16 120, 5.2, to fp32 187, 4.4 (out of fp16 190: a
// thread's two stores of 16 bytes are half a line apart from its neighbours').
template <typename KT, typename YT>
__global__ __launch_bounds__(KV_COPY) void kv_read_kernel(pio_kv_cache c, int layer, int layers,
                                                         const int32_t* __restrict__ seq,
                                                         const int32_t* __restrict__ row_start,
                                                         const int32_t* __restrict__ first, int n, YT* __restrict__ k,
                                                         YT* __restrict__ v, int64_t row_stride, int64_t layer_stride,
                                                         int per_block) {
    __shared__ int where[3];                   // page, row in it; whether a request has the row
    const int row = kv_row_of(blockIdx.x, gridDim.x), tid = threadIdx.x, lg = kv_log2(c.page_size);
    if (tid == 0) where[0] = where[2] = -1;
    __syncthreads();
    for (int i = tid; i < n; i += KV_COPY) {
        const int r0 = row_start[i], r1 = row_start[i + 1], s = seq[i], f = first ? first[i] : 0;
        if (row < r0 || row >= r1) continue;
        const int L = kv_seq_len(c, s);
        const int64_t pos = first ? f + ((int64_t)row - r0) : L - ((int64_t)r1 - row);
        bool has = pos >= 0 && pos < L;
        int page = -1, held_up = 0;
        if (L >= 0) {                      // (both loads at once)
            held_up = kv_work(c).held_up[s];
            page = c.table[(int64_t)s * c.max_pages + (has ? pos >> lg : 0)];
        }
        // Behind a refused reserve the last tokens are not those that the caller counts from, and what is not there the
        // reserve has reported.
        has = has && (first || !held_up);
        if (!has) page = -1;
        if (page >= 0 && page < c.n_pages) {
            where[0] = page;
            where[1] = (int)(pos & (c.page_size - 1));
        } else if (has || !held_up) {
            atomicOr(kv_work(c).status, KV_BAD);
        }
        where[2] = i;
    }
    __syncthreads();
    if (where[2] < 0) return;          // behind the last request
    const bool there = where[0] >= 0;
    const int at = there ? where[1] : 0, l0 = blockIdx.y * per_block;
    const int64_t head = (int64_t)c.page_size * kv_token_bytes(c), plane = head * c.n_kv_heads * c.n_pages;
    const char* base = (const char*)c.kv + head * c.n_kv_heads * (there ? where[0] : 0) + 2 * (layer + l0) * plane;
    const int width = c.n_kv_heads * c.head_dim / 8, pieces = (min(layers, l0 + per_block) - l0) * 2 * width;
    const KvDiv by_layer(2 * width), by_head(c.head_dim / 8);
    for (int u0 = tid; u0 < pieces; u0 += KV_FLIGHT * KV_COPY) {
        uint32_t codes[KV_FLIGHT], scale[KV_FLIGHT];
        Raw8<KT> raw[KV_FLIGHT];
#pragma unroll
        for (int i = 0; i < KV_FLIGHT; i++) {
            if (u0 + i * KV_COPY >= pieces) break;
            const KvPiece p(u0 + i * KV_COPY, by_layer, by_head);
            const char* from = base + (2 * p.l + p.kind) * plane + p.h * head;
            if constexpr (std::is_same_v<KT, KvMx4>) {
                codes[i] = *(const uint32_t*)(from + at * (c.head_dim / 2) + 4 * p.piece);
                scale[i] = (uint8_t)from[c.page_size * (c.head_dim / 2 + (p.piece >> 2)) + at];
            } else {
                raw[i] = raw8_load<KT>((const KT*)from + (int64_t)at * c.head_dim + 8 * p.piece);
            }
        }
#pragma unroll
        for (int i = 0; i < KV_FLIGHT; i++) {
            const int u = u0 + i * KV_COPY;
            if (u >= pieces) break;
            const KvPiece p(u, by_layer, by_head);
            float x[8];
            if constexpr (std::is_same_v<KT, KvMx4>) kv_mx4_widen(codes[i], scale[i], x);
            else raw8_widen<KT>(raw[i], x);
            __attribute__((aligned(16))) YT y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = from_f32<YT>(there ? x[j] : NAN);
            // (past the caches, which have the pages to hold)
            KvU4* to = (KvU4*)((p.kind ? v : k) + (l0 + p.l) * layer_stride + row * row_stride + 8 * p.e);
#pragma unroll
            for (int j = 0; j < (int)sizeof(YT) / 2; j++) __builtin_nontemporal_store(((const KvU4*)y)[j], to + j);
        }
    }
}

// ------------------------------------------------------------ fork, drop ----
// A workgroup per request. Which requests are wrong is decided from what no
// request of the call writes (a source is never a target), so each decides alone.
__global__ __launch_bounds__(KV_COPY) void kv_fork_kernel(pio_kv_cache c, const int32_t* __restrict__ src,
                                                         const int32_t* __restrict__ dst, int n) {
    const int i = blockIdx.x, tid = threadIdx.x, lg = kv_log2(c.page_size);
    const int s = src[i], d = dst[i];
    int bad = !kv_seq_ok(c, s) || !kv_seq_ok(c, d);
    for (int j = tid; j < n; j += KV_COPY) bad |= src[j] == d || (j < i && dst[j] == d);
    int L = 0, pages = 0, first = 0;
    if (kv_seq_ok(c, s) && kv_seq_ok(c, d)) {
        const int32_t* row = c.table + (int64_t)s * c.max_pages;
        if (tid < c.max_pages) first = row[tid];       // beside the length, not behind it
        L = kv_seq_len(c, s);
        // a target that an earlier request names is refused above, whatever its length is by now
        bad |= L < 0 || c.lens[d] != 0;
        pages = L < 0 ? 0 : kv_pages_of(L, lg);
        bad |= tid < pages && (first < 0 || first >= c.n_pages);
        for (int j = tid + KV_COPY; j < pages; j += KV_COPY) bad |= row[j] < 0 || row[j] >= c.n_pages;
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0) atomicOr(kv_work(c).status, KV_BAD);
        return;
    }
    for (int j = tid; j < pages; j += KV_COPY) {
        const int p = j == tid ? first : c.table[(int64_t)s * c.max_pages + j];
        c.table[(int64_t)d * c.max_pages + j] = p;
        atomicAdd(&c.refs[p], 1);
    }
    if (tid == 0) {
        c.lens[d] = L;
        kv_work(c).held_up[d] = 0;     // a new sequence
    }
}

__global__ __launch_bounds__(KV_COPY) void kv_drop_kernel(pio_kv_cache c, const int32_t* __restrict__ seq,
                                                         const int32_t* __restrict__ count, int n) {
    const int i = blockIdx.x, tid = threadIdx.x, lg = kv_log2(c.page_size);
    const int s = seq[i], k = count ? count[i] : INT_MAX;
    int bad = !kv_seq_ok(c, s) || k < 0;
    for (int j = tid; j < i; j += KV_COPY) bad |= seq[j] == s;
    bad = __syncthreads_or(bad);
    // (a sequence that an earlier request names is left to that one)
    const int L = bad ? -1 : kv_seq_len(c, s);
    if (L < 0) {
        if (tid == 0) atomicOr(kv_work(c).status, KV_BAD);
        return;
    }
    if (count && kv_work(c).held_up[s]) return;            // the tokens that it would take back never came
    const int left = L > k ? L - k : 0, p1 = kv_pages_of(L, lg);
    __syncthreads();                   // every thread has read the length
    for (int j = kv_pages_of(left, lg) + tid; j < p1; j += KV_COPY) {
        int32_t* cell = c.table + (int64_t)s * c.max_pages + j;
        const int p = *cell;
        *cell = -1;
        if (p >= 0 && p < c.n_pages) atomicAdd(&c.refs[p], -1);
        else atomicOr(kv_work(c).status, KV_BAD);
    }
    if (tid == 0) {
        c.lens[s] = left;
        if (!count) kv_work(c).held_up[s] = 0;
    }
}

}  // namespace pio

using namespace pio;

PIO_EXPORT size_t pio_kv_work_bytes(const pio_kv_cache* c) {
    if (!c || c->max_seqs <= 0 || c->n_pages <= 0) return 0;
    return kv_work_ints(*c) * sizeof(int32_t);
}

PIO_EXPORT int pio_kv_work_create(pio_kv_cache* c, int device) {
    PIO_REQUIRE(c, "pio_kv_work_create: null cache");
    c->work = nullptr;
    const size_t bytes = pio_kv_work_bytes(c);
    PIO_REQUIRE(bytes, "pio_kv_work_create: empty cache dimension");
    PIO_REQUIRE(device >= 0, "pio_kv_work_create: device %d", device);
    PIO_REQUIRE(!capture_id(current_stream()), "pio_kv_work_create: the stream is capturing");
    return device_own((void**)&c->work, bytes, device);
}

PIO_EXPORT void pio_kv_work_destroy(pio_kv_cache* c, int device) {
    if (!c || !c->work) return;
    device_disown(c->work, device);
    c->work = nullptr;
}

PIO_EXPORT int pio_kv_init(const pio_kv_cache* c, void* stream) {
    PIO_TRY(kv_check(c, "pio_kv_init"));
    const int64_t cells = std::max<int64_t>((int64_t)c->max_seqs * c->max_pages, c->n_pages);
    const unsigned grid = (unsigned)std::min<int64_t>(2048, (cells + KV_COPY - 1) / KV_COPY);
    kv_init_kernel<<<grid, KV_COPY, 0, pick_stream(stream)>>>(*c);
    PIO_LAUNCHED();
    return PIO_OK;
}

PIO_EXPORT int pio_kv_status(const pio_kv_cache* c, void* stream) {
    PIO_TRY(kv_check(c, "pio_kv_status"));
    hipStream_t st = pick_stream(stream);
    PIO_REQUIRE(!capture_id(st), "pio_kv_status: the stream is capturing (it cannot be waited for)");
    int bits = 0;
    PIO_HIP(hipMemcpyAsync(&bits, c->work, sizeof(int), hipMemcpyDeviceToHost, st));
    PIO_HIP(hipStreamSynchronize(st));
    if (!bits) return PIO_OK;
    kv_settle_kernel<<<std::min(ceil_div(c->max_seqs, KV_COPY), 1024), KV_COPY, 0, st>>>(*c);
    PIO_LAUNCHED();
    PIO_HIP(hipStreamSynchronize(st));
    if (bits & KV_BAD)
        return set_error(PIO_ERR_INVALID, "kv cache: a call named a sequence, count or page that it does not have, one "
                                          "sequence twice, forked onto a sequence that is not empty, or wrote "
                                          "into a page that several sequences hold");
    return set_error(PIO_ERR_OOM, "kv cache: pio_kv_reserve found too few free pages or too short table rows");
}

PIO_EXPORT int pio_kv_reserve(const pio_kv_cache* c, const int32_t* seq, const int32_t* count, int n, void* stream) {
    PIO_TRY(kv_requests(c, seq, count, n, "pio_kv_reserve"));
    if (n == 0) return PIO_OK;
    hipStream_t st = pick_stream(stream);
    if (c->n_pages <= KV_PLAN) kv_reserve_plan_kernel<1><<<1, KV_PLAN, 0, st>>>(*c, seq, count, n);
    else kv_reserve_plan_kernel<KV_SCAN><<<1, KV_PLAN, 0, st>>>(*c, seq, count, n);
    PIO_LAUNCHED();
    return kv_copy(*c, n, false, st);
}

PIO_EXPORT int pio_kv_write(const pio_kv_cache* c, int layer, int layers, const int32_t* seq, const int32_t* row_start,
                            int n, const void* k, const void* v, int dtype, int rows, int64_t row_stride,
                            int64_t layer_stride, void* stream) {
    const char* nm = "pio_kv_write";
    PIO_TRY(kv_requests(c, seq, row_start, n, nm));
    PIO_REQUIRE(layer >= 0 && layers >= 0 && layers <= c->n_layers - layer, "%s: layers %d + %d of %d", nm, layer, layers,
                c->n_layers);
    PIO_REQUIRE(dtype == PIO_F32 || dtype == PIO_F16, "%s: dtype %d (fp32 or fp16)", nm, dtype);
    PIO_REQUIRE(rows >= 0 && rows < 1 << 24, "%s: %d rows (fewer than 2^24)", nm, rows);    // (2^32 threads of a grid)
    if (n == 0 || rows == 0 || layers == 0) return PIO_OK;
    PIO_REQUIRE(k && v, "%s: null k or v", nm);
    PIO_REQUIRE(aligned16(k) && aligned16(v), "%s: k or v not 16-byte aligned", nm);
    const int64_t width = (int64_t)c->n_kv_heads * c->head_dim;
    if (row_stride == 0) row_stride = width;
    if (layer_stride == 0) layer_stride = (int64_t)rows * row_stride;
    PIO_REQUIRE(row_stride % 8 == 0 && layer_stride % 8 == 0 && row_stride >= width && layer_stride >= 0,
                "%s: strides %lld, %lld (multiples of 8, rows of %lld)", nm, (long long)row_stride,
                (long long)layer_stride, (long long)width);
    // enough workgroups for the device, and no more: each looks its row up once
    const int per_block = (int)std::max<int64_t>(1, std::min<int64_t>({layers, (int64_t)rows * layers / (c->kv_dtype == PIO_MX4 ? 4096 : 2048), (1 << 28) / width}));
    const dim3 grid(rows, ceil_div(layers, per_block));
    PIO_REQUIRE(grid.y <= 65535, "%s: too many layers", nm);
    hipStream_t st = pick_stream(stream);
#define KV_WRITE(XT, KT)                                                                                             \
    kv_write_kernel<XT, KT><<<grid, KV_COPY, 0, st>>>(*c, layer, layers, seq, row_start, n, (const XT*)k, (const XT*)v, \
                                                     row_stride, layer_stride, per_block)
    if (dtype == PIO_F32) {
        if (c->kv_dtype == PIO_F32) KV_WRITE(float, float);
        else if (c->kv_dtype == PIO_F16) KV_WRITE(float, _Float16);
        else KV_WRITE(float, KvMx4);
    } else {
        if (c->kv_dtype == PIO_F32) KV_WRITE(_Float16, float);
        else if (c->kv_dtype == PIO_F16) KV_WRITE(_Float16, _Float16);
        else KV_WRITE(_Float16, KvMx4);
    }
#undef KV_WRITE
    PIO_LAUNCHED();
    return PIO_OK;
}

// Whether a row of k shares elements with one of v, `bytes` behind k: rows and layers of `width` elements that do not overlap
// among themselves. The greater of the strides is at least as long as all that the smaller one spans.
static bool kv_rows_meet(int64_t bytes, int size, int64_t width, int rows, int64_t row_stride, int layers, int64_t layer_stride) {
    if (layers == 1) layer_stride = INT64_MAX / 4;
    const bool rows_within = row_stride <= layer_stride;
    const int64_t s2 = rows_within ? layer_stride : row_stride, s1 = rows_within ? row_stride : layer_stride;
    const int64_t n2 = rows_within ? layers : rows, n1 = rows_within ? rows : layers;
    const int64_t d = (bytes < 0 ? -bytes : bytes) / size;                 // (both are 16-byte aligned)
    for (int k2 = 0; k2 < 2; k2++) {
        const int64_t off = std::abs(d - std::min(d / s2 + k2, n2 - 1) * s2);
        for (int k1 = 0; k1 < 2; k1++)
            if (std::abs(off - std::min(off / s1 + k1, n1 - 1) * s1) < width) return true;
    }
    return false;
}

PIO_EXPORT int pio_kv_read(const pio_kv_cache* c, int layer, int layers, const int32_t* seq, const int32_t* row_start,
                           const int32_t* first, int n, void* k, void* v, int dtype, int rows, int64_t row_stride,
                           int64_t layer_stride, void* stream) {
    const char* nm = "pio_kv_read";
    PIO_TRY(kv_check(c, nm));
    PIO_REQUIRE(n >= 0 && n <= PIO_KV_MAX_REQUESTS, "%s: %d requests (0..%d)", nm, n, PIO_KV_MAX_REQUESTS);
    PIO_REQUIRE(n == 0 || (seq && row_start), "%s: null request list", nm);
    for (const int32_t* p : {seq, row_start, first})
        PIO_REQUIRE(((uintptr_t)p & 3u) == 0, "%s: request list not 4-byte aligned", nm);
    PIO_REQUIRE(layer >= 0 && layers >= 0 && layers <= c->n_layers - layer, "%s: layers %d + %d of %d", nm, layer, layers,
                c->n_layers);
    PIO_REQUIRE(dtype == PIO_F32 || dtype == PIO_F16, "%s: dtype %d (fp32 or fp16)", nm, dtype);
    PIO_REQUIRE(rows >= 0 && rows < 1 << 24, "%s: %d rows (fewer than 2^24)", nm, rows);    // (2^32 threads of a grid)
    if (n == 0 || rows == 0 || layers == 0) return PIO_OK;
    PIO_REQUIRE(k && v && k != v, "%s: null k or v, or both the same", nm);
    PIO_REQUIRE(aligned16(k) && aligned16(v), "%s: k or v not 16-byte aligned", nm);
    const int64_t width = (int64_t)c->n_kv_heads * c->head_dim;
    if (row_stride == 0) row_stride = width;
    if (layer_stride == 0) layer_stride = (int64_t)rows * row_stride;
    PIO_REQUIRE(row_stride % 8 == 0 && layer_stride % 8 == 0 && row_stride >= width && layer_stride >= 0,
                "%s: strides %lld, %lld (multiples of 8, rows of %lld)", nm, (long long)row_stride,
                (long long)layer_stride, (long long)width);
    // one layer behind the other, or one row's layers behind the other's
    PIO_REQUIRE(layers == 1 || (layer_stride >= width && ((layer_stride - width) / row_stride >= rows - 1 ||
                                                          (row_stride - width) / layer_stride >= layers - 1)),
                "%s: strides %lld, %lld: rows or layers overlap", nm, (long long)row_stride, (long long)layer_stride);
    PIO_REQUIRE(!kv_rows_meet((const char*)v - (const char*)k, dtype == PIO_F32 ? 4 : 2, width, rows, row_stride, layers,
                              layer_stride),
                "%s: k and v overlap", nm);
    const int per_block = (int)std::max<int64_t>(1, std::min<int64_t>({layers, (int64_t)rows * layers / 4096, (1 << 28) / width}));
    const dim3 grid(rows, ceil_div(layers, per_block));
    PIO_REQUIRE(grid.y <= 65535, "%s: too many layers", nm);
    hipStream_t st = pick_stream(stream);
#define KV_READ(KT, YT)                                                                                              \
    kv_read_kernel<KT, YT><<<grid, KV_COPY, 0, st>>>(*c, layer, layers, seq, row_start, first, n, (YT*)k, (YT*)v, \
                                                    row_stride, layer_stride, per_block)
    if (dtype == PIO_F32) {
        if (c->kv_dtype == PIO_F32) KV_READ(float, float);
        else if (c->kv_dtype == PIO_F16) KV_READ(_Float16, float);
        else KV_READ(KvMx4, float);
    } else {
        if (c->kv_dtype == PIO_F32) KV_READ(float, _Float16);
        else if (c->kv_dtype == PIO_F16) KV_READ(_Float16, _Float16);
        else KV_READ(KvMx4, _Float16);
    }
#undef KV_READ
    PIO_LAUNCHED();
    return PIO_OK;
}

PIO_EXPORT int pio_kv_fork(const pio_kv_cache* c, const int32_t* src, const int32_t* dst, int n, void* stream) {
    PIO_TRY(kv_requests(c, src, dst, n, "pio_kv_fork"));
    if (n == 0) return PIO_OK;
    kv_fork_kernel<<<n, KV_COPY, 0, pick_stream(stream)>>>(*c, src, dst, n);
    PIO_LAUNCHED();
    return PIO_OK;
}

PIO_EXPORT int pio_kv_drop(const pio_kv_cache* c, const int32_t* seq, const int32_t* count, int n, void* stream) {
    PIO_TRY(kv_requests(c, seq, seq, n, "pio_kv_drop"));
    PIO_REQUIRE(((uintptr_t)count & 3u) == 0, "pio_kv_drop: counts not 4-byte aligned");
    if (n == 0) return PIO_OK;
    kv_drop_kernel<<<n, KV_COPY, 0, pick_stream(stream)>>>(*c, seq, count, n);
    PIO_LAUNCHED();
    return PIO_OK;
}

PIO_EXPORT int pio_kv_compact(const pio_kv_cache* c, void* stream) {
    PIO_TRY(kv_check(c, "pio_kv_compact"));
    hipStream_t st = pick_stream(stream);
    if (c->n_pages <= KV_PLAN) kv_compact_few_kernel<<<1, KV_PLAN, 0, st>>>(*c);
    else kv_compact_plan_kernel<<<1, KV_PLAN, 0, st>>>(*c);
    PIO_LAUNCHED();
    return kv_copy(*c, c->n_pages / 2, true, st);
}
