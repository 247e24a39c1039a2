// A key-value cache in pages, for many requests: their rows appended with the
// rotation on the way, and attention of a block of rows per request over it.
//
// The arithmetic is that of the one-sequence path (attention.cu): tile-exact
// Q2.14 online softmax, reference golden_tiled_flash_attention_q2_14_impl
// host/host_qwen_8x64.cpp:3610-3739, rotation rotate_fix16_pair_with_quantized_rope
// host:4765-4788.  The reference has one sequence with one contiguous cache.
//
// Attention takes a request's 64-position tiles through three steps, of which only the last goes tile by tile.
//   scores  QK: scores (int16) and each tile's maximum;
//   values  the running maximum is the prefix maximum of the tiles' maxima, so a tile's probabilities
//           and its values tv (int16) need nothing else of the tiles before it;
//   join    replays the recurrence of (sum, acc), which rounds at every tile, in order, and
//           divides.  Between tiles that raise the maximum it only adds.
// So a request's length is split over as many warps as it has tiles.  There are two ways, between which
// choose() decides by what both were measured to take:
//   k_attend                     one launch, a cluster of up to 8 CTAs per (request, key head), everything
//                                in shared memory.  For few or short texts, which latency bounds: one request
//                                of 513 positions 7.7 us (three launches 11.1), 64 of up to 2304 29.8 (34).
//   k_scores, k_values, k_join   one launch each over all tiles, scores and tv through the L2.  For many long
//                                texts, which HBM and instructions bound, and for one that is longer
//                                than a cluster can hold: 64 requests of 8192 positions 131 us for 537 MB of
//                                keys and values (4.1 TB/s; a copy alone would take 82), one of 32768 28.4.
//
// Products are formed by int8 matrix instructions, exactly.  A product is
// rnd4(x sat16(16 y)) with y the cached value: with c = y limited to [-2048, 2048]
// it is x c, plus (8 - x) >> 4 where c = 2048 (16 y saturates to 32767 there).  x and c
// are split into bytes, x = 256 xh + xl, so that four byte products with whole-number
// sums in 32 bits give the sum, and where a tile holds some c = 2048 a fifth and sixth,
// of that 0/1 mask with the bytes of (8 - x) >> 4, the rest.  Scores: a bank or the total
// saturates only where |q| reaches 8192 (128 * 2^13 * 2^11 = 2^31); such query rows are
// scored one by one.  Values: 64 products of at most 2^25 never leave 32 bits.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <new>
#include <string>
#include <type_traits>

#include "llmx.h"
#include "cluster.cuh"
#include "device_util.cuh"
#include "fixed.cuh"
#include "host_model.h"
#include "kernels.cuh"

namespace {

using llmx::kTile;
using llmx::pdl_trigger;
using llmx::pdl_wait;
using llmx::rnd;
using llmx::sat16;
using llmx::sat32;

constexpr uint32_t kMaxRequests = 1024, kMaxHeads = 1024, kMaxLength = 1u << 20, kMaxColumns = 128, kMaxPageLen = 65536;
constexpr uint32_t kMaxAppendRows = 1u << 20;
constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kSmemOfSm = 227 * 1024;
constexpr int kMaxSmem = 160 * 1024;  // what any call of k_scores, k_values or k_join asks for
constexpr int kErrRequest = 1;    // offsets or length of a request out of range
constexpr int kErrPage = 2;       // a page number out of range
constexpr int kErrBudget = 4;     // more positions than the handle has room for

// A request as k_scores leaves it for the launches after it.
struct __align__(16) Meta {
    int slot;   // first tile slot: slots go by key head, column block, tile
    int item;   // first (key head, tile)
    int tiles;
    int rows;   // -1: void
};

struct Call {
    const int16_t *q;
    size_t ld_q;
    int16_t *out;
    size_t ld_out;
    const int16_t *k, *v;
    const int32_t *table;
    size_t ld_table;
    const uint32_t *offsets, *lengths;
    uint32_t rows, requests, longest, pages;
    int heads, kv, group, dim, page_len, max_block;
    uint32_t page8, page8_magic;  // page_len / 8, and for dividing by it
    uint32_t page_bytes, row_bytes;
    int scale8;                   // fm(1/sqrt(dim)), Q8.8
    long long capacity;           // (key head, tile) items
    // workspace
    Meta *meta;          // [requests + 1]: the last one's rows say whether some request is void
    uint32_t *score;     // [slot][64 positions][4 column pairs], biased
    uint4 *top;          // [slot][4 blocks of 16 positions]: the maxima of 4 column pairs, biased
    int16_t *tv;         // [slot][8][dim]
    int2 *fsum;          // [slot][8]: P(m_before - m), the sum of P
    const int16_t *exps; // [2049] of differences 0, -1, ... -2048
    int *error;
    int blocks;              // k_attend: column blocks of a cluster at most
    int tiles, cluster_log;  // k_attend: of a CTA at most; CTAs of a (request, key head): up to 8, a power of 2
};

// ---- small pieces -------------------------------------------------------------------
static __device__ __forceinline__ uint32_t div_page(const Call &c, uint32_t p8) {
    return c.page8 == 1 ? p8 : __umulhi(p8, c.page8_magic);
}
// The page of positions 8 p8 .. 8 p8 + 7 (page lengths are multiples of 8).  worst: the largest number met, which
// is reported at the kernel's end; one out of range is read as the last page.
static __device__ __forceinline__ uint32_t page_of(const Call &c, const int32_t *table, uint32_t p8, uint32_t &worst) {
    const uint32_t page = (uint32_t)table[div_page(c, p8)];
    worst = max(worst, page);
    return min(page, c.pages - 1);
}
// First of their rows of key head h.
static __device__ __forceinline__ const char *rows_of(const Call &c, const int16_t *cache, uint32_t page, uint32_t p8, int h) {
    const uint32_t inside = p8 - div_page(c, p8) * c.page8;
    return reinterpret_cast<const char *>(cache) + ((unsigned long long)page * c.page_bytes + ((uint32_t)h * c.page_len + inside * 8) * c.row_bytes);
}
static __device__ __forceinline__ void report(const Call &c, uint32_t worst) {
    if (worst >= c.pages) atomicOr(c.error, kErrPage);
}
// (not .nc: the launch before may still be writing the cache when this one starts)
static __device__ __forceinline__ uint4 ld16(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
static __device__ __forceinline__ uint32_t limit2(uint32_t v) { return __vmaxs2(__vmins2(v, 0x08000800u), 0xf800f800u); }
// Of four high bytes of limited values: 1 where the byte is 8 (the value 2048).
static __device__ __forceinline__ uint32_t at_limit(uint32_t h) { return (h >> 3) & ~(h >> 4) & 0x01010101u; }
// (8 - x) >> 4 of two 16-bit values, as 16 bits each
static __device__ __forceinline__ uint32_t rest2(uint32_t x) {
    const int a = (8 - llmx::lo16(x)) >> 4, b = (8 - llmx::hi16(x)) >> 4;
    return ((uint32_t)a & 0xffffu) | ((uint32_t)b << 16);
}
static __device__ __forceinline__ uint32_t low4(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x6420); }
static __device__ __forceinline__ uint32_t high4(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7531); }

// D = A B + C, A 16 x 32 and B 32 x 8 bytes; s and u: signed and unsigned.
#define LLMX_MMA(name, ta, tb)                                                                                                  \
    static __device__ __forceinline__ void name(int(&d)[4], const uint32_t(&a)[4], uint32_t b0, uint32_t b1, const int(&c)[4]) { \
        asm("mma.sync.aligned.m16n8k32.row.col.s32." ta "." tb ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"  \
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                                     \
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));          \
    }
LLMX_MMA(mma_su, "s8", "u8")
LLMX_MMA(mma_us, "u8", "s8")
LLMX_MMA(mma_uu, "u8", "u8")
#undef LLMX_MMA

// 8 x 8 values of 16 bits over a warp, transposed.
static __device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Two 32-bit values saturated to 16 bits each, the first in the low half.
static __device__ __forceinline__ uint32_t pack_sat16(int lo, int hi) {
    uint32_t r;
    asm("cvt.pack.sat.s16.s32 %0, %1, %2;" : "=r"(r) : "r"(hi), "r"(lo));
    return r;
}
// A score before its saturation to 16 bits: rnd8 of rnd8 of a total times fm(1/sqrt(d)) (the
// first never saturates: the factor is below 1), with both roundings' halves added at once.
static __device__ __forceinline__ int score_of(int total, int scale8) {
    return (int)(((long long)total * scale8 + (128 + (128 << 8))) >> 16);
}
// A score with its four saturating banks, by one lane: a decode step of 64 requests of up to 2304 positions takes 30 us, 106 where
// one of 16 query heads has an element of 32.0 or more, 277 where all have.
static __device__ __noinline__ int score_exact(const int16_t *q, const int16_t *k, int dim, int scale8) {
    long long bank[4] = {0, 0, 0, 0};
    for (int e = 0; e < dim; e++) bank[e & 3] += llmx::qk_prod(q[e], llmx::q412(k[e]));
    long long t = 0;
    for (int i = 0; i < 4; i++) t += sat32(bank[i]);
    return score_of(sat32(t), scale8);
}

// Rows and tiles of request b; false where it is void.
static __device__ __forceinline__ bool request(const Call &c, uint32_t b, int &rows, int &tiles) {
    const uint32_t o0 = c.offsets[b], o1 = c.offsets[b + 1], length = c.lengths[b];
    rows = (int)(o1 - o0);
    tiles = rows ? (int)((length + kTile - 1) / kTile) : 0;
    return o0 <= o1 && o1 <= c.rows && o1 - o0 <= (uint32_t)c.max_block && length <= c.longest;
}

// The requests' first slots and items, into shared memory (and by CTA 0 into the
// workspace); returns the number of items, 0 when the call needs more than the handle has.
static __device__ int plan(const Call &c, Meta *meta) {
    __shared__ long long part[2][kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long slots = 0, items = 0;  // of the requests before this round's
    bool some_void = false;
    for (uint32_t first = 0; first < c.requests; first += kThreads) {
        const uint32_t b = first + threadIdx.x;
        Meta m{0, 0, 0, -1};
        long long s = 0, i = 0;
        if (b < c.requests) {
            int rows, tiles;
            if (request(c, b, rows, tiles)) {
                m.rows = rows;
                m.tiles = tiles;
                i = (long long)c.kv * m.tiles;
                s = i * ((m.rows * c.group + 7) / 8);
            } else {
                some_void = true;
                if (blockIdx.x == 0) atomicOr(c.error, kErrRequest);
            }
        }
        long long ss = s, ii = i;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long a = __shfl_up_sync(0xffffffffu, ss, o), d = __shfl_up_sync(0xffffffffu, ii, o);
            if (lane >= o) {
                ss += a;
                ii += d;
            }
        }
        __syncthreads();  // the last round's parts are read
        if (lane == 31) {
            part[0][warp] = ss;
            part[1][warp] = ii;
        }
        __syncthreads();
        long long s0 = slots, i0 = items;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) {
                s0 += part[0][w];
                i0 += part[1][w];
            }
            slots += part[0][w];
            items += part[1][w];
        }
        if (b < c.requests) {
            m.slot = (int)(s0 + ss - s);
            m.item = (int)(i0 + ii - i);
            meta[b] = m;
        }
    }
    const bool fits = items <= c.capacity;  // (an item has a slot per column block: they fit as well)
    some_void = __syncthreads_or(some_void);
    if (!fits)
        for (uint32_t b = threadIdx.x; b < c.requests; b += kThreads) meta[b] = Meta{0, 0, 0, -1};
    if (blockIdx.x == 0) {
        if (!fits && threadIdx.x == 0) atomicOr(c.error, kErrBudget);
        if (threadIdx.x == 0) c.meta[c.requests] = Meta{0, 0, 0, some_void};
        for (uint32_t b = threadIdx.x; b < c.requests; b += kThreads) c.meta[b] = meta[b];
    }
    __syncthreads();
    return fits ? (int)items : 0;
}

// A (request, key head) at hand.
struct Strip {
    const int32_t *table;
    int h, rows, length, blocks;
    uint32_t row0;
    int col0;  // first of the columns at hand (k_attend may have a part of them), `blocks` blocks of 8
};
// One (request, key head, tile) after another.
struct Cursor {
    int b, h, t;  // request, key head, tile
    int tiles, rows, length, blocks;
    uint32_t row0;
    int slot0;    // of tile 0 in the first column block of this key head
    const int32_t *table;

    __device__ void enter(const Call &c, const Meta *meta, int request, int head) {
        b = request;
        h = head;
        const Meta m = meta[b];
        tiles = m.tiles;
        rows = m.rows;
        length = (int)c.lengths[b];
        row0 = c.offsets[b];
        blocks = (rows * c.group + 7) >> 3;
        slot0 = m.slot + h * blocks * tiles;
        table = c.table + (size_t)b * c.ld_table;
    }
    // item: below the number of items
    __device__ void start(const Call &c, const Meta *meta, int item) {
        int lo = 0, hi = (int)c.requests - 1;  // the last request with item >= its first: it has items
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (meta[mid].item <= item) lo = mid;
            else hi = mid - 1;
        }
        const Meta m = meta[lo];
        const int head = (item - m.item) / m.tiles;
        enter(c, meta, lo, head);
        t = item - m.item - head * m.tiles;
    }
    // The next item, which there is.  Returns whether it is of another request or key head.
    __device__ bool next(const Call &c, const Meta *meta) {
        if (++t < tiles) return false;
        t = 0;
        int r = b, head = h + 1;
        if (head == c.kv) {
            head = 0;
            do r++;
            while (meta[r].tiles == 0);
        }
        enter(c, meta, r, head);
        return true;
    }
    // Slot of this tile in column block nb.
    __device__ int slot(int nb) const { return slot0 + nb * tiles + t; }
    __device__ Strip strip() const { return Strip{table, h, rows, length, blocks, row0, 0}; }
};

static __device__ __forceinline__ void range_of(int items, int &first, int &end) {
    const int each = (int)(((long long)items + gridDim.x - 1) / gridDim.x);
    first = (int)min((long long)blockIdx.x * each, (long long)items);
    end = min(first + each, items);
}

// ---- scores -------------------------------------------------------------------------
// Scores are kept biased (with the sign bit turned), so that unsigned minima, maxima and
// differences of packed pairs do.
constexpr uint32_t kBias2 = 0x80008000u;

// What a CTA keeps of a column (a query row) of the (request, key head) at hand.
struct Column {
    int bias[kMaxColumns];  // 2048 times its sum
    int seen[kMaxColumns];  // positions that it sees
    int wide[kMaxColumns];  // a bank may saturate
};
// Queries as the lanes' shares of B, [block][KS][32 lanes] {low, low, high, high}, and the same of
// (8 - q) >> 4; by `warps` warps.
template <int KS>
static __device__ __forceinline__ void stage_queries(const Call &c, const Strip &z, int warp, int warps, uint4 *queries, uint4 *rests, Column &column) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int columns = z.rows * c.group - z.col0;
    for (int nb = warp; nb < z.blocks; nb += warps) {
        const int col = nb * 8 + g, j = (z.col0 + col) / c.group;
        const int16_t *q = c.q + (size_t)(z.row0 + j) * c.ld_q + (size_t)(z.h * c.group + z.col0 + col - j * c.group) * c.dim + 8 * t4;
        uint32_t big = 0;
        int sum = 0;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const uint4 w = col < columns && 32 * s + 8 * t4 < c.dim ? *reinterpret_cast<const uint4 *>(q + 32 * s) : make_uint4(0, 0, 0, 0);
            // above 8192: the top three of 16 bits differ
            big |= (w.x ^ (w.x << 1)) | (w.x ^ (w.x << 2)) | (w.y ^ (w.y << 1)) | (w.y ^ (w.y << 2)) | (w.z ^ (w.z << 1)) | (w.z ^ (w.z << 2)) |
                   (w.w ^ (w.w << 1)) | (w.w ^ (w.w << 2));
            // (a total reaches 2^31 only where every q is -8192, the first one too)
            if (s == 0 && t4 == 0 && (w.x & 0xffffu) == 0xe000u) big |= 0x8000u;
            sum += llmx::lo16(w.x) + llmx::hi16(w.x) + llmx::lo16(w.y) + llmx::hi16(w.y) + llmx::lo16(w.z) + llmx::hi16(w.z) + llmx::lo16(w.w) +
                   llmx::hi16(w.w);
            queries[(nb * KS + s) * 32 + lane] = make_uint4(low4(w.x, w.y), low4(w.z, w.w), high4(w.x, w.y), high4(w.z, w.w));
            const uint4 r = make_uint4(rest2(w.x), rest2(w.y), rest2(w.z), rest2(w.w));
            rests[(nb * KS + s) * 32 + lane] = make_uint4(low4(r.x, r.y), low4(r.z, r.w), high4(r.x, r.y), high4(r.z, r.w));
        }
        big |= __shfl_xor_sync(0xffffffffu, big, 1);
        big |= __shfl_xor_sync(0xffffffffu, big, 2);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (t4 == 0) {
            column.bias[col] = 2048 * sum;
            column.seen[col] = col < columns ? z.length - z.rows + 1 + j : 0;
            column.wide[col] = (int)(big & 0x80008000u);
        }
    }
}

// The pages of 16 positions' keys, and this lane's share of them: rows g and g + 8, dimensions 32 s + 8 t4
// .. + 7.  What is not there is read from a place that is: scores of positions behind the last are
// not looked at, and the queries' dimensions behind the last are 0.
struct KeyPages {
    uint32_t page[2];
    __device__ __forceinline__ void load(const Call &c, const Strip &z, int p0, uint32_t &worst) {
#pragma unroll
        for (int r = 0; r < 2; r++) page[r] = p0 + 8 * r < z.length ? page_of(c, z.table, (uint32_t)(p0 >> 3) + r, worst) : 0;
    }
};
template <int KS>
struct KeyRows {
    const char *row[2];
    int last;  // bytes to the last step's dimensions
    __device__ __forceinline__ void start(const Call &c, const Strip &z, const KeyPages &pages, int p0) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
        for (int r = 0; r < 2; r++) row[r] = rows_of(c, c.k, pages.page[r], (uint32_t)(p0 >> 3) + r, z.h) + (g * c.row_bytes + 16 * t4);
        last = 32 * (KS - 1) + 8 * t4 < c.dim ? 64 * (KS - 1) : -16 * t4;
    }
    __device__ __forceinline__ void load(int s, uint4 (&raw)[2][KS]) const {
#pragma unroll
        for (int r = 0; r < 2; r++) raw[r][s] = ld16(row[r] + (s == KS - 1 ? last : 64 * s));
    }
};
template <int KS>
static __device__ __forceinline__ void load_keys(const Call &c, const Strip &z, const KeyPages &pages, int p0, uint4 (&raw)[2][KS]) {
    KeyRows<KS> rows;
    rows.start(c, z, pages, p0);
#pragma unroll
    for (int s = 0; s < KS; s++) rows.load(s, raw);
}

// What scores 16 positions (the rows of A) against 8 columns (query rows): the sums of the byte products.
struct Sums {
    int hh[4], mid[4], ll[4];
    __device__ __forceinline__ void start(const Column &column, int nb) {
        const int2 bias = *reinterpret_cast<const int2 *>(&column.bias[nb * 8 + 2 * (threadIdx.x & 3)]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            hh[i] = mid[i] = 0;
            ll[i] = i & 1 ? -bias.y : -bias.x;
        }
    }
    __device__ __forceinline__ void add(const uint32_t (&kl)[4], const uint32_t (&kh)[4], uint4 q) {
        mma_us(hh, kh, q.z, q.w, hh);
        mma_uu(mid, kh, q.x, q.y, mid);
        mma_uu(ll, kl, q.x, q.y, ll);
        mma_us(mid, kl, q.z, q.w, mid);
    }
    __device__ __forceinline__ void add_rest(const uint32_t (&kh)[4], uint4 r) {
        uint32_t m[4];
#pragma unroll
        for (int i = 0; i < 4; i++) m[i] = kh[i] >> 4 & 0x01010101u;
        mma_us(mid, m, r.z, r.w, mid);
        mma_uu(ll, m, r.x, r.y, ll);
    }
};
// The scores from them: w[0] position p0 + g, w[1] p0 + 8 + g, columns 2 t4 and 2 t4 + 1 of block nb, biased.
// Returns their columns' maxima over the positions that they see, in lanes 0 to 3 (of column pair t4).
static __device__ __forceinline__ uint32_t finish_scores(const Call &c, const Strip &z, const Sums &u, int nb, int p0, const Column &column, uint32_t (&w)[2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    int sc[4];
#pragma unroll
    for (int i = 0; i < 4; i++) sc[i] = score_of((int)(((uint32_t)u.hh[i] << 16) + ((uint32_t)u.mid[i] << 8) + (uint32_t)u.ll[i]), c.scale8);
    const int2 wide = *reinterpret_cast<const int2 *>(&column.wide[nb * 8 + 2 * t4]);
    if (__any_sync(0xffffffffu, (wide.x | wide.y) != 0)) {
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            const int col = nb * 8 + 2 * t4 + (i & 1), p = p0 + g + (i >> 1) * 8;
            if (!column.wide[col] || p >= z.length) continue;
            uint32_t none = 0;
            const int j = (z.col0 + col) / c.group;
            const int16_t *q = c.q + (size_t)(z.row0 + j) * c.ld_q + (size_t)(z.h * c.group + z.col0 + col - j * c.group) * c.dim;
            const int16_t *k = reinterpret_cast<const int16_t *>(rows_of(c, c.k, page_of(c, z.table, (uint32_t)p >> 3, none), (uint32_t)p >> 3, z.h) + (p & 7) * c.row_bytes);
            const int y = score_exact(q, k, c.dim, c.scale8);
            if (i == 0) sc[0] = y;
            else if (i == 1) sc[1] = y;
            else if (i == 2) sc[2] = y;
            else sc[3] = y;
        }
    }
    w[0] = pack_sat16(sc[0], sc[1]) ^ kBias2;
    w[1] = pack_sat16(sc[2], sc[3]) ^ kBias2;
    uint32_t top = __vmaxu2(w[0], w[1]);
    if (p0 + 16 > z.length - z.rows + 1) {  // some column does not see all 16 positions
        const int2 n = *reinterpret_cast<const int2 *>(&column.seen[nb * 8 + 2 * t4]);
        auto seen = [&](int p) { return (p < n.x ? 0xffffu : 0u) | (p < n.y ? 0xffff0000u : 0u); };
        top = __vmaxu2(w[0] & seen(p0 + g), w[1] & seen(p0 + 8 + g));
    }
#pragma unroll
    for (int o = 4; o < 32; o *= 2) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
    return top;
}

// The byte planes of one step of 32 dimensions, limited and from 0 to 4096: min(k, 2048), then max(k + 2048, 0).
// Returns the high ones together.
static __device__ __forceinline__ uint32_t step_planes(const uint4 a, const uint4 b, uint32_t (&kl)[4], uint32_t (&kh)[4]) {
    auto shift = [](uint32_t w) { return __viaddmax_s16x2(__vmins2(w, 0x08000800u), 0x08000800u, 0u); };
    const uint4 x = make_uint4(shift(a.x), shift(a.y), shift(a.z), shift(a.w)), y = make_uint4(shift(b.x), shift(b.y), shift(b.z), shift(b.w));
    kl[0] = low4(x.x, x.y);
    kl[1] = low4(y.x, y.y);
    kl[2] = low4(x.z, x.w);
    kl[3] = low4(y.z, y.w);
    kh[0] = high4(x.x, x.y);
    kh[1] = high4(y.x, y.y);
    kh[2] = high4(x.z, x.w);
    kh[3] = high4(y.z, y.w);
    return kh[0] | kh[1] | kh[2] | kh[3];
}
// Scores a warp's 16 positions against all column blocks and loads the next ones' keys, at pn, meanwhile;
// store(nb, maxima, scores).
template <int KS, bool kOne, class Store>
static __device__ __forceinline__ void score_tile(const Call &c, const Strip &z, int p0, uint4 (&raw)[2][KS], const Strip &zn, const KeyPages &pages, int pn,
                                                  const uint4 *queries, const uint4 *rests, const Column &column, Store store) {
    const int lane = threadIdx.x & 31;
    KeyRows<KS> next;
    next.start(c, zn, pages, pn);
    uint32_t kl[KS][4], kh[KS][4], limit = 0;
#pragma unroll
    for (int s = 0; s < KS; s++) {
        limit |= step_planes(raw[0][s], raw[1][s], kl[s], kh[s]);
        next.load(s, raw);
    }
    // some value is at the upper limit (its high byte is 16)
    const bool some = __any_sync(0xffffffffu, (limit & 0x10101010u) != 0);
#pragma unroll 1
    for (int nb = 0; nb < (kOne ? 1 : z.blocks); nb++) {
        Sums u;
        u.start(column, nb);
#pragma unroll
        for (int s = 0; s < KS; s++) u.add(kl[s], kh[s], queries[(nb * KS + s) * 32 + lane]);
        if (some)
#pragma unroll
            for (int s = 0; s < KS; s++) u.add_rest(kh[s], rests[(nb * KS + s) * 32 + lane]);
        uint32_t w[2];
        const uint32_t top = finish_scores(c, z, u, nb, p0, column, w);
        store(nb, top, w);
        __syncwarp();  // (lanes 0 to 3 stored more)
    }
}

// One CTA's run of tiles, a warp per 16 positions: the 16 rows of A, loaded straight from HBM as its lanes
// hold them, two tiles ahead in registers; the queries are B.  Four CTAs an SM by registers.  64 x 8192:
// 54 us, 278 MB at 5.1 TB/s (78 % of a copy), 50 % of the issue slots and 53 % of the ALU (splitting keys into
// bytes); five CTAs with the planes formed step by step 55.6.
template <int KS, bool kOne>  // steps of 32 dimensions; one column block
__global__ void __launch_bounds__(kThreads, 4) k_scores(const Call c) {
    extern __shared__ __align__(1024) unsigned char dynamic[];
    __shared__ __align__(16) Column column;
    const int most = kOne ? 1 : (c.max_block * c.group + 7) / 8;  // column blocks
    uint4 *queries = reinterpret_cast<uint4 *>(dynamic);          // [most][KS][32]
    uint4 *rests = queries + most * KS * 32;
    Meta *meta = reinterpret_cast<Meta *>(rests + most * KS * 32);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_trigger();
    const int items = plan(c, meta);
    int first, end;
    range_of(items, first, end);
    if (first >= end) return;
    uint32_t worst = 0;
    Cursor cur;
    cur.start(c, meta, first);
    Strip z = cur.strip();
    uint4 raw[2][KS];
    KeyPages pages;
    pages.load(c, z, cur.t * kTile + warp * 16, worst);
    load_keys<KS>(c, z, pages, cur.t * kTile + warp * 16, raw);
    pages.load(c, z, (cur.t + 1) * kTile + warp * 16, worst);
    for (int item = first; item < end;) {  // a (request, key head)
        __syncthreads();                   // the last one's columns are done with
        stage_queries<KS>(c, z, warp, kWarps, queries, rests, column);
        __syncthreads();
        const int n = min(cur.tiles - cur.t, end - item);
        size_t at = (size_t)cur.slot(0) * 4 + warp;  // the block of 16 positions in the first column block
        const size_t step = (size_t)cur.tiles * 4;
        int p0 = cur.t * kTile + warp * 16;
        const Strip here = z;
        for (int k = 0; k < n; k++, p0 += kTile, at += 4) {
            // the next tile's keys are on their way while this one's are used, the next one's page numbers too
            const bool inside = k + 1 < n, more = inside || item + n < end;
            if (!inside && more) {
                cur.t += n - 1;
                cur.next(c, meta);
                z = cur.strip();
                pages.load(c, z, warp * 16, worst);
            }
            const int pn = inside ? p0 + kTile : warp * 16;
            score_tile<KS, kOne>(c, here, p0, raw, z, pages, pn, queries, rests, column, [&](int nb, uint32_t top, const uint32_t(&w)[2]) {
                const size_t block = at + nb * step;
                c.score[block * 64 + lane] = w[0];
                c.score[block * 64 + 32 + lane] = w[1];
                if (lane < 4) reinterpret_cast<uint32_t *>(c.top)[block * 4 + lane] = top;
            });
            pages.load(c, z, pn + kTile, worst);
        }
        item += n;
    }
    report(c, worst);
}

// ---- values -------------------------------------------------------------------------
constexpr int kExpWords = 1028;                 // 2049 entries of 16 bits, rounded up to 16 bytes
constexpr int kDepth = 2;                       // tiles of a warp's ring
constexpr int kSlice = kTile * 64;              // bytes of a tile's share: 64 positions, 32 elements
constexpr int kRing = kWarps * kDepth * kSlice;

static __device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// A tile's values of 32 elements into a warp's ring: a position's 64 bytes in a row, its 16-byte units
// turned by row / 2 mod 4, so that the 8 rows that a matrix load takes, and those that a copy writes, lie in
// different banks.  A lane copies one unit of 8 positions, from one page, in an order of its own.  What
// is not there comes from a place that is: its probabilities are 0, its elements not stored.
static __device__ __forceinline__ void fetch_values(const Call &c, const Strip &z, int t, int part, unsigned char *ring, uint32_t &worst) {
    const int lane = threadIdx.x & 31, unit = lane & 3, j = lane >> 2;
    const uint32_t p8 = min((uint32_t)(t * 8 + j), (uint32_t)(z.length - 1) >> 3);
    const char *rows = rows_of(c, c.v, page_of(c, z.table, p8, worst), p8, z.h) + (part * 32 + unit * 8 < c.dim ? part * 64 + unit * 16 : 0);
    // row i ^ j goes to j * 512 + (i ^ j) * 64 + (unit ^ (i ^ j) / 2 mod 4) * 16 (a slice starts at a multiple of 512)
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring) + j * 512 + j * 64 + ((unit ^ (j >> 1)) & 3) * 16;
#pragma unroll
    for (int i = 0; i < 8; i++) copy16(dst ^ (uint32_t)(i * 64 + (i >> 1 & 3) * 16), rows + (uint32_t)(i ^ j) * c.row_bytes);
}
static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// The four registers of an octet of elements: the words of positions 8 j + 2 t4, + 1, element g.
static __device__ __forceinline__ void load_octet(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// Byte planes of a tile's 32 elements as A: [step of 32 positions][16 elements].  A lane's bytes of positions
// are those of 8 j + 2 t4 and the next, j = 0, 1 (first words) and j = 2, 3.
struct Planes {
    uint32_t l[2][2][4], h[2][2][4];
    // Returns whether some value is not within [-2048, 2047] (the high byte's bits 3 to 7 differ).
    template <bool kLimit>
    __device__ __forceinline__ bool load(const unsigned char *ring) {
        const int lane = threadIdx.x & 31;
        // octet o of a row is its unit o ^ row / 2 mod 4
        const uint32_t row = (uint32_t)__cvta_generic_to_shared(ring) + lane * 64 + (lane >> 1 & 3) * 16;
        uint32_t out = 0;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int o = 0; o < 4; o++) {
                uint32_t r[4];
                load_octet((row ^ (uint32_t)(o * 16)) + s * 2048, r);
                if (kLimit)
#pragma unroll
                    for (int i = 0; i < 4; i++) r[i] = limit2(r[i]);
                l[s][o >> 1][o & 1] = low4(r[0], r[1]);
                l[s][o >> 1][2 + (o & 1)] = low4(r[2], r[3]);
                h[s][o >> 1][o & 1] = high4(r[0], r[1]);
                h[s][o >> 1][2 + (o & 1)] = high4(r[2], r[3]);
                if (!kLimit)
#pragma unroll
                    for (int i = 0; i < 2; i++) out |= h[s][o >> 1][2 * i + (o & 1)] ^ (h[s][o >> 1][2 * i + (o & 1)] << 1);
            }
        return !kLimit && __any_sync(0xffffffffu, (out & 0xf0f0f0f0u) != 0);
    }
};

// Place of lane u's 16 bytes of B among 32: turned, so that the bytes of a column pair's two positions, which 16 lanes
// store, lie in as many banks as they can.
static __device__ __forceinline__ int place_of(int u) { return u ^ (u >> 3 << 1); }

// Probabilities of 16 positions (block blk of a tile) against 8 columns, as bytes in the order of B.
// Lane: column pair lane & 3, positions 8 r + 2 t and the next; s: their scores, biased; m: the pair's
// maxima; prob: [2 steps][32 lanes] {low, low, high, high}.
static __device__ __forceinline__ void probabilities(const int16_t *exps, uint32_t s0, uint32_t s1, uint32_t m, int p, int seen0, int seen1, int blk,
                                                     uint4 *prob) {
    const int lane = threadIdx.x & 31, cp = lane & 3, t = lane >> 2 & 3, r = lane >> 4;
    const uint32_t floor = __vmaxu2(m, 0x08000800u) - 0x08000800u;
    // differences to the maximum, 0 to 2048 (what is not seen may hold anything)
    const uint32_t d0 = m - __vminu2(__vmaxu2(s0, floor), m), d1 = m - __vminu2(__vmaxu2(s1, floor), m);
    uint32_t a0 = (uint16_t)exps[d0 & 0xffffu], b0 = (uint16_t)exps[d0 >> 16], a1 = (uint16_t)exps[d1 & 0xffffu], b1 = (uint16_t)exps[d1 >> 16];
    a0 = p < seen0 ? a0 : 0;
    b0 = p < seen1 ? b0 : 0;
    a1 = p + 1 < seen0 ? a1 : 0;
    b1 = p + 1 < seen1 ? b1 : 0;
    const uint32_t a = __byte_perm(a0, a1, 0x5140), b = __byte_perm(b0, b1, 0x5140);  // {low, low, high, high}
    // (place_of(cp * 8 + t), and of the next column's, 4 further)
    const int at = cp * 8 + (t ^ 2 * cp);
    uint16_t *dst = reinterpret_cast<uint16_t *>(prob + (blk >> 1) * 32) + 2 * (blk & 1) + r;
    dst[8 * at] = (uint16_t)a;
    dst[8 * at + 4] = (uint16_t)(a >> 16);
    dst[8 * (at ^ 4)] = (uint16_t)b;
    dst[8 * (at ^ 4) + 4] = (uint16_t)(b >> 16);
}

// A tile's values against 8 columns: y[o] is the word of column g, elements 8 o + 2 t4 and the next, of
// the part's 32.  kLimit: values were limited, and some may be at the upper limit.
template <bool kLimit>
static __device__ __forceinline__ void weigh(const Planes &v, const uint4 (&b)[2], uint32_t (&y)[4]) {
    uint4 rest[2];  // of the probabilities
    if (kLimit)
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint32_t r0 = rest2(__byte_perm(b[s].x, b[s].z, 0x5140)), r1 = rest2(__byte_perm(b[s].x, b[s].z, 0x7362));
            const uint32_t r2 = rest2(__byte_perm(b[s].y, b[s].w, 0x5140)), r3 = rest2(__byte_perm(b[s].y, b[s].w, 0x7362));
            rest[s] = make_uint4(low4(r0, r1), low4(r2, r3), high4(r0, r1), high4(r2, r3));
        }
#pragma unroll
    for (int mb = 0; mb < 2; mb++) {
        // The high products' sums become a part of the middle ones' and these of the low ones'; and rnd8 of rnd6 of
        // the sum is (sum + 2^5 + 2^13) >> 14; the sum is below 2^31 - 2^16.
        int d[4] = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 2; s++) mma_su(d, v.h[s][mb], b[s].z, b[s].w, d);
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] *= 256;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            mma_su(d, v.h[s][mb], b[s].x, b[s].y, d);
            mma_uu(d, v.l[s][mb], b[s].z, b[s].w, d);
        }
        uint32_t m[2][4];
        if (kLimit)
#pragma unroll
            for (int s = 0; s < 2; s++) {
#pragma unroll
                for (int i = 0; i < 4; i++) m[s][i] = at_limit(v.h[s][mb][i]);
                mma_us(d, m[s], rest[s].z, rest[s].w, d);
            }
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = (int)((uint32_t)d[i] * 256u + 8224u);
#pragma unroll
        for (int s = 0; s < 2; s++) mma_uu(d, v.l[s][mb], b[s].x, b[s].y, d);
        if (kLimit)
#pragma unroll
            for (int s = 0; s < 2; s++) mma_uu(d, m[s], rest[s].x, rest[s].y, d);
        y[2 * mb] = transpose8(pack_sat16(d[0] >> 14, d[1] >> 14));
        y[2 * mb + 1] = transpose8(pack_sat16(d[2] >> 14, d[3] >> 14));
    }
}
// The columns' sums of P: lanes 0 to 3 get those of 2 t4 and 2 t4 + 1.
static __device__ __forceinline__ int2 sum_of(const uint4 (&b)[2]) {
    const uint32_t one[4] = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
    int d[4] = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 2; s++) mma_uu(d, one, b[s].z, b[s].w, d);
    d[0] *= 256;
    d[1] *= 256;
#pragma unroll
    for (int s = 0; s < 2; s++) mma_uu(d, one, b[s].x, b[s].y, d);
    return make_int2(d[0], d[1]);
}

constexpr int kChunk = 4;  // tiles of a (request, key head) whose probabilities k_values forms at once

// The warps' shares of a tile's elements: `part` of 32, and with fewer parts than warps every `step`-th tile.
struct Share {
    int part, first, step, shift, octets;  // (octets of elements)
    __device__ __forceinline__ Share(int dim, int warp) {
        const int log = dim > 64 ? 2 : dim > 32 ? 1 : 0;  // 4, 2 or 1 (of three parts the fourth warp has none)
        part = warp & ((1 << log) - 1);
        first = part * 32 < dim ? warp >> log : INT_MAX;
        step = kWarps >> log;
        shift = 2 - log;
        octets = min((dim - part * 32) >> 3, 4);
    }
    __device__ __forceinline__ int count(int n) const { return n > first ? (n - first + step - 1) >> shift : 0; }
};

// One CTA's run of tiles, in chunks of up to kChunk: their probabilities, by all warps, through shared
// memory (two buffers in turn, so one barrier a chunk does); then every warp weighs its 32 elements
// of every tile, for itself, from a ring of two tiles that cp.async fills.  64 x 8192: 65 us at 4.4 TB/s, 41 %
// of the issue slots: latency (loads, barriers, shared memory) with the 16 warps an SM that registers leave;
// five CTAs with one buffer of probabilities 27 us more, starting before k_scores' end no less.
template <bool kOne>
__global__ void __launch_bounds__(kThreads, 4) k_values(const Call c) {
    extern __shared__ __align__(1024) unsigned char dynamic[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3, cp = t4;
    const int most = kOne ? 1 : (c.max_block * c.group + 7) / 8;  // column blocks
    const int chunk = kOne ? kChunk : max(1, kChunk / most);
    unsigned char *ring = dynamic + warp * kDepth * kSlice;
    uint4 *prob = reinterpret_cast<uint4 *>(dynamic + kRing);  // [2][chunk][most][64]
    uint32_t *exps_w = reinterpret_cast<uint32_t *>(prob + 2 * chunk * most * 64);
    const int16_t *exps = reinterpret_cast<const int16_t *>(exps_w);
    uint32_t *before = exps_w + kExpWords + warp * most * 4;  // the warp's own: maxima of column pairs up to the chunk
    uint32_t *tops_of = exps_w + kExpWords + kWarps * most * 4;                  // [2][kWarps][most * 4]
    int *seen = reinterpret_cast<int *>(tops_of + 2 * kWarps * most * 4);         // [2][most * 8]
    Meta *meta = reinterpret_cast<Meta *>(seen + 2 * most * 8);
    for (int i = threadIdx.x; i < kExpWords; i += kThreads) exps_w[i] = reinterpret_cast<const uint32_t *>(c.exps)[i];
    pdl_wait();
    pdl_trigger();
    for (uint32_t b = threadIdx.x; b < c.requests; b += kThreads) meta[b] = c.meta[b];
    __syncthreads();
    const Meta last = meta[c.requests - 1];
    // void requests have no items but their place in the order
    const int items = last.item + c.kv * last.tiles;
    int first, end;
    range_of(items, first, end);
    if (first >= end) return;
    uint32_t worst = 0;
    const Share share(c.dim, warp);
    const int pos = warp * 16 + 8 * (lane >> 4) + 2 * (lane >> 2 & 3);  // of a tile: this lane's first of two
    Cursor cur;
    cur.start(c, meta, first);
    bool moved = true;
    int turn = 0, buffer = 0;
    int from = 0, into = 0, flying = 0, ahead = 0;  // the ring: next slot to use and to fill, tiles in it, of the next chunk
    // of a chunk's tiles: scores of this lane's two positions and column pair; maxima of 16 positions, 16 words of
    // two tiles a load
    uint32_t score[kChunk][2], top[kChunk / 2];
    auto load_scores = [&](int slot, int n) {
        const uint32_t *s = c.score + (size_t)slot * 256 + pos * 4 + cp;
        const uint32_t *t = reinterpret_cast<const uint32_t *>(c.top) + (size_t)slot * 16 + lane;
#pragma unroll
        for (int k = 0; k < kChunk; k++) {
            const int at = min(k, n - 1) * 256;
            score[k][0] = s[at];
            score[k][1] = s[at + 4];
        }
#pragma unroll
        for (int k = 0; k < kChunk / 2; k++) top[k] = 32 * k + lane < 16 * n ? t[32 * k] : 0;
    };
    auto length_of = [&](int item) { return min(min(chunk, cur.tiles - cur.t), end - item); };
    if constexpr (kOne) load_scores(cur.slot(0), length_of(first));
    for (int item = first; item < end;) {
        const Strip z = cur.strip();
        const int n = length_of(item), t0 = cur.t, slot0 = cur.slot(0), tiles = cur.tiles;
        // tiles of this chunk that are this warp's; those that the last chunk's loop has fetched already
        const int mine = share.count(n);
        int fetched = ahead;
        auto fetch = [&](const Strip &of, int t) {
            fetch_values(c, of, t, share.part, ring + into * kSlice, worst);
            commit();
            into ^= 1;
            flying++;
        };
        for (; flying < kDepth && fetched < mine; fetched++) fetch(z, t0 + share.first + fetched * share.step);
        if (moved) {  // the maxima of the tiles before
            turn ^= 1;
            for (int nb = 0; nb < z.blocks; nb++) {
                const uint4 *tops = c.top + (size_t)(slot0 + nb * tiles - t0) * 4;
                uint4 m = make_uint4(0, 0, 0, 0);
#pragma unroll 4
                for (int i = threadIdx.x; i < t0 * 4; i += kThreads) {
                    const uint4 w = tops[i];
                    m = make_uint4(__vmaxu2(m.x, w.x), __vmaxu2(m.y, w.y), __vmaxu2(m.z, w.z), __vmaxu2(m.w, w.w));
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    m.x = __vmaxu2(m.x, __shfl_xor_sync(0xffffffffu, m.x, o));
                    m.y = __vmaxu2(m.y, __shfl_xor_sync(0xffffffffu, m.y, o));
                    m.z = __vmaxu2(m.z, __shfl_xor_sync(0xffffffffu, m.z, o));
                    m.w = __vmaxu2(m.w, __shfl_xor_sync(0xffffffffu, m.w, o));
                }
                if (lane == 0) *reinterpret_cast<uint4 *>(tops_of + (turn * kWarps + warp) * most * 4 + nb * 4) = m;
            }
            // (two buffers: warps may still be at the last one's)
            for (int col = threadIdx.x; col < z.blocks * 8; col += kThreads)
                seen[turn * most * 8 + col] = col < z.rows * c.group ? z.length - z.rows + 1 + col / c.group : 0;
            __syncthreads();
            for (int i = lane; i < z.blocks * 4; i += 32) {
                uint32_t m = 0;
#pragma unroll
                for (int w = 0; w < kWarps; w++) m = __vmaxu2(m, tops_of[(turn * kWarps + w) * most * 4 + i]);
                before[i] = m;
            }
            __syncwarp();
        }
        uint4 *pb = prob + (buffer ? chunk * most * 64 : 0);
        buffer ^= 1;
        for (int nb = 0; nb < (kOne ? 1 : z.blocks); nb++) {
            const int slot = slot0 + nb * tiles;
            if constexpr (!kOne) load_scores(slot, n);
            // maxima of this lane's column pair up to each tile
            uint32_t m[kChunk];
#pragma unroll
            for (int k = 0; k < kChunk / 2; k++) {
                uint32_t w = top[k];
                w = __vmaxu2(w, __shfl_xor_sync(0xffffffffu, w, 4));
                w = __vmaxu2(w, __shfl_xor_sync(0xffffffffu, w, 8));
                m[2 * k] = __shfl_sync(0xffffffffu, w, cp);
                m[2 * k + 1] = __shfl_sync(0xffffffffu, w, 16 + cp);
            }
            uint32_t was = before[nb * 4 + cp];
            const int seen0 = seen[turn * most * 8 + nb * 8 + 2 * cp], seen1 = seen[turn * most * 8 + nb * 8 + 2 * cp + 1];
#pragma unroll
            for (int k = 0; k < kChunk; k++)
                if (kOne || k < n) {  // (the last tile again behind it)
                    const int p = (t0 + min(k, n - 1)) * kTile;
                    m[k] = __vmaxu2(m[k], was);
                    probabilities(exps, score[k][0], score[k][1], m[k], p + pos, seen0, seen1, warp, pb + (k * most + nb) * 64);
                    if (warp == 0 && lane < 4 && k < n) {
                        const uint32_t d = m[k] - __vmaxu2(was, __vmaxu2(m[k], 0x08000800u) - 0x08000800u);
                        int2 *f = c.fsum + (size_t)(slot + k) * 8 + 2 * lane;
                        f[0].x = exps[d & 0xffffu];
                        f[1].x = exps[d >> 16];
                    }
                    was = m[k];
                }
            __syncwarp();
            if (lane < 4) before[nb * 4 + lane] = was;
            __syncwarp();
        }
        item += n;
        int coming = 0;  // tiles of the next chunk that are this warp's
        ahead = 0;
        if (item < end) {
            cur.t += n - 1;
            moved = cur.next(c, meta);
            if constexpr (kOne) load_scores(cur.slot(0), length_of(item));  // on their way while the values are weighed
            coming = share.count(length_of(item));
        }
        const Strip zn = cur.strip();
        __syncthreads();
#pragma unroll 1
        for (int k = share.first; k < n; k += share.step) {
            if (flying == kDepth) asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            Planes v;
            const bool limit = v.load<false>(ring + from * kSlice);
            if (limit) v.load<true>(ring + from * kSlice);
            from ^= 1;
            flying--;
            __syncwarp();
            if (fetched < mine) fetch(z, t0 + share.first + fetched++ * share.step);
            else if (ahead < coming) fetch(zn, cur.t + share.first + ahead++ * share.step);
            for (int nb = 0; nb < (kOne ? 1 : z.blocks); nb++) {
                const uint4 *p = pb + (k * most + nb) * 64 + place_of(lane), b2[2] = {p[0], p[32]};
                uint32_t y[4];
                if (limit) weigh<true>(v, b2, y);
                else weigh<false>(v, b2, y);
                const size_t slot = (size_t)(slot0 + nb * tiles + k);
                uint32_t *dst = reinterpret_cast<uint32_t *>(c.tv + (slot * 8 + g) * c.dim + share.part * 32 + 2 * t4);
#pragma unroll
                for (int o = 0; o < 4; o++)
                    if (o < share.octets) dst[4 * o] = y[o];
                if (share.part == 0) {
                    const int2 sum = sum_of(b2);
                    int2 *f = c.fsum + slot * 8 + 2 * t4;
                    if (g == 0) {
                        f[0].y = sum.x;
                        f[1].y = sum.y;
                    }
                    __syncwarp();
                }
            }
        }
    }
    report(c, worst);
}

// ---- join ---------------------------------------------------------------------------
// The request of row r: the last one whose rows start at or before it.  By a whole warp;
// at most 1024 requests in two steps.
static __device__ __forceinline__ uint32_t request_of(const uint32_t *offsets, uint32_t requests, uint32_t r) {
    const uint32_t lane = threadIdx.x & 31, step = (requests + 31) / 32;
    uint32_t at = lane * step;
    uint32_t before = __ballot_sync(0xffffffffu, at < requests && __ldcg(offsets + min(at, requests - 1)) <= r);
    const uint32_t block = before ? (31 - __clz(before)) * step : 0;
    if (step == 1) return block;
    at = block + lane;
    before = __ballot_sync(0xffffffffu, lane < step && at < requests && __ldcg(offsets + min(at, requests - 1)) <= r);
    return before ? block + 31 - __clz(before) : block;
}

// The same where offsets may be out of order, which misleads a search: the first request whose row it is, of those that
// are not void; the number of requests where there is none.  By a whole warp.
static __device__ __noinline__ uint32_t claimant_of(const uint32_t *offsets, const Meta *meta, uint32_t requests, uint32_t r) {
    for (uint32_t first = 0; first < requests; first += 32) {
        const uint32_t b = first + (threadIdx.x & 31);
        bool mine = false;
        if (b < requests) {  // (a row in front of the request's is far behind it in 32 bits)
            const int rows = __ldcg(&meta[b].rows);
            mine = rows > 0 && r - __ldcg(offsets + b) < (uint32_t)rows;
        }
        const uint32_t who = __ballot_sync(0xffffffffu, mine);
        if (who) return first + (uint32_t)__ffs(who) - 1;
    }
    return requests;
}

constexpr int kShortTiles = 255;  // tiles whose sums stay below 2^31: of values 2^23 each, of probabilities 2^22
constexpr int kMaxStretches = 3;  // per warp
constexpr int kAhead = 16;        // tiles loaded at once
constexpr int kMaxJoinWarps = 16;

// x times a factor f < 1 (Q2.14), rounded
static __device__ __forceinline__ int times(int x, int f) { return (int)(((long long)x * (4 * f) + 32768) >> 16); }
// Sum of a word's low or high half and x
static __device__ __forceinline__ int add_low(uint32_t w, int x) {
    int r;
    asm("dp2a.lo.s32.s32 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0x0001), "r"(x));
    return r;
}
static __device__ __forceinline__ int add_high(uint32_t w, int x) {
    int r;
    asm("dp2a.lo.s32.s32 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0x0100), "r"(x));
    return r;
}
// Four elements of a row over its sum, as two words
static __device__ __forceinline__ uint2 quotient(const int (&x)[4], int sum) {
    const long long inv = sat16(rnd((long long)llmx::recip_q16(sum < 16 ? 16 : sum), 8));
    auto one = [&](int y) { return (int)(((long long)y * inv + 32768) >> 16); };
    return make_uint2(pack_sat16(one(x[0]), one(x[1])), pack_sat16(one(x[2]), one(x[3])));
}

// What tiles without a factor, but for the first one's, do to a row's four elements: their sums, and (of a
// long text) how far from what comes in they can get on the way, by the least and the largest value.
struct Stretch {
    int s[4];
    uint32_t lo, hi;  // of pairs of elements; once closed, the furthest down and up, over 256 (2^14 tiles of 2^15 at most)
    int factor, start, tiles, psum;
    // A tile's P add up to 2^20 at most, those of a long stretch to more than 32 bits hold.  From kFull on four times the sum
    // are 2^31 or more, and what they are added to is not negative: the sum saturates, by how much need not be known.
    static constexpr int kFull = 1 << 29;
    // p: of 32 tiles at most
    template <bool kLong>
    __device__ __forceinline__ void add_psum(int p) {
        psum += p;
        if constexpr (kLong) psum = min(psum, kFull);
    }
    template <bool kLong>
    __device__ __forceinline__ void close(int end, int p) {
        tiles = end - start;
        add_psum<kLong>(p);
        if constexpr (kLong) {
            lo = (uint32_t)(tiles * min(llmx::lo16(lo), llmx::hi16(lo)));
            hi = (uint32_t)(tiles * max(llmx::lo16(hi), llmx::hi16(hi)));
        }
    }
    __device__ __forceinline__ void clear(int f, int t) {
        s[0] = s[1] = s[2] = s[3] = 0;
        lo = hi = 0;
        factor = f;
        start = t;
        psum = 0;
    }
    template <bool kLong>
    __device__ __forceinline__ void add(uint2 v) {
        s[0] = add_low(v.x, s[0]);
        s[1] = add_high(v.x, s[1]);
        s[2] = add_low(v.y, s[2]);
        s[3] = add_high(v.y, s[3]);
        if constexpr (kLong) {
            lo = __vmins2(lo, __vmins2(v.x, v.y));
            hi = __vmaxs2(hi, __vmaxs2(v.x, v.y));
        }
    }
};

// One query head's row per CTA.  A lane has four elements, a warp an equal part of the tiles.  Between
// tiles that raise the maximum (whose factor is not 1: few in a long text) the recurrence only adds,
// so a warp gives what its tiles do to any value that comes in as a few stretches, and the first
// warp, which starts from 0, puts them together; tiles beyond a warp's kMaxStretches it goes
// through itself, and a stretch on which something might saturate tile by tile.  Tile by tile throughout
// it took 224 us of a request of 32768 positions with cold caches, so 18; 64 x 8192: 66, so 21 (34 MB).  A text whose positions
// all weigh the same goes tile by tile: all three launches 44 us for 28 at 32768 positions, 3.7 ms for 0.44 at 2^20.
template <bool kLong>
__global__ void __launch_bounds__(32 * kMaxJoinWarps) k_join(const Call c) {
    extern __shared__ __align__(1024) unsigned char dynamic[];
    __shared__ int counts[kMaxJoinWarps], rest[kMaxJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
    const int quads = c.dim >> 2;
    Stretch *stretches = reinterpret_cast<Stretch *>(dynamic);  // [warps - 1][kMaxStretches][32]
    // This launch starts once every CTA of k_values has waited for k_scores, so that what came before k_scores'
    // end (the requests, and what k_scores made of them) can be read, through the L2, before its own wait.
    const uint32_t row = blockIdx.x / c.heads;
    const int head = (int)(blockIdx.x - row * c.heads);
    const uint32_t b = request_of(c.offsets, c.requests, row);
    uint32_t begin = __ldcg(c.offsets + b);
    const uint32_t behind = __ldcg(c.offsets + b + 1);
    auto meta_of = [&](uint32_t b) {
        const int4 m4 = __ldcg(reinterpret_cast<const int4 *>(c.meta + b));
        return Meta{m4.x, m4.y, m4.z, m4.w};
    };
    Meta m = meta_of(b);
    pdl_wait();
    pdl_trigger();
    if (row < begin || row >= behind || m.rows < 0) {  // of no request, or of a void one, or not found
        if (__ldcg(&c.meta[c.requests].rows) == 0) return;
        const uint32_t other = claimant_of(c.offsets, c.meta, c.requests, row);
        if (other == c.requests) return;
        begin = __ldcg(c.offsets + other);
        m = meta_of(other);
    }
    const int h = head / c.group, col = (int)(row - begin) * c.group + head - h * c.group;
    const int blocks = (m.rows * c.group + 7) / 8;
    const size_t at = ((size_t)m.slot + (size_t)(h * blocks + (col >> 3)) * m.tiles) * 8 + (col & 7);
    const uint2 *tv = reinterpret_cast<const uint2 *>(c.tv + at * c.dim) + min(lane, quads - 1);
    const int2 *fsum = c.fsum + at;
    const uint32_t step = 8 * quads;  // from a tile to the next
    auto begin_of = [&](int w) { return m.tiles * w / warps; };

    int sum = 0, x[4] = {0, 0, 0, 0};
    auto apply = [&](const Stretch &p) {
        if (p.factor != 16384) {  // a factor of 1 leaves everything as it is
            sum = times(sum, p.factor);
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = times(x[k], p.factor);
        }
        if constexpr (kLong) {
            // x + 256 h is above 2^31 - 1 just where floor(x / 256) + h is above 2^23 - 1, below -2^31 where that is below
            // -2^23; likewise of sum + 4 psum: nothing here leaves 32 bits.
            const bool far = (max(max(x[0], x[1]), max(x[2], x[3])) >> 8) + (int)p.hi > INT_MAX >> 8 ||
                             (min(min(x[0], x[1]), min(x[2], x[3])) >> 8) + (int)p.lo < INT_MIN >> 8 || (sum >> 2) + p.psum > INT_MAX >> 2;
            if (__any_sync(0xffffffffu, far)) {
#pragma unroll 1
                for (int t = p.start; t < p.start + p.tiles; t++) {
                    const uint2 v = tv[(size_t)t * step];
                    sum = llmx::add_sat(sum, 4 * fsum[t * 8].y);
                    x[0] = llmx::add_sat(x[0], llmx::lo16(v.x) * 256);
                    x[1] = llmx::add_sat(x[1], llmx::hi16(v.x) * 256);
                    x[2] = llmx::add_sat(x[2], llmx::lo16(v.y) * 256);
                    x[3] = llmx::add_sat(x[3], llmx::hi16(v.y) * 256);
                }
                return;
            }
        }
        sum += 4 * p.psum;
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = (int)((uint32_t)x[k] + 256u * (uint32_t)p.s[k]);
    };
    // Tiles t0 .. t1 - 1 as stretches, which are applied or kept in mine[]; returns where the place for them ran out.
    auto walk = [&](int t0, int t1, bool use, Stretch *mine, int &count) {
        Stretch p;
        bool open = false;
        for (int w0 = t0; w0 < t1; w0 += 32) {
            const int n = min(32, t1 - w0);
            const int2 f = lane < n ? fsum[(w0 + lane) * 8] : make_int2(16384, 0);
            uint2 v[kAhead];
            auto load = [&](int b0) {
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    v[i] = make_uint2(0, 0);
                    if (b0 + i < n) v[i] = tv[(size_t)(w0 + b0 + i) * step];
                }
            };
            // with the factors, not after them: 64 x 8192 132.6 -> 131.2 in all; a text of 32768 positions 28.5 -> 29.2
            if constexpr (!kLong) load(0);
            uint32_t turns = __ballot_sync(0xffffffffu, f.x != 16384);
            if (!open) {
                p.clear(__shfl_sync(0xffffffffu, f.x, 0), w0);
                turns &= ~1u;
                open = true;
            }
            int from = 0;  // of this window's tiles, the first whose P is not in the stretch
#pragma unroll 1
            for (int b0 = 0; b0 < n; b0 += kAhead) {
                if (kLong || b0) load(b0);
                if ((turns >> b0 & ((1u << kAhead) - 1)) == 0) {
#pragma unroll
                    for (int i = 0; i < kAhead; i++) p.add<kLong>(v[i]);
                    continue;
                }
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    const int t = b0 + i;
                    if (turns >> t & 1u) {  // the stretch ends here
                        if (!use && count + 1 == kMaxStretches) {
                            p.close<kLong>(w0 + t, __reduce_add_sync(0xffffffffu, lane >= from && lane < t ? f.y : 0));
                            mine[count++ * 32] = p;
                            return w0 + t;
                        }
                        p.close<kLong>(w0 + t, __reduce_add_sync(0xffffffffu, lane >= from && lane < t ? f.y : 0));
                        from = t;
                        if (use) apply(p);
                        else mine[count++ * 32] = p;
                        p.clear(__shfl_sync(0xffffffffu, f.x, t), w0 + t);
                    }
                    p.add<kLong>(v[i]);
                }
            }
            p.add_psum<kLong>(__reduce_add_sync(0xffffffffu, lane >= from ? f.y : 0));
        }
        if (open) {
            p.close<kLong>(t1, 0);
            if (use) apply(p);
            else mine[count++ * 32] = p;
        }
        return t1;
    };
    int count = 0;
    const int left = walk(begin_of(warp), begin_of(warp + 1), warp == 0, stretches + (warp - 1) * kMaxStretches * 32 + lane, count);
    if (warps > 1) {
        if (lane == 0) {
            counts[warp] = count;
            rest[warp] = left;
        }
        __syncthreads();
        if (warp != 0) return;
#pragma unroll 1
        for (int w = 1; w < warps; w++) {
#pragma unroll 1
            for (int k = 0; k < counts[w]; k++) apply(stretches[((w - 1) * kMaxStretches + k) * 32 + lane]);
            if (rest[w] < begin_of(w + 1)) walk(rest[w], begin_of(w + 1), true, nullptr, count);
        }
    }
    if (lane < quads) *reinterpret_cast<uint2 *>(c.out + (size_t)row * c.ld_out + (size_t)head * c.dim + 4 * lane) = quotient(x, sum);
}

// ---- all at once --------------------------------------------------------------------
// A cluster of CTAs per (request, key head), each with an equal part of its tiles, goes through the
// three steps with everything in shared memory: scores, the maxima of the CTAs before from these,
// probabilities (in place of the scores), values, which go to the CTA that has their column, and the
// recurrence there.  Latency bounds it (issue slots 25 to 29 %): two meetings of the cluster, keys before values,
// and at 64 requests of up to 2304 positions 1024 CTAs in two turns, 29.8 us for 71 MB.
struct Places {  // in dynamic shared memory, in bytes
    int prob, exps, runs, tops, base, maxima, tv, fsum, column, queries, size;
    __host__ __device__ Places(int tiles, int cluster, int most, int dim) {
        int at = kWarps * kSlice;  // (a tile a warp)
        auto place = [&](int n) {
            const int was = at;
            at += (n + 15) / 16 * 16;
            return was;
        };
        const int own = (most * 8 + cluster - 1) / cluster;  // columns of a CTA
        prob = place(tiles * most * 1024);
        exps = place(kExpWords * 4);
        runs = place((tiles + 1) * most * 16);
        tops = place(tiles * most * 64);
        base = place(most * 16);
        maxima = place(cluster * most * 16);
        tv = place(own * tiles * cluster * dim * 2);
        fsum = place(own * tiles * cluster * 8);
        column = place((int)sizeof(Column));
        queries = place(2 * most * ((dim + 31) / 32) * 512);
        size = at;
    }
};
static __device__ __forceinline__ void put(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
// (aligned: a warp's lanes meet first, here and before the arrival and the matrix instructions that follow
// what only some of them did)
static __device__ __forceinline__ void cluster_meet() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int KS, bool kOne>
__global__ void __launch_bounds__(kThreads, 4) k_attend(const Call c) {
    extern __shared__ __align__(1024) unsigned char dynamic[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const int most = kOne ? 1 : c.blocks;
    const int log = c.cluster_log, cluster = 1 << log;
    const Places at(c.tiles, cluster, most, c.dim);
    unsigned char *ring = dynamic + warp * kSlice;
    uint4 *queries = reinterpret_cast<uint4 *>(dynamic + at.queries), *rests = queries + most * KS * 32;
    uint32_t *score = reinterpret_cast<uint32_t *>(dynamic + at.prob);  // [tiles][most][64 positions][4 pairs], then the probabilities
    const int16_t *exps = reinterpret_cast<const int16_t *>(dynamic + at.exps);
    uint32_t *runs = reinterpret_cast<uint32_t *>(dynamic + at.runs);      // [tiles + 1][most * 4] maxima up to a tile of this CTA's
    uint32_t *tops = reinterpret_cast<uint32_t *>(dynamic + at.tops);      // [tiles][most][4 blocks][4 pairs]
    uint32_t *base = reinterpret_cast<uint32_t *>(dynamic + at.base);      // [most * 4] maxima of the CTAs before
    uint32_t *maxima = reinterpret_cast<uint32_t *>(dynamic + at.maxima);  // [cluster][most * 4]
    Column &column = *reinterpret_cast<Column *>(dynamic + at.column);
    for (int i = threadIdx.x; i < kExpWords; i += kThreads)
        reinterpret_cast<uint32_t *>(dynamic + at.exps)[i] = reinterpret_cast<const uint32_t *>(c.exps)[i];
    pdl_wait();
    pdl_trigger();
    __shared__ int all_tiles[kWarps];
    const int strip = (int)(blockIdx.x >> log), rank = (int)(blockIdx.x & (unsigned)(cluster - 1));
    const int b = strip / c.kv, h = strip - b * c.kv, nb0 = (int)blockIdx.y * most;
    const uint32_t o0 = c.offsets[b], o1 = c.offsets[b + 1], len = c.lengths[b];
    if (o0 > o1 || o1 > c.rows || o1 - o0 > (uint32_t)c.max_block || len > c.longest) {
        if (threadIdx.x == 0) atomicOr(c.error, kErrRequest);
        return;  // (the whole cluster)
    }
    const int rows = (int)(o1 - o0), columns = min(rows * c.group - nb0 * 8, most * 8);
    if (columns <= 0) return;
    __syncwarp();
    llmx::cluster_arrive();
    const Strip z{c.table + (size_t)b * c.ld_table, h, rows, (int)len, (columns + 7) >> 3, o0, nb0 * 8};
    const int n = (z.length + kTile - 1) / kTile, t0 = n * rank >> log, own = (n * (rank + 1) >> log) - t0;
    const int pairs = z.blocks * 4;
    uint32_t worst = 0;

    // ---- scores
    const Share share(c.dim, warp);
    int fetched = share.first;
    auto fetch = [&]() {
        if (fetched < own) {
            fetch_values(c, z, t0 + fetched, share.part, ring, worst);
            fetched += share.step;
        }
        commit();
    };
    {
        uint4 raw[2][KS];
        KeyPages pages;
        int p0 = t0 * kTile + warp * 16;
        if (own > 0) {
            pages.load(c, z, p0, worst);
            load_keys<KS>(c, z, pages, p0, raw);
        }
        pages.load(c, z, p0 + kTile, worst);
        stage_queries<KS>(c, z, warp, kWarps, queries, rests, column);
        fetch();
        // whether the whole call is within what the handle was made for
        int sum = 0;
        for (uint32_t i = threadIdx.x; i < c.requests; i += kThreads) {
            int rows, tiles;
            if (request(c, i, rows, tiles)) sum += tiles;
        }
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) all_tiles[warp] = sum;
        __syncthreads();
#pragma unroll 1
        for (int k = 0; k < own; k++, p0 += kTile) {
            score_tile<KS, kOne>(c, z, p0, raw, z, pages, p0 + kTile, queries, rests, column, [&](int nb, uint32_t top, const uint32_t(&w)[2]) {
                const int block = (k * most + nb) * 4 + warp;
                score[block * 64 + lane] = w[0];
                score[block * 64 + 32 + lane] = w[1];
                if (lane < 4) tops[block * 4 + lane] = top;
            });
            pages.load(c, z, p0 + 2 * kTile, worst);
        }
    }
    __syncthreads();
    llmx::cluster_wait();  // every CTA of the cluster is there
    // ---- maxima
    for (int i = threadIdx.x; i < pairs; i += kThreads) {
        uint32_t m = 0;
        const uint32_t *top = tops + (i >> 2) * 16 + (i & 3);
        for (int k = 0; k < own; k++, top += most * 16) {
            runs[k * most * 4 + i] = m;
            m = __vmaxu2(m, __vmaxu2(__vmaxu2(top[0], top[4]), __vmaxu2(top[8], top[12])));
        }
        runs[own * most * 4 + i] = m;
        for (int r = rank + 1; r < cluster; r++) put(llmx::remote(maxima + rank * most * 4 + i, (uint32_t)r), m);
    }
    cluster_meet();
    for (int i = threadIdx.x; i < pairs; i += kThreads) {
        uint32_t m = 0;
        for (int r = 0; r < rank; r++) m = __vmaxu2(m, maxima[r * most * 4 + i]);
        base[i] = m;
    }
    __syncthreads();
    // ---- probabilities: a tile against 8 columns a warp, in place
    // Column nb * 8 + i belongs to CTA i mod cluster (at most 8), which holds `stride` tiles of each of its columns.
    const int stride = c.tiles << log, of_block = 8 >> log;
    auto owner = [&](int offset, int i) { return llmx::remote(dynamic + offset, (uint32_t)(i & (cluster - 1))); };
    const int cp = lane & 3, pos = 8 * (lane >> 4) + 2 * (lane >> 2 & 3);
    const uint32_t factor0 = owner(at.fsum, 2 * cp), factor1 = owner(at.fsum, 2 * cp + 1);
    for (int k = 0, nb = warp; k < own;) {
        if (!kOne && nb >= z.blocks) {
            nb -= z.blocks;
            k++;
            continue;
        }
        if (kOne) {  // (one block: the warps take the tiles in turn)
            k = nb;
            if (k >= own) break;
        }
        const int block = kOne ? 0 : nb, col = block * 8 + 2 * cp;
        uint32_t *here = score + (k * most + block) * 256;
        uint32_t w[4][2];
#pragma unroll
        for (int blk = 0; blk < 4; blk++)
#pragma unroll
            for (int i = 0; i < 2; i++) w[blk][i] = here[blk * 64 + (pos + i) * 4 + cp];
        const uint32_t before = base[block * 4 + cp], was = __vmaxu2(before, runs[k * most * 4 + block * 4 + cp]),
                       m = __vmaxu2(before, runs[(k + 1) * most * 4 + block * 4 + cp]);
        const int2 seen = *reinterpret_cast<const int2 *>(&column.seen[col]);
        const int p = (t0 + k) * kTile;
        __syncwarp();
#pragma unroll
        for (int blk = 0; blk < 4; blk++)
            probabilities(exps, w[blk][0], w[blk][1], m, p + pos + 16 * blk, seen.x, seen.y, blk, reinterpret_cast<uint4 *>(here));
        if (lane < 4) {
            const uint32_t d = m - __vmaxu2(was, __vmaxu2(m, 0x08000800u) - 0x08000800u);
            const uint32_t f0 = (uint32_t)(((block * of_block + (2 * cp >> log)) * stride + t0 + k) * 8);
            const uint32_t f1 = (uint32_t)(((block * of_block + (2 * cp + 1 >> log)) * stride + t0 + k) * 8);
            if (col < columns) put(factor0 + f0, (uint32_t)exps[d & 0xffffu]);
            if (col + 1 < columns) put(factor1 + f1, (uint32_t)exps[d >> 16]);
        }
        nb += kWarps;
    }
    __syncthreads();
    // ---- values
    const uint32_t values = owner(at.tv, g) + (uint32_t)(share.part * 64 + 4 * t4);
#pragma unroll 1
    for (int k = share.first; k < own; k += share.step) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        Planes v;
        const bool limit = v.load<false>(ring);
        if (limit) v.load<true>(ring);
        __syncwarp();
        fetch();
        for (int nb = 0; nb < (kOne ? 1 : z.blocks); nb++) {
            const uint4 *p = reinterpret_cast<const uint4 *>(score) + (k * most + nb) * 64 + place_of(lane), b2[2] = {p[0], p[32]};
            uint32_t y[4];
            if (limit) weigh<true>(v, b2, y);
            else weigh<false>(v, b2, y);
            if (nb * 8 + g < columns) {
                const uint32_t to = values + (uint32_t)(((nb * of_block + (g >> log)) * stride + t0 + k) * 2 * c.dim);
#pragma unroll
                for (int o = 0; o < 4; o++)
                    if (o < share.octets) put(to + 16 * o, y[o]);
            }
            __syncwarp();
            if (share.part == 0) {
                const int2 sum = sum_of(b2);
                const uint32_t f0 = (uint32_t)(((nb * of_block + (2 * cp >> log)) * stride + t0 + k) * 8);
                const uint32_t f1 = (uint32_t)(((nb * of_block + (2 * cp + 1 >> log)) * stride + t0 + k) * 8);
                if (g == 0 && nb * 8 + 2 * cp < columns) put(factor0 + f0 + 4, (uint32_t)sum.x);
                if (g == 0 && nb * 8 + 2 * cp + 1 < columns) put(factor1 + f1 + 4, (uint32_t)sum.y);
                __syncwarp();
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    report(c, worst);
    cluster_meet();  // nothing is sent to another CTA from here on
    long long total = 0;
    for (int w = 0; w < kWarps; w++) total += all_tiles[w];
    if (total * c.kv > c.capacity) {
        if (threadIdx.x == 0) atomicOr(c.error, kErrBudget);
        return;
    }
    // ---- join: a column a warp, four elements a lane (too few tiles for anything to saturate)
    const int quads = c.dim >> 2;
    for (int idx = warp;; idx += kWarps) {
        const int col = kOne || log == 3 ? (idx << log) + rank : (idx >> (3 - log)) * 8 + ((idx & (of_block - 1)) << log) + rank;
        if (col >= columns) break;
        const uint2 *tv = reinterpret_cast<const uint2 *>(dynamic + at.tv) + (size_t)idx * stride * quads + min(lane, quads - 1);
        const int2 *fsum = reinterpret_cast<const int2 *>(dynamic + at.fsum) + idx * stride;
        int sum = 0, x[4] = {0, 0, 0, 0};
#pragma unroll 4
        for (int t = 0; t < n; t++) {
            const uint2 w = tv[t * quads];
            const int2 f = fsum[t];
            if (f.x != 16384) {
                sum = times(sum, f.x);
#pragma unroll
                for (int k = 0; k < 4; k++) x[k] = times(x[k], f.x);
            }
            sum += 4 * f.y;
            x[0] += llmx::lo16(w.x) * 256;
            x[1] += llmx::hi16(w.x) * 256;
            x[2] += llmx::lo16(w.y) * 256;
            x[3] += llmx::hi16(w.y) * 256;
        }
        const int j = (z.col0 + col) / c.group, head = h * c.group + z.col0 + col - j * c.group;
        if (lane < quads) *reinterpret_cast<uint2 *>(c.out + (size_t)(z.row0 + j) * c.ld_out + (size_t)head * c.dim + 4 * lane) = quotient(x, sum);
    }
}

// ---- append -------------------------------------------------------------------------
struct AppendCall {
    const int16_t *qkv;
    size_t ld_qkv;
    int16_t *q;
    size_t ld_q;
    int16_t *k, *v;
    const int32_t *table;
    size_t ld_table;
    const int16_t *rope;
    uint32_t positions;
    const uint32_t *offsets, *lengths;
    uint32_t rows, requests, pages;
    int heads, kv, dim, page_len;
    uint32_t parts_magic;  // for dividing by dim / 16
    int *error;
};

// Two pairs.  A table may hold any 16-bit values: x0 c - x1 s stays within 2^31 - 2^15 even so, and x1 c + x0 s
// leaves 32 bits in one case only, as 2^31, where the wrapped sum is one that nothing else gives.
static __device__ __forceinline__ void turn2(uint32_t x0, uint32_t x1, uint32_t c, uint32_t s, uint32_t &y0, uint32_t &y1) {
    auto minus = [](int a, int ca, int b, int cb) { return (a * ca + 128 - b * cb) >> 8; };
    auto plus = [](int a, int ca, int b, int cb) {
        const int w = (int)((uint32_t)(a * ca) + (uint32_t)(b * cb) + 128u);
        return (w == INT_MIN + 128 ? INT_MAX : w) >> 8;
    };
    const int c0 = llmx::lo16(c), c1 = llmx::hi16(c), s0 = llmx::lo16(s), s1 = llmx::hi16(s);
    const int a0 = llmx::lo16(x0), a1 = llmx::hi16(x0), b0 = llmx::lo16(x1), b1 = llmx::hi16(x1);
    y0 = pack_sat16(minus(a0, c0, b0, s0), minus(a1, c1, b1, s1));
    y1 = pack_sat16(plus(b0, c0, a0, s0), plus(b1, c1, a1, s1));
}

// A CTA per row; a thread turns 8 pairs (i, i + dim/2) of a head, or copies 16 values.  The row's own values are on
// their way while its request, its position, and by that its page and its turn are looked up, one after
// another: that is what a row takes.  8192 rows of 16 + 2 + 2 heads of 128: 21.2 us for 85 MB, 53 % of the issue slots; with
// 2, 3, 4 or 6 rows a CTA 21.4 to 24.5, and 64 rows 2.9 to 5.1 for 2.6.
__global__ void __launch_bounds__(256) k_append(const AppendCall c) {
    pdl_wait();
    pdl_trigger();
    const uint32_t r = blockIdx.x;
    const int parts = c.dim >> 4, half = c.dim >> 1, items = (c.heads + 2 * c.kv) * parts;  // 16 values each
    auto load = [&](int i, int &head, int &part, uint4 &x0, uint4 &x1) {
        head = parts == 1 ? i : (int)__umulhi((uint32_t)i, c.parts_magic);
        part = i - head * parts;
        const int16_t *src = c.qkv + (size_t)r * c.ld_qkv + (size_t)head * c.dim;
        const bool turned = head < c.heads + c.kv;
        x0 = *reinterpret_cast<const uint4 *>(src + (turned ? 8 : 16) * part);
        x1 = *reinterpret_cast<const uint4 *>(src + (turned ? half + 8 * part : 16 * part + 8));
    };
    int head = 0, part = 0;
    uint4 x0, x1;
    if ((int)threadIdx.x < items) load((int)threadIdx.x, head, part, x0, x1);
    // the first warp looks the row's place up
    __shared__ uint32_t where[3];  // page (kNowhere: the row is left out), position, and that within the page
    constexpr uint32_t kNowhere = 0xffffffffu;
    if (threadIdx.x < 32) {
        const uint32_t b = request_of(c.offsets, c.requests, r);
        const uint32_t first = __ldcg(c.offsets + b), last = __ldcg(c.offsets + b + 1), length = __ldcg(c.lengths + b);
        const long long position = (long long)length - (long long)(last - first) + (r - first);
        const uint32_t at = (uint32_t)position / (uint32_t)c.page_len;
        uint32_t page = kNowhere;
        if (r >= first && r < last && position >= 0) {  // of a request, and not in front of the sequence
            int bad = 0;
            if (position >= c.positions || at >= c.ld_table) {
                bad = kErrRequest;
            } else {
                page = (uint32_t)__ldcg(c.table + (size_t)b * c.ld_table + at);
                if (page >= c.pages) {
                    page = kNowhere;
                    bad = kErrPage;
                }
            }
            if (bad && threadIdx.x == 0) atomicOr(c.error, bad);
        }
        if (threadIdx.x == 0) {
            where[0] = page;
            where[1] = (uint32_t)position;
            where[2] = (uint32_t)position - at * (uint32_t)c.page_len;
        }
    }
    __syncthreads();
    const uint32_t page = where[0], position = where[1];
    const size_t inside = where[2];
    if (page == kNowhere) return;
    const int16_t *turn = c.rope + (size_t)position * c.dim;
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        if (i != (int)threadIdx.x) load(i, head, part, x0, x1);
        uint4 y0 = x0, y1 = x1;
        int16_t *dst;
        int at0 = 16 * part, at1 = 16 * part + 8;
        if (head < c.heads + c.kv) {
            const uint4 cs = *reinterpret_cast<const uint4 *>(turn + 8 * part), sn = *reinterpret_cast<const uint4 *>(turn + half + 8 * part);
            turn2(x0.x, x1.x, cs.x, sn.x, y0.x, y1.x);
            turn2(x0.y, x1.y, cs.y, sn.y, y0.y, y1.y);
            turn2(x0.z, x1.z, cs.z, sn.z, y0.z, y1.z);
            turn2(x0.w, x1.w, cs.w, sn.w, y0.w, y1.w);
            at0 = 8 * part;
            at1 = half + 8 * part;
        }
        if (head < c.heads) dst = c.q + (size_t)r * c.ld_q + (size_t)head * c.dim;
        else {
            const bool key = head < c.heads + c.kv;
            dst = (key ? c.k : c.v) + (((size_t)page * c.kv + (head - c.heads - (key ? 0 : c.kv))) * c.page_len + inside) * c.dim;
        }
        *reinterpret_cast<uint4 *>(dst + at0) = y0;
        *reinterpret_cast<uint4 *>(dst + at1) = y1;
    }
}

}  // namespace

struct llmx_paged {
    int dev = 0, sms = 0;
    int heads = 0, kv = 0, dim = 0, page_len = 0;
    bool one = false;  // one column block
    uint32_t max_requests = 0, max_block = 0, max_length = 0;
    long long capacity = 0;  // (key head, tile) items of a call
    uint64_t positions = 0;  // of all requests of a call
    size_t scores_smem = 0, values_smem = 0;
    int scores_ctas = 0, values_ctas = 0;  // that are on the device at once
    int way = -1;  // of attention calls, for tests: see way_of; -1: as choose() estimates
    unsigned char *memory = nullptr;
    Meta *meta = nullptr;
    uint32_t *score = nullptr;
    uint4 *top = nullptr;
    int16_t *tv = nullptr, *exps = nullptr;
    int2 *fsum = nullptr;
    int *error = nullptr;
    uint64_t bytes = 0;
};

namespace {

int fail(int code, const std::string &msg) {
    llmx::set_last_error("paged: " + msg);
    return code;
}
int cuda_fail(const char *what, cudaError_t e) {
    (void)cudaGetLastError();
    return fail(e == cudaErrorMemoryAllocation ? LLMX_ERR_NOMEM : LLMX_ERR_CUDA,
                std::string(what) + ": " + cudaGetErrorString(e));
}

// The handle's device is current for the length of a call.
struct DeviceScope {
    int before = -1, dev;
    cudaError_t err;
    explicit DeviceScope(int d) : dev(d) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != dev) err = cudaSetDevice(dev);
    }
    ~DeviceScope() {
        if (before >= 0 && before != dev) cudaSetDevice(before);
    }
};

// The kernels for a head dimension, and for one column block or more.
const void *attend_kernel(int dim, bool one) {
    switch ((dim + 31) / 32) {
        case 1: return one ? (const void *)k_attend<1, true> : (const void *)k_attend<1, false>;
        case 2: return one ? (const void *)k_attend<2, true> : (const void *)k_attend<2, false>;
        case 3: return one ? (const void *)k_attend<3, true> : (const void *)k_attend<3, false>;
        default: return one ? (const void *)k_attend<4, true> : (const void *)k_attend<4, false>;
    }
}
const void *scores_kernel(int dim, bool one) {
    switch ((dim + 31) / 32) {
        case 1: return one ? (const void *)k_scores<1, true> : (const void *)k_scores<1, false>;
        case 2: return one ? (const void *)k_scores<2, true> : (const void *)k_scores<2, false>;
        case 3: return one ? (const void *)k_scores<3, true> : (const void *)k_scores<3, false>;
        default: return one ? (const void *)k_scores<4, true> : (const void *)k_scores<4, false>;
    }
}
const void *values_kernel(bool one) { return one ? (const void *)k_values<true> : (const void *)k_values<false>; }

template <class T>
cudaError_t launch(const void *fn, unsigned grid, int threads, size_t smem, const T &call, cudaStream_t s, int cluster = 0,
                   unsigned grid_y = 1) {
    T copy = call;
    void *args[] = {&copy};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, grid_y);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

// How k_attend takes a call, or ctas = 0 where the three launches are faster.
struct Clusters {
    uint64_t ctas = 0;
    int log = 0, tiles = 0, blocks = 0, smem = 0;
};
// As one number: 0 for three launches, else 16 log + blocks (1 to 16).
int way_of(int log, int blocks) { return 16 * log + blocks; }
// Estimates whose order was fitted to measurements of every way (2090 calls: 1 to 64 query heads of 16 to 128, 1 to 128
// requests of up to 20 to 16000 positions, all as long and of any length, 1 to 8 rows; caches in HBM and in the L2): what is picked
// was 1.8 % slower than the best way on average (4.9 % by the estimate before, which knew 16 heads of 128 only), more than
// 20 % in 45 of them, 56 % at most (24 requests of up to 320, 3 rows: 15.9 us by clusters of 4, 10.2 of 2). 420 of the calls
// were drawn, from about what perf/more_operators.py draws, and each counted as 4 to 12 of the 1670 of a grid, those of
// requests of any length least: ragged blocks of 2 to 5 rows are where it picks worst.
//   Three launches: a start, more per further column block, and the tiles that an SM has.
//   Clusters: a CTA's tiles, slower for each CTA that shares its SM and each further block; CTAs beyond those that the
// SMs hold at once (4, or what their memory allows, and a little less for larger clusters) come in later turns, which a
// part of one costs like most of a whole one.
// Lengths are on the device: requests count as long as the longest, as far as the handle's room for all allows. The shorter
// they are on average, the fewer tiles three launches have and the cheaper are the later turns.
// 16 heads of 128, 1 row: 64 of 1024 19.7 us by clusters of 4, 26.6 of 8, 27.6 by three launches; one of 2048 11.0 (of 8) and
// 12.2, of 4096 17.5 and 14.5; 64 of 4096 85 and 76.
Clusters choose(const llmx_paged *p, uint64_t requests, int all, int most) {
    Clusters best;
    const uint64_t strips = requests * (uint64_t)p->kv;
    const double fill = std::min(1.0, ((double)p->positions / kTile + 0.5 * (double)requests) / ((double)requests * all));
    const double per_tile = 0.2 + 0.2 * ((p->dim + 31) / 32), shorter = std::pow(fill, 2.5), fewer = std::pow(fill, 0.3);
    double least = 18.2 + 1.06 * (most - 1) + 0.56 * per_tile * fill * (double)strips * all / p->sms * (1 + 0.87 * (most - 1));
    if (p->way > 0) least = HUGE_VAL;
    if (all > kShortTiles || p->way == 0) return best;
    for (int log = 0; log <= 3; log++) {
        const int cluster = 1 << log, tiles = (all + cluster - 1) / cluster;
        if (log && cluster > all) break;
        for (int blocks = 1; blocks <= most; blocks++) {
            const int groups = (most + blocks - 1) / blocks;
            if (blocks > 1 && (most + blocks - 2) / (blocks - 1) == groups) continue;  // no fewer groups for more blocks
            const Places at(tiles, cluster, blocks, p->dim);
            if (at.size > kMaxSmem) continue;
            const double room = std::min(4, kSmemOfSm / (at.size + 2048)), load = fewer * (double)strips * cluster * groups / p->sms;
            const double work = tiles * per_tile * (1 + 0.4 * (blocks - 1));
            const double turn = work * (2.16 + (blocks > 1 ? 0.17 : groups > 1 ? 0.22 : 0.12) * std::min(load, room));
            const double turns = std::max(1.0, load / (room * (1 - 0.027 * log)));
            const double us = 4.3 + turn + (turns - 1 + 0.39 * (std::ceil(turns - 1e-9) - turns)) * (8.9 + 0.9 * turn * shorter);
            if (us < least && (p->way < 0 || p->way == way_of(log, blocks))) {
                least = us;
                best.ctas = strips * cluster;
                best.log = log;
                best.tiles = tiles;
                best.blocks = blocks;
                best.smem = at.size;
            }
        }
    }
    return best;
}

void release(llmx_paged *p) {
    cudaFree(p->memory);
    delete p;
}

// What append and attention have in common.  0: fine.
int check(const llmx_paged *p, uint32_t requests, const uint32_t *offsets, const uint32_t *lengths, const int32_t *table,
          size_t ld_table, const int16_t *k, const int16_t *v, uint32_t pages) {
    if (requests > p->max_requests)
        return fail(LLMX_ERR_ARG, "requests " + std::to_string(requests) + " above max_requests " + std::to_string(p->max_requests));
    if (!offsets || !lengths || !table || !k || !v) return fail(LLMX_ERR_ARG, "null pointer");
    if (pages == 0 || pages > (uint32_t)INT_MAX) return fail(LLMX_ERR_ARG, "pages must be 1..2^31-1, got " + std::to_string(pages));
    if (ld_table == 0) return fail(LLMX_ERR_ARG, "ld_table must be at least 1");
    if (((uintptr_t)offsets | (uintptr_t)lengths | (uintptr_t)table) & 3u)
        return fail(LLMX_ERR_ARG, "offsets, lengths and table must be 4-byte aligned");
    if (((uintptr_t)k | (uintptr_t)v) & 15u) return fail(LLMX_ERR_ARG, "k and v must be 16-byte aligned");
    return LLMX_OK;
}
int check_rows(const char *what, const void *p, size_t ld, size_t width) {
    if (!p) return fail(LLMX_ERR_ARG, "null pointer");
    if (ld < width || ld % 8 != 0) return fail(LLMX_ERR_ARG, std::string("ld of ") + what + " must be a multiple of 8 not below its width");
    if ((uintptr_t)p & 15u) return fail(LLMX_ERR_ARG, std::string(what) + " must be 16-byte aligned");
    return LLMX_OK;
}

}  // namespace

extern "C" int llmx_paged_create(int device, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t page_len,
                                 uint32_t max_requests, uint32_t max_block, uint32_t max_length, uint64_t max_positions,
                                 void *stream, llmx_paged **out) {
    if (!out) return fail(LLMX_ERR_ARG, "null pointer");
    *out = nullptr;
    if (kv_heads == 0 || heads == 0 || heads > kMaxHeads || heads % kv_heads != 0)
        return fail(LLMX_ERR_ARG, "heads must be 1..1024 and a multiple of kv_heads");
    if (head_dim == 0 || head_dim % 16 != 0 || head_dim > 128)
        return fail(LLMX_ERR_ARG, "head_dim must be a multiple of 16 up to 128, got " + std::to_string(head_dim));
    if (page_len == 0 || page_len % 8 != 0 || page_len > kMaxPageLen)
        return fail(LLMX_ERR_ARG, "page_len must be a multiple of 8 up to 65536, got " + std::to_string(page_len));
    if ((uint64_t)kv_heads * page_len * head_dim >= 1ull << 31) return fail(LLMX_ERR_ARG, "a page must hold fewer than 2^31 values");
    if (max_requests == 0 || max_requests > kMaxRequests)
        return fail(LLMX_ERR_ARG, "max_requests must be 1..1024, got " + std::to_string(max_requests));
    if (max_block == 0 || max_block > (uint32_t)llmx::kMaxRows)
        return fail(LLMX_ERR_ARG, "max_block must be 1..8, got " + std::to_string(max_block));
    if (heads / kv_heads * max_block > kMaxColumns)
        return fail(LLMX_ERR_ARG, "heads / kv_heads * max_block must be at most 128");
    if (max_length == 0 || max_length > kMaxLength)
        return fail(LLMX_ERR_ARG, "max_length must be 1..2^20, got " + std::to_string(max_length));
    if (max_positions == 0) return fail(LLMX_ERR_ARG, "max_positions must be at least 1");
    // every request's last tile may be a partial one
    const uint64_t positions = std::min<uint64_t>(max_positions, (uint64_t)max_requests * max_length);
    const uint64_t tiles = std::min<uint64_t>(positions / kTile + max_requests, (uint64_t)max_requests * ((max_length + kTile - 1) / kTile));
    const uint64_t blocks = (heads / kv_heads * max_block + 7) / 8;
    const uint64_t slots = tiles * kv_heads * blocks;
    if (slots > (uint64_t)INT_MAX) return fail(LLMX_ERR_ARG, "max_positions is too large for these heads");
    DeviceScope scope(device);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    llmx_paged *p = new (std::nothrow) llmx_paged;
    if (!p) return fail(LLMX_ERR_NOMEM, "host allocation failed");
    p->dev = device;
    p->heads = (int)heads;
    p->kv = (int)kv_heads;
    p->dim = (int)head_dim;
    p->page_len = (int)page_len;
    p->max_requests = max_requests;
    p->max_block = max_block;
    p->max_length = max_length;
    p->one = blocks == 1;
    p->capacity = (long long)(tiles * kv_heads);
    p->positions = positions;
    size_t at = 0;
    auto place = [&](size_t n) {
        const size_t was = at;
        at += (n + 255) / 256 * 256;
        return was;
    };
    const size_t error_at = place(4), exps_at = place(kExpWords * 4), meta_at = place((max_requests + 1) * sizeof(Meta)),
                 score_at = place(slots * 8 * kTile * 2), top_at = place(slots * 64), tv_at = place(slots * 8 * head_dim * 2),
                 fsum_at = place(slots * 64);
    p->bytes = at;
    p->scores_smem = 2 * blocks * ((head_dim + 31) / 32) * 512 + (size_t)max_requests * sizeof(Meta);
    const size_t chunk = std::max<size_t>(1, kChunk / blocks);
    p->values_smem = kRing + 2 * chunk * blocks * 1024 + kExpWords * 4 + (3 * kWarps + 4) * blocks * 16 + (size_t)max_requests * sizeof(Meta);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int16_t e16[2049], p18[2049], host[kExpWords * 2] = {};
    llmx::build_exp_tables(e16, p18);
    for (int i = 0; i <= 2048; i++) host[i] = p18[2048 - i];
    cudaError_t e;
    if ((e = cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, device)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(scores_kernel(p->dim, p->one), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(values_kernel(p->one), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(attend_kernel(p->dim, true), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(attend_kernel(p->dim, false), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaFuncSetAttribute((const void *)k_join<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaFuncSetAttribute((const void *)k_join<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaMalloc(reinterpret_cast<void **>(&p->memory), at)) != cudaSuccess ||
        (e = cudaMemsetAsync(p->memory + error_at, 0, 4, s)) != cudaSuccess ||
        (e = cudaMemcpyAsync(p->memory + exps_at, host, sizeof(host), cudaMemcpyHostToDevice, s)) != cudaSuccess ||
        (e = cudaStreamSynchronize(s)) != cudaSuccess) {
        release(p);
        return cuda_fail("create", e);
    }
    int per_sm[2] = {0, 0};
    if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm[0], scores_kernel(p->dim, p->one), kThreads, p->scores_smem)) != cudaSuccess ||
        (e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm[1], values_kernel(p->one), kThreads, p->values_smem)) != cudaSuccess) {
        release(p);
        return cuda_fail("create", e);
    }
    p->scores_ctas = p->sms * std::max(per_sm[0], 1);
    p->values_ctas = p->sms * std::max(per_sm[1], 1);
    auto as = [&](auto *&ptr, size_t where) { ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(p->memory + where); };
    as(p->error, error_at);
    as(p->exps, exps_at);
    as(p->meta, meta_at);
    as(p->score, score_at);
    as(p->top, top_at);
    as(p->tv, tv_at);
    as(p->fsum, fsum_at);
    *out = p;
    return LLMX_OK;
}

extern "C" int llmx_paged_destroy(llmx_paged *p) {
    if (!p) return LLMX_OK;
    DeviceScope scope(p->dev);
    release(p);
    return LLMX_OK;
}

extern "C" int llmx_paged_append(llmx_paged *p, const int16_t *qkv, uint32_t rows, size_t ld_qkv, const uint32_t *offsets,
                                 const uint32_t *lengths, uint32_t requests, const int16_t *rope, uint32_t positions,
                                 const int32_t *table, size_t ld_table, int16_t *k, int16_t *v, uint32_t pages, int16_t *q,
                                 size_t ld_q, void *stream) {
    if (!p) return fail(LLMX_ERR_ARG, "null handle");
    if (rows > kMaxAppendRows) return fail(LLMX_ERR_ARG, "rows must be at most 2^20, got " + std::to_string(rows));
    if (rows == 0 || requests == 0) return LLMX_OK;
    const size_t width = (size_t)(p->heads + 2 * p->kv) * p->dim, q_width = (size_t)p->heads * p->dim;
    if (ld_qkv == 0) ld_qkv = width;
    if (ld_q == 0) ld_q = q_width;
    int rc = check(p, requests, offsets, lengths, table, ld_table, k, v, pages);
    if (rc == LLMX_OK) rc = check_rows("qkv", qkv, ld_qkv, width);
    if (rc == LLMX_OK) rc = check_rows("q", q, ld_q, q_width);
    if (rc == LLMX_OK && (!rope || ((uintptr_t)rope & 15u))) rc = fail(LLMX_ERR_ARG, "rope must be 16-byte aligned and not NULL");
    if (rc != LLMX_OK) return rc;
    DeviceScope scope(p->dev);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    AppendCall c{};
    c.qkv = qkv;
    c.ld_qkv = ld_qkv;
    c.q = q;
    c.ld_q = ld_q;
    c.k = k;
    c.v = v;
    c.table = table;
    c.ld_table = ld_table;
    c.rope = rope;
    c.positions = positions;
    c.offsets = offsets;
    c.lengths = lengths;
    c.rows = rows;
    c.requests = requests;
    c.pages = pages;
    c.heads = p->heads;
    c.kv = p->kv;
    c.dim = p->dim;
    c.page_len = p->page_len;
    c.error = p->error;
    c.parts_magic = (uint32_t)(((1ull << 32) + p->dim / 16 - 1) / (p->dim / 16));
    const int work = (p->heads + 2 * p->kv) * (p->dim / 16);
    const cudaError_t e = launch((const void *)k_append, rows, std::min(256, (work + 31) / 32 * 32), 0, c, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LLMX_OK : cuda_fail("append", e);
}

extern "C" int llmx_paged_attention(llmx_paged *p, const int16_t *q, uint32_t rows, size_t ld_q, const uint32_t *offsets,
                                    const uint32_t *lengths, uint32_t requests, uint32_t longest, const int32_t *table,
                                    size_t ld_table, const int16_t *k, const int16_t *v, uint32_t pages, int16_t *out,
                                    size_t ld_out, void *stream) {
    if (!p) return fail(LLMX_ERR_ARG, "null handle");
    if (rows > kMaxAppendRows) return fail(LLMX_ERR_ARG, "rows must be at most 2^20, got " + std::to_string(rows));
    if (longest > p->max_length)
        return fail(LLMX_ERR_ARG, "longest " + std::to_string(longest) + " above max_length " + std::to_string(p->max_length));
    if (longest == 0) longest = p->max_length;
    if (rows == 0 || requests == 0) return LLMX_OK;
    const size_t width = (size_t)p->heads * p->dim;
    if (ld_q == 0) ld_q = width;
    if (ld_out == 0) ld_out = width;
    int rc = check(p, requests, offsets, lengths, table, ld_table, k, v, pages);
    if (rc == LLMX_OK) rc = check_rows("q", q, ld_q, width);
    if (rc == LLMX_OK) rc = check_rows("out", out, ld_out, width);
    if (rc == LLMX_OK && (longest + p->page_len - 1) / p->page_len > ld_table)
        rc = fail(LLMX_ERR_ARG, "a table row of " + std::to_string(ld_table) + " pages does not hold " + std::to_string(longest) + " positions");
    if (rc != LLMX_OK) return rc;
    DeviceScope scope(p->dev);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    Call c{};
    c.q = q;
    c.ld_q = ld_q;
    c.out = out;
    c.ld_out = ld_out;
    c.k = k;
    c.v = v;
    c.table = table;
    c.ld_table = ld_table;
    c.offsets = offsets;
    c.lengths = lengths;
    c.rows = rows;
    c.requests = requests;
    c.longest = longest;
    c.pages = pages;
    c.heads = p->heads;
    c.kv = p->kv;
    c.group = p->heads / p->kv;
    c.dim = p->dim;
    c.page_len = p->page_len;
    c.max_block = (int)p->max_block;
    c.page8 = (uint32_t)p->page_len / 8;
    // p8 < 2^17 + 8 and page8 <= 2^13: (2^32 + page8 - 1) / page8 divides exactly
    c.page8_magic = (uint32_t)(((1ull << 32) + c.page8 - 1) / c.page8);
    c.row_bytes = (uint32_t)p->dim * 2;
    c.page_bytes = (uint32_t)p->kv * (uint32_t)p->page_len * c.row_bytes;
    c.scale8 = llmx::qk_scale_q1616(p->dim) >> 8;
    c.capacity = p->capacity;
    c.meta = p->meta;
    c.score = p->score;
    c.top = p->top;
    c.tv = p->tv;
    c.fsum = p->fsum;
    c.exps = p->exps;
    c.error = p->error;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int all = (int)((longest + kTile - 1) / kTile), most = (c.max_block * c.group + 7) / 8;
    const Clusters how = choose(p, requests, all, most);
    if (how.ctas) {
        c.cluster_log = how.log;
        c.tiles = how.tiles;
        c.blocks = how.blocks;
        const cudaError_t e = launch(attend_kernel(p->dim, how.blocks == 1), (unsigned)how.ctas, kThreads, (size_t)how.smem, c, s, 1 << how.log,
                                     (unsigned)((most + how.blocks - 1) / how.blocks));
        return e == cudaSuccess ? LLMX_OK : cuda_fail("attention", e);
    }
    const uint64_t items = (uint64_t)requests * p->kv * ((longest + kTile - 1) / kTile);
    auto grid = [&](int ctas) { return (unsigned)std::min<uint64_t>(items, (uint64_t)ctas); };
    cudaError_t e = launch(scores_kernel(p->dim, p->one), grid(p->scores_ctas), kThreads, p->scores_smem, c, s);
    if (e == cudaSuccess) e = launch(values_kernel(p->one), grid(p->values_ctas), kThreads, p->values_smem, c, s);
    if (e == cudaSuccess) {
        const int tiles = (int)((longest + kTile - 1) / kTile);
        // few columns: a warp per kAhead tiles, for latency; many: no more warps than fill the SMs
        const uint64_t columns = (uint64_t)rows * p->heads;
        const int warps = (int)std::max<uint64_t>(1, std::min<uint64_t>({kMaxJoinWarps, (uint64_t)(tiles + kAhead - 1) / kAhead, (uint64_t)p->sms * 32 / columns}));
        const bool far = tiles > kShortTiles;
        const size_t smem = (size_t)(warps - 1) * kMaxStretches * 32 * sizeof(Stretch);
        e = launch(far ? (const void *)k_join<true> : (const void *)k_join<false>, rows * (unsigned)p->heads, 32 * warps, smem, c, s);
    }
    return e == cudaSuccess ? LLMX_OK : cuda_fail("attention", e);
}

extern "C" int llmx_selftest_paged_way(llmx_paged *p, int way, uint32_t requests, uint32_t longest, int *taken) {
    if (!p || !taken) return fail(LLMX_ERR_ARG, "null pointer");
    if (way < -1 || way > way_of(3, 16)) return fail(LLMX_ERR_ARG, "way must be -1..64, got " + std::to_string(way));
    if (requests == 0 || requests > p->max_requests || longest == 0 || longest > p->max_length)
        return fail(LLMX_ERR_ARG, "sizes that the handle is not for");
    p->way = way;
    const Clusters how = choose(p, requests, (int)((longest + kTile - 1) / kTile), ((int)p->max_block * (p->heads / p->kv) + 7) / 8);
    *taken = how.ctas ? way_of(how.log, how.blocks) : 0;
    return LLMX_OK;
}

extern "C" int llmx_paged_error(llmx_paged *p, void *stream) {
    if (!p) return fail(LLMX_ERR_ARG, "null handle");
    DeviceScope scope(p->dev);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int word = 0;
    cudaError_t e = cudaMemcpyAsync(&word, p->error, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && word) {
        e = cudaMemsetAsync(p->error, 0, 4, s);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    }
    if (e != cudaSuccess) return cuda_fail("error", e);
    if (!word) return LLMX_OK;
    std::string what;
    if (word & kErrRequest) what += " a request's offsets, length or position";
    if (word & kErrPage) what += std::string(what.empty() ? "" : ",") + " a page number";
    if (word & kErrBudget) what += std::string(what.empty() ? "" : ",") + " more positions than the handle has room for";
    return fail(LLMX_ERR_RANGE, "out of range:" + what);
}

extern "C" uint64_t llmx_paged_device_bytes(const llmx_paged *p) { return p ? p->bytes : 0; }
