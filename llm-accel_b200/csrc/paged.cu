// A key-value cache in pages, for many requests: their rows appended with the
// rotation on the way, and attention of a block of rows per request over it.
//
// The arithmetic is that of the one-sequence path (attention.cu): tile-exact
// Q2.14 online softmax, reference golden_tiled_flash_attention_q2_14_impl
// host/host_qwen_8x64.cpp:3610-3739, rotation rotate_fix16_pair_with_quantized_rope
// host:4765-4788.  The reference has one sequence with one contiguous cache.
//
// Attention is three launches over the requests' 64-position tiles.
//   k_scores  QK: scores (int16) and each tile's maximum;
//   k_values  the running maximum is the prefix maximum of the tiles' maxima, so a
//             tile's probabilities and its values tv (int16) need nothing else of the
//             tiles before it;
//   k_join    replays the recurrence of (sum, acc), which rounds at every tile, in
//             order, and divides.
// So the cache's length is split over as many CTAs as there are tiles, and nothing
// waits for anything but a launch.
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
#include <cstdint>
#include <new>
#include <string>
#include <type_traits>

#include "llmx.h"
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
    Meta *meta;          // [requests]
    int16_t *score;      // [slot][8 columns][64 positions]
    int16_t *top;        // [slot][8] maxima
    int16_t *tv;         // [slot][8][dim]
    int2 *fsum;          // [slot][8]: P(m_before - m), the sum of P
    const int16_t *exps; // [2049]
    int *error;
};

// ---- small pieces -------------------------------------------------------------------
static __device__ __forceinline__ uint32_t div_page(const Call &c, uint32_t p8) {
    return c.page8 == 1 ? p8 : __umulhi(p8, c.page8_magic);
}
// First row of positions 8 inside .. of key head h in the page that entry `at` of a table names.
static __device__ __forceinline__ const char *page_rows(const Call &c, const int16_t *cache, const int32_t *table, uint32_t at, uint32_t inside, int h) {
    uint32_t page = (uint32_t)table[at];
    if (page >= c.pages) {
        atomicOr(c.error, kErrPage);
        page = 0;
    }
    return reinterpret_cast<const char *>(cache) + (unsigned long long)page * c.page_bytes + ((uint32_t)h * c.page_len + inside * 8) * c.row_bytes;
}
// First row of positions 8 p8 .. 8 p8 + 7 (page lengths are multiples of 8).
static __device__ __forceinline__ const char *rows_at(const Call &c, const int16_t *cache, const int32_t *table, uint32_t p8, int h) {
    const uint32_t at = div_page(c, p8);
    return page_rows(c, cache, table, at, p8 - at * c.page8, h);
}
// (not .nc: the launch before may still be writing the cache when this one starts)
static __device__ __forceinline__ uint4 ld16(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
static __device__ __forceinline__ uint32_t min16x2(uint32_t a, uint32_t b) { return __vmins2(a, b); }
static __device__ __forceinline__ uint32_t max16x2(uint32_t a, uint32_t b) { return __vmaxs2(a, b); }
static __device__ __forceinline__ uint32_t limit2(uint32_t v) { return max16x2(min16x2(v, 0x08000800u), 0xf800f800u); }
// Of four high bytes of limited values: 1 where the byte is 8 (the value 2048).
static __device__ __forceinline__ uint32_t at_limit(uint32_t h) { return (h >> 3) & ~(h >> 4) & 0x01010101u; }
// (8 - x) >> 4 of two 16-bit values, as 16 bits each
static __device__ __forceinline__ uint32_t rest2(uint32_t x) {
    const int a = (8 - llmx::lo16(x)) >> 4, b = (8 - llmx::hi16(x)) >> 4;
    return ((uint32_t)a & 0xffffu) | ((uint32_t)b << 16);
}
static __device__ __forceinline__ uint32_t low4(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x6420); }
static __device__ __forceinline__ uint32_t high4(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7531); }

// D += A B, A 16 x 32 and B 32 x 8 bytes; S and U: signed and unsigned.
#define LLMX_MMA(name, ta, tb)                                                                                           \
    static __device__ __forceinline__ void name(int(&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, \
                                                uint32_t b1) {                                                           \
        asm("mma.sync.aligned.m16n8k32.row.col.s32." ta "." tb ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" \
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])                                                             \
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));                                                     \
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
// A score with its four saturating banks.
static __device__ __noinline__ int score_exact(const int16_t *q, const int16_t *k, int dim, int scale8) {
    long long bank[4] = {0, 0, 0, 0};
    for (int e = 0; e < dim; e++) bank[e & 3] += llmx::qk_prod(q[e], llmx::q412(k[e]));
    long long t = 0;
    for (int i = 0; i < 4; i++) t += sat32(bank[i]);
    return score_of(sat32(t), scale8);
}

// The requests' first slots and items, into shared memory (and by CTA 0 into the
// workspace); returns the number of items, 0 when the call needs more than the handle has.
static __device__ int plan(const Call &c, Meta *meta) {
    __shared__ long long part[2][kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long slots = 0, items = 0;  // of the requests before this round's
    for (uint32_t first = 0; first < c.requests; first += kThreads) {
        const uint32_t b = first + threadIdx.x;
        Meta m{0, 0, 0, -1};
        long long s = 0, i = 0;
        if (b < c.requests) {
            const uint32_t o0 = c.offsets[b], o1 = c.offsets[b + 1], length = c.lengths[b];
            if (o0 <= o1 && o1 <= c.rows && o1 - o0 <= (uint32_t)c.max_block && length <= c.longest) {
                m.rows = (int)(o1 - o0);
                m.tiles = m.rows ? (int)((length + kTile - 1) / kTile) : 0;
                i = (long long)c.kv * m.tiles;
                s = i * ((m.rows * c.group + 7) / 8);
            } else if (blockIdx.x == 0) {
                atomicOr(c.error, kErrRequest);
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
    __syncthreads();
    if (!fits)
        for (uint32_t b = threadIdx.x; b < c.requests; b += kThreads) meta[b] = Meta{0, 0, 0, -1};
    if (blockIdx.x == 0) {
        if (!fits && threadIdx.x == 0) atomicOr(c.error, kErrBudget);
        for (uint32_t b = threadIdx.x; b < c.requests; b += kThreads) c.meta[b] = meta[b];
    }
    __syncthreads();
    return fits ? (int)items : 0;
}

// One (request, key head, tile) after another.
struct Cursor {
    int b, h, t;  // request, key head, tile
    int tiles, rows, length, blocks;
    int slot0;    // of tile 0 in the first column block of this key head
    const int32_t *table;

    __device__ void enter(const Call &c, const Meta *meta, int request, int head) {
        b = request;
        h = head;
        const Meta m = meta[b];
        tiles = m.tiles;
        rows = m.rows;
        length = (int)c.lengths[b];
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
};

static __device__ __forceinline__ void range_of(int items, int &first, int &end) {
    const int each = (int)(((long long)items + gridDim.x - 1) / gridDim.x);
    first = (int)min((long long)blockIdx.x * each, (long long)items);
    end = min(first + each, items);
}

// ---- scores -------------------------------------------------------------------------
// What k_scores keeps of a column (a query row) of the (request, key head) at hand.
struct __align__(16) Column {
    int seen;  // positions that it sees
    int bias;  // 2048 times its sum
    int wide;  // a bank may saturate
    int pad;
};

// A warp scores 16 positions against 8 columns (query rows) at a time: the positions are
// the rows of A, and a lane's 16-byte load of a key row's 8 dimensions is, split into
// bytes, its share of A for both byte planes; no shared memory is passed through.  The
// queries' shares of B, with those of (8 - q) >> 4, wait in shared memory.  Keys are limited by two
// instructions a pair: min(k, 2048), then max(k + 2048, 0), so both planes are
// unsigned and 2048 times the sum of q is taken off again.
template <int KS>  // steps of 32 dimensions
__global__ void __launch_bounds__(kThreads, 5) k_scores(const Call c) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ int tops[2][kWarps][kMaxColumns];
    __shared__ Column column[kMaxColumns];
    const int most = (c.max_block * c.group + 7) / 8;  // column blocks
    uint4 *queries = reinterpret_cast<uint4 *>(dynamic);  // [most][KS][32 lanes] {low, low, high, high}
    uint4 *rests = queries + most * KS * 32;              // the same of (8 - q) >> 4
    Meta *meta = reinterpret_cast<Meta *>(rests + most * KS * 32);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    pdl_wait();
    pdl_trigger();
    const int items = plan(c, meta);
    int first, end;
    range_of(items, first, end);
    if (first >= end) return;

    Cursor cur;
    cur.start(c, meta, first);
    uint4 raw[2][KS];  // key rows g and g + 8 of the warp's 16 positions
    auto load = [&](const Cursor &u) {
        const int p0 = u.t * kTile + warp * 16;
        if (p0 + 16 <= u.length && c.dim == 32 * KS) {
            const uint32_t p8 = (uint32_t)p0 >> 3, at = div_page(c, p8), inside = p8 - at * c.page8;
            const char *row = page_rows(c, c.k, u.table, at, inside, u.h) + g * (64 * KS) + 16 * t4;
#pragma unroll
            for (int s = 0; s < KS; s++) raw[0][s] = ld16(row + 64 * s);
            // 8 positions on: in the same page, or at the next one's start
            row = inside + 1 < c.page8 ? row + 8 * 64 * KS : page_rows(c, c.k, u.table, at + 1, 0, u.h) + g * (64 * KS) + 16 * t4;
#pragma unroll
            for (int s = 0; s < KS; s++) raw[1][s] = ld16(row + 64 * s);
            return;
        }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int p = p0 + 8 * r;
            const char *row = p < u.length ? rows_at(c, c.k, u.table, (uint32_t)p >> 3, u.h) + g * c.row_bytes + 16 * t4 : nullptr;
#pragma unroll
            for (int s = 0; s < KS; s++)
                raw[r][s] = p + g < u.length && 32 * s + 8 * t4 < c.dim ? ld16(row + 64 * s) : make_uint4(0, 0, 0, 0);
        }
    };
    load(cur);
    bool moved = true;
    for (int item = first; item < end; item++) {
        const Cursor now = cur;
        if (moved) {
            __syncthreads();  // the last key head's columns are done with
            const int columns = now.rows * c.group;
            const uint32_t row0 = c.offsets[now.b];
            for (int nb = warp; nb < now.blocks; nb += kWarps) {
                const int col = nb * 8 + g, j = col / c.group;
                const int16_t *q = c.q + (size_t)(row0 + j) * c.ld_q + (size_t)(now.h * c.group + col - j * c.group) * c.dim + 8 * t4;
                uint32_t big = 0;
                int sum = 0;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    const uint4 w = col < columns && 32 * s + 8 * t4 < c.dim ? *reinterpret_cast<const uint4 *>(q + 32 * s) : make_uint4(0, 0, 0, 0);
                    // above 8192: the top three of 16 bits differ
                    big |= (w.x ^ (w.x << 1)) | (w.x ^ (w.x << 2)) | (w.y ^ (w.y << 1)) | (w.y ^ (w.y << 2)) | (w.z ^ (w.z << 1)) |
                           (w.z ^ (w.z << 2)) | (w.w ^ (w.w << 1)) | (w.w ^ (w.w << 2));
                    // (a total reaches 2^31 only where every q is -8192, the first one too)
                    if (s == 0 && t4 == 0 && (w.x & 0xffffu) == 0xe000u) big |= 0x8000u;
                    sum += llmx::lo16(w.x) + llmx::hi16(w.x) + llmx::lo16(w.y) + llmx::hi16(w.y) + llmx::lo16(w.z) + llmx::hi16(w.z) +
                           llmx::lo16(w.w) + llmx::hi16(w.w);
                    queries[(nb * KS + s) * 32 + lane] = make_uint4(low4(w.x, w.y), low4(w.z, w.w), high4(w.x, w.y), high4(w.z, w.w));
                    const uint4 r = make_uint4(rest2(w.x), rest2(w.y), rest2(w.z), rest2(w.w));
                    rests[(nb * KS + s) * 32 + lane] = make_uint4(low4(r.x, r.y), low4(r.z, r.w), high4(r.x, r.y), high4(r.z, r.w));
                }
                big |= __shfl_xor_sync(0xffffffffu, big, 1);
                big |= __shfl_xor_sync(0xffffffffu, big, 2);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (t4 == 0) column[col] = Column{col < columns ? now.length - now.rows + 1 + j : 0, 2048 * sum, (int)(big & 0x80008000u), 0};
            }
            __syncthreads();
        }
        const int p0 = now.t * kTile + warp * 16;
        // byte planes of the keys, from 0 to 4096
        uint32_t kh[KS][4], kl[KS][4], limit = 0;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                auto shift = [](uint32_t w) { return __viaddmax_s16x2(min16x2(w, 0x08000800u), 0x08000800u, 0u); };
                const uint4 w = make_uint4(shift(raw[r][s].x), shift(raw[r][s].y), shift(raw[r][s].z), shift(raw[r][s].w));
                kl[s][r] = low4(w.x, w.y);
                kl[s][r + 2] = low4(w.z, w.w);
                kh[s][r] = high4(w.x, w.y);
                kh[s][r + 2] = high4(w.z, w.w);
                limit |= kh[s][r] | kh[s][r + 2];
            }
        // some high byte is 16: the value 4096, at the upper limit
        const bool some = __any_sync(0xffffffffu, (limit & 0x10101010u) != 0);
        // the next item's keys are on their way while this one's are used
        if (item + 1 < end) {
            moved = cur.next(c, meta);
            load(cur);
        }
        int(&top_of)[kMaxColumns] = tops[item & 1][warp];
        if (p0 >= now.length)
            for (int col = lane; col < now.blocks * 8; col += 32) top_of[col] = -32768;
        const bool whole = p0 + 16 <= now.length - now.rows + 1;  // every column sees all 16 positions
        for (int nb = 0; p0 < now.length && nb < now.blocks; nb++) {
            int hh[4] = {0, 0, 0, 0}, mid[4] = {0, 0, 0, 0}, ll[4] = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const uint4 q = queries[(nb * KS + s) * 32 + lane];
                mma_us(hh, kh[s][0], kh[s][1], kh[s][2], kh[s][3], q.z, q.w);
                mma_uu(mid, kh[s][0], kh[s][1], kh[s][2], kh[s][3], q.x, q.y);
                mma_uu(ll, kl[s][0], kl[s][1], kl[s][2], kl[s][3], q.x, q.y);
                mma_us(mid, kl[s][0], kl[s][1], kl[s][2], kl[s][3], q.z, q.w);
            }
            if (some) {
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    const uint4 r = rests[(nb * KS + s) * 32 + lane];
                    uint32_t m[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) m[i] = kh[s][i] >> 4 & 0x01010101u;
                    mma_us(mid, m[0], m[1], m[2], m[3], r.z, r.w);
                    mma_uu(ll, m[0], m[1], m[2], m[3], r.x, r.y);
                }
            }
            const Column ca = column[nb * 8 + 2 * t4], cb = column[nb * 8 + 2 * t4 + 1];
            int sc[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                sc[i] = score_of((int)(((uint32_t)hh[i] << 16) + ((uint32_t)mid[i] << 8) + (uint32_t)ll[i] - (uint32_t)(i & 1 ? cb.bias : ca.bias)),
                                 c.scale8);
            if (__any_sync(0xffffffffu, (ca.wide | cb.wide) != 0)) {
#pragma unroll 1
                for (int i = 0; i < 4; i++) {
                    const int col = nb * 8 + 2 * t4 + (i & 1), p = p0 + g + (i >> 1) * 8;
                    if (!column[col].wide || p >= now.length) continue;
                    const int j = col / c.group;
                    const int16_t *q = c.q + (size_t)(c.offsets[now.b] + j) * c.ld_q + (size_t)(now.h * c.group + col - j * c.group) * c.dim;
                    const int y = score_exact(q, reinterpret_cast<const int16_t *>(rows_at(c, c.k, now.table, (uint32_t)p >> 3, now.h) + (p & 7) * c.row_bytes), c.dim, c.scale8);
                    if (i == 0) sc[0] = y;
                    else if (i == 1) sc[1] = y;
                    else if (i == 2) sc[2] = y;
                    else sc[3] = y;
                }
            }
            // column g, positions 2 t4, 2 t4 + 1 (and + 8) after the transposition
            const uint32_t w0 = transpose8(pack_sat16(sc[0], sc[1])), w1 = transpose8(pack_sat16(sc[2], sc[3]));
            uint32_t *dst = reinterpret_cast<uint32_t *>(c.score + ((size_t)now.slot(nb) * 8 + g) * kTile + warp * 16 + 2 * t4);
            dst[0] = w0;
            dst[4] = w1;
            uint32_t top = max16x2(w0, w1);
            if (!whole) {
                const int seen = column[nb * 8 + g].seen - (p0 + 2 * t4);
                auto masked = [](uint32_t w, int n) { return n >= 2 ? w : n == 1 ? (w & 0xffffu) | 0x80000000u : 0x80008000u; };
                top = max16x2(masked(w0, seen), masked(w1, seen - 8));
            }
            top = max16x2(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max16x2(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (t4 == 0) top_of[nb * 8 + g] = max(llmx::lo16(top), llmx::hi16(top));
        }
        __syncthreads();
        // (the other buffer is in use until every thread is here again)
        for (int col = threadIdx.x; col < now.blocks * 8; col += kThreads) {
            int top = tops[item & 1][0][col];
#pragma unroll
            for (int w = 1; w < kWarps; w++) top = max(top, tops[item & 1][w][col]);
            c.top[(size_t)now.slot(col >> 3) * 8 + (col & 7)] = (int16_t)top;
        }
    }
}

// ---- values -------------------------------------------------------------------------
constexpr int kExpWords = 1028;  // 2049 entries of 16 bits, rounded up to 16 bytes
constexpr int kRowBytes = 256;   // of a value row in shared memory
constexpr int kValueBytes = kTile * kRowBytes;

// A stage of k_values' ring: a tile's value rows, then per column block the scores (1 KB) and maxima
// (16 bytes).
static __host__ __device__ int stage_bytes(int blocks) { return kValueBytes + blocks * (8 * kTile * 2 + 16); }
constexpr int kStages = 2;

static __device__ __forceinline__ void copy16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
static __device__ __forceinline__ void copy16(void *dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(there ? 16 : 0)
                 : "memory");
}

// A warp forms 32 of a tile's elements: the elements are the rows of A, so that a lane needs
// the bytes of four positions in a word, a 4 x 4 transposition of bytes in its
// registers.  Value rows come through shared memory, whole lines at a time: 16 bytes go to
// unit u ^ 2 (row / 8 mod 4) of their row, so that the four rows that a quarter of a warp
// reads lie in different banks.  A tile's probabilities are formed once, by all
// warps, and pass through shared memory in the order of B.
__global__ void __launch_bounds__(kThreads, 5) k_values(const Call c) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const int most = (c.max_block * c.group + 7) / 8;  // column blocks
    constexpr int stages = kStages;
    const int stage_size = stage_bytes(most);
    unsigned char *ring = dynamic;
    uint4 *prob = reinterpret_cast<uint4 *>(ring + stages * stage_size);  // [most][2 steps][32 lanes] {low, low, high, high}
    uint32_t *exps_w = reinterpret_cast<uint32_t *>(prob + most * 64);
    const int16_t *exps = reinterpret_cast<const int16_t *>(exps_w) + 2048;  // of differences <= 0
    int *seen = reinterpret_cast<int *>(exps_w + kExpWords);  // [most * 8] positions that a column sees
    int *psum = seen + most * 8;                              // [4][most * 8] sums of P over 16 positions
    int *factor = psum + 4 * most * 8;                        // [most * 8]
    int *before = factor + most * 8 + warp * most * 8;        // [most * 8] the warp's own running maxima
    Meta *meta = reinterpret_cast<Meta *>(factor + (1 + kWarps) * most * 8);
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

    // the elements are shared out over `parts` warps; with fewer than four, the others take other column blocks
    const int parts = (c.dim + 31) >> 5, turns = 4 / parts, part = warp % parts, turn = warp / parts;
    const int e0 = part * 32 + g * 4;  // this lane's elements: e0 .. e0 + 3
    const bool mine = e0 < c.dim;

    auto fetch = [&](const Cursor &u, int stage) {
        unsigned char *dst = ring + stage * stage_size;
        const int unit = threadIdx.x & 15, r8 = threadIdx.x >> 4;
        const int left = u.length - u.t * kTile;
        if (unit * 8 < c.dim) {
            const uint32_t p8 = (uint32_t)u.t * 8;
            uint32_t at = div_page(c, p8), inside = p8 - at * c.page8;
            unsigned char *to = dst + r8 * kRowBytes;
            const char *rows = nullptr;
            const uint32_t mine = r8 * c.row_bytes + unit * 16;
            if (left >= kTile && inside + 8 <= c.page8) {  // whole, in one page
                rows = page_rows(c, c.v, u.table, at, inside, u.h) + mine;
#pragma unroll
                for (int j = 0; j < 8; j++) copy16(to + 8 * j * kRowBytes + (unit ^ (2 * (j & 3))) * 16, rows + j * 8 * c.row_bytes);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (8 * j < left && (j == 0 || inside == c.page8)) {  // the next page
                        if (j) {
                            at++;
                            inside = 0;
                        }
                        rows = page_rows(c, c.v, u.table, at, inside, u.h) + mine;
                    }
                    const bool there = 8 * j + r8 < left;
                    copy16(to + 8 * j * kRowBytes + (unit ^ (2 * (j & 3))) * 16, there ? (const void *)rows : (const void *)c.v, there);
                    rows += 8 * c.row_bytes;
                    inside++;
                }
            }
        }
        unsigned char *score = dst + kValueBytes, *top = score + most * (8 * kTile * 2);
        for (int i = threadIdx.x; i < u.blocks * 64; i += kThreads) {  // (columns' rows of 8 units, turned by 2 (column mod 4))
            const int col = i >> 3 & 7, w = i & 7;
            copy16(score + (i - w + (w ^ (2 * (col & 3)))) * 16, c.score + ((size_t)u.slot(i >> 6) * 64 + (i & 63)) * 8);
        }
        if (threadIdx.x < u.blocks) copy16(top + threadIdx.x * 16, c.top + (size_t)u.slot(threadIdx.x) * 8);
    };
    Cursor cur, ahead;
    cur.start(c, meta, first);
    ahead = cur;
    int fetched = first;
    for (int i = 0; i < stages - 1; i++) {
        if (fetched < end) {
            if (fetched > first) ahead.next(c, meta);
            fetch(ahead, i);
            fetched++;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int stage = 0;
    bool moved = true;
    for (int item = first; item < end; item++) {
        const int blocks = cur.blocks;
        if (moved) {
            // the maxima of the tiles before, by every warp for itself
            for (int nb = 0; nb < blocks; nb++) {
                const uint4 *tops = reinterpret_cast<const uint4 *>(c.top) + cur.slot(nb) - cur.t;
                uint4 m = make_uint4(0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u);
                for (int i = lane; i < cur.t; i += 32) {
                    const uint4 w = tops[i];
                    m = make_uint4(max16x2(m.x, w.x), max16x2(m.y, w.y), max16x2(m.z, w.z), max16x2(m.w, w.w));
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    m.x = max16x2(m.x, __shfl_xor_sync(0xffffffffu, m.x, o));
                    m.y = max16x2(m.y, __shfl_xor_sync(0xffffffffu, m.y, o));
                    m.z = max16x2(m.z, __shfl_xor_sync(0xffffffffu, m.z, o));
                    m.w = max16x2(m.w, __shfl_xor_sync(0xffffffffu, m.w, o));
                }
                const uint32_t w = g < 4 ? (g < 2 ? m.x : m.y) : (g < 6 ? m.z : m.w);
                if (t4 == 0) before[nb * 8 + g] = g & 1 ? llmx::hi16(w) : llmx::lo16(w);
            }
            __syncthreads();  // (the last key head's columns are done with)
            for (int col = threadIdx.x; col < blocks * 8; col += kThreads)
                seen[col] = col < cur.rows * c.group ? cur.length - cur.rows + 1 + col / c.group : 0;
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(stages - 2) : "memory");
        __syncthreads();
        unsigned char *here = ring + stage * stage_size;
        if (fetched < end) {  // into the stage of the item before, which is free
            ahead.next(c, meta);
            fetch(ahead, stage == 0 ? stages - 1 : stage - 1);
            fetched++;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        // probabilities: 16 positions a warp, lane: column g, 4 positions
        for (int nb = 0; nb < blocks; nb++) {
            const int col = nb * 8 + g, was = before[col];
            const int16_t *top = reinterpret_cast<const int16_t *>(here + kValueBytes + most * (8 * kTile * 2)) + col;
            const int m = max(was, (int)*top);
            const uint2 w = *reinterpret_cast<const uint2 *>(here + kValueBytes + (col * 8 + ((2 * warp + (t4 >> 1)) ^ (2 * (g & 3)))) * 16 + (t4 & 1) * 8);
            const int left = seen[col] - (cur.t * kTile + warp * 16 + 4 * t4);
            const int s[4] = {llmx::lo16(w.x), llmx::hi16(w.x), llmx::lo16(w.y), llmx::hi16(w.y)};
            int p[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // (what lies behind the last position that is seen may hold anything)
                p[i] = i < left ? exps[min(max(s[i] - m, -2048), 0)] : 0;
                sum += p[i];
            }
            const uint32_t w0 = (uint32_t)p[0] | (uint32_t)p[1] << 16, w1 = (uint32_t)p[2] | (uint32_t)p[3] << 16;
            uint32_t *dst = reinterpret_cast<uint32_t *>(prob + nb * 64 + (warp >> 1) * 32 + g * 4 + 2 * (warp & 1) + (t4 >> 1)) + (t4 & 1);
            dst[0] = low4(w0, w1);
            dst[2] = high4(w0, w1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (t4 == 0) {
                psum[warp * most * 8 + col] = sum;
                before[col] = m;
                if (warp == 0) factor[col] = exps[max(was - m, -2048)];
            }
        }
        __syncthreads();
        for (int col = threadIdx.x; col < blocks * 8; col += kThreads) {
            const int *ps = psum + col;
            c.fsum[(size_t)cur.slot(col >> 3) * 8 + (col & 7)] = make_int2(factor[col], ps[0] + ps[most * 8] + ps[2 * most * 8] + ps[3 * most * 8]);
        }
        if (turn < turns && turn < blocks) {
            // byte planes of the values: [step][element pair][row or row + 8, positions 0-3 or 4-7]
            uint32_t vh[2][2][4], vl[2][2][4];
            unsigned char *v = here + 8 * t4 * kRowBytes + ((part * 4 + (g >> 1)) ^ (2 * t4)) * 16 + (g & 1) * 8;
            bool limit = false;
#pragma unroll 1
            for (;;) {
                uint32_t out = 0;
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        uint2 w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const uint2 *>(v + (32 * s + 4 * half + i) * kRowBytes);
#pragma unroll
                        for (int mb = 0; mb < 2; mb++) {
                            const uint32_t w0 = mb ? w[0].y : w[0].x, w1 = mb ? w[1].y : w[1].x, w2 = mb ? w[2].y : w[2].x, w3 = mb ? w[3].y : w[3].x;
                            const uint32_t a = __byte_perm(w0, w1, 0x5140), b = __byte_perm(w2, w3, 0x5140);
                            const uint32_t d = __byte_perm(w0, w1, 0x7362), e = __byte_perm(w2, w3, 0x7362);
                            vl[s][mb][2 * half] = __byte_perm(a, b, 0x5410);
                            vh[s][mb][2 * half] = __byte_perm(a, b, 0x7632);
                            vl[s][mb][2 * half + 1] = __byte_perm(d, e, 0x5410);
                            vh[s][mb][2 * half + 1] = __byte_perm(d, e, 0x7632);
                            out |= (vh[s][mb][2 * half] ^ (vh[s][mb][2 * half] << 1)) | (vh[s][mb][2 * half + 1] ^ (vh[s][mb][2 * half + 1] << 1));
                        }
                    }
                // some high byte is not in [-8, 7] (its bits 3 to 7 differ): limited where they lie, and once more
                if (limit || !__any_sync(0xffffffffu, mine && (out & 0xf0f0f0f0u) != 0)) break;
                limit = true;
#pragma unroll 1
                for (int i = 0; i < 16; i++) {
                    uint2 *w = reinterpret_cast<uint2 *>(v + ((i & 8) * 4 + (i & 7)) * kRowBytes);
                    *w = make_uint2(limit2(w->x), limit2(w->y));
                }
            }
            for (int nb = turn; nb < blocks; nb += turns) {
                const uint4 b0 = prob[nb * 64 + lane], b1 = prob[nb * 64 + 32 + lane];
                uint32_t tv[2][2];  // [column 2 t4 + j][elements e0, e0 + 1 and e0 + 2, e0 + 3]
#pragma unroll
                for (int mb = 0; mb < 2; mb++) {
                    int hh[4] = {0, 0, 0, 0}, mid[4] = {0, 0, 0, 0}, ll[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const uint4 b = s ? b1 : b0;
                        const uint32_t(&h)[4] = vh[s][mb], (&l)[4] = vl[s][mb];
                        mma_su(hh, h[0], h[1], h[2], h[3], b.z, b.w);
                        mma_su(mid, h[0], h[1], h[2], h[3], b.x, b.y);
                        mma_uu(ll, l[0], l[1], l[2], l[3], b.x, b.y);
                        mma_uu(mid, l[0], l[1], l[2], l[3], b.z, b.w);
                        if (limit) {
                            const uint32_t r0 = rest2(__byte_perm(b.x, b.z, 0x5140)), r1 = rest2(__byte_perm(b.x, b.z, 0x7362));
                            const uint32_t r2 = rest2(__byte_perm(b.y, b.w, 0x5140)), r3 = rest2(__byte_perm(b.y, b.w, 0x7362));
                            uint32_t m[4];
#pragma unroll
                            for (int i = 0; i < 4; i++) m[i] = at_limit(h[i]);
                            mma_us(mid, m[0], m[1], m[2], m[3], high4(r0, r1), high4(r2, r3));
                            mma_uu(ll, m[0], m[1], m[2], m[3], low4(r0, r1), low4(r2, r3));
                        }
                    }
                    int y[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int ts = (int)(((uint32_t)hh[i] << 16) + ((uint32_t)mid[i] << 8) + (uint32_t)ll[i]);
                        y[i] = ((ts >> 5) + 257) >> 9;  // rnd8 of rnd6: (ts + 2^5 + 2^13) / 2^14, within 32 bits
                    }
                    tv[0][mb] = pack_sat16(y[0], y[2]);
                    tv[1][mb] = pack_sat16(y[1], y[3]);
                }
                if (mine) {
                    int16_t *dst = c.tv + ((size_t)cur.slot(nb) * 8 + 2 * t4) * c.dim + e0;
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(tv[0][0], tv[0][1]);
                    *reinterpret_cast<uint2 *>(dst + c.dim) = make_uint2(tv[1][0], tv[1][1]);
                }
            }
        }
        stage = stage + 1 == stages ? 0 : stage + 1;
        moved = item + 1 < end && cur.next(c, meta);
    }
}

// ---- join ---------------------------------------------------------------------------
// The request of row r: the last one whose rows start at or before it.  By a whole warp;
// at most 1024 requests in two steps.
static __device__ __forceinline__ uint32_t request_of(const uint32_t *offsets, uint32_t requests, uint32_t r) {
    const uint32_t lane = threadIdx.x & 31, step = (requests + 31) / 32;
    uint32_t at = lane * step;
    uint32_t before = __ballot_sync(0xffffffffu, at < requests && offsets[at] <= r);
    const uint32_t block = before ? (31 - __clz(before)) * step : 0;
    if (step == 1) return block;
    at = block + lane;
    before = __ballot_sync(0xffffffffu, lane < step && at < requests && offsets[at] <= r);
    return before ? block + 31 - __clz(before) : block;
}

// What a stretch of tiles makes of a value x that comes in: x + s, limited to [lo, hi] (sums that
// saturate at every step combine to that).  Without kLong no sum can reach the limits.
template <bool kLong>
struct Stretch;
template <>
struct Stretch<false> {
    int s;
    __device__ void start() { s = 0; }
    __device__ void add(int v) { s += v; }
    __device__ int of(int x) const { return x + s; }
};
template <>
struct Stretch<true> {
    long long s;
    int lo, hi;
    __device__ void start() {
        s = 0;
        lo = INT_MIN;
        hi = INT_MAX;
    }
    __device__ void add(int v) {
        s += v;
        lo = llmx::add_sat(lo, v);
        hi = llmx::add_sat(hi, v);
    }
    __device__ int of(int x) const { return (int)min(max(x + s, (long long)lo), (long long)hi); }
};

constexpr int kShortTiles = 255;  // tiles whose sums stay below 2^31: of values 2^23 each, of probabilities 2^22
constexpr int kMaxStretches = 3;  // per warp
constexpr int kAhead = 8;         // tiles loaded at once
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

// One query head's row per CTA.  A lane has four elements, a warp an equal part of the tiles.  Between
// tiles that raise the maximum (whose factor is not 1: few in a long text) the recurrence only adds,
// so a warp gives what its tiles do to any value that comes in as a few stretches (a factor, then a
// sum), and the first warp, which starts from 0, puts them together; tiles beyond a warp's
// kMaxStretches it goes through itself.
template <bool kLong>
__global__ void __launch_bounds__(32 * kMaxJoinWarps) k_join(const Call c) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    struct Four {
        Stretch<kLong> e[4];
    };
    __shared__ Stretch<kLong> norms[kMaxJoinWarps][kMaxStretches];
    __shared__ int factors[kMaxJoinWarps][kMaxStretches], counts[kMaxJoinWarps], rest[kMaxJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
    const int quads = c.dim >> 2;
    Four *stretches = reinterpret_cast<Four *>(dynamic);  // [warps - 1][kMaxStretches][quads]
    pdl_wait();
    pdl_trigger();
    const uint32_t row = blockIdx.x / c.heads;
    const int head = (int)(blockIdx.x - row * c.heads);
    const uint32_t b = request_of(c.offsets, c.requests, row);
    const uint32_t begin = c.offsets[b], behind = c.offsets[b + 1];
    const Meta m = c.meta[b];
    if (row < begin || row >= behind || m.rows < 0) return;  // of no request, or of a void one
    const int h = head / c.group, col = (int)(row - begin) * c.group + head - h * c.group;
    const int blocks = (m.rows * c.group + 7) / 8;
    const size_t at = ((size_t)m.slot + (size_t)(h * blocks + (col >> 3)) * m.tiles) * 8 + (col & 7);
    const uint2 *tv = reinterpret_cast<const uint2 *>(c.tv + at * c.dim) + min(lane, quads - 1);
    const int2 *fsum = c.fsum + at;
    const int step = 8 * quads;  // from a tile to the next
    const int first = (int)((long long)m.tiles * warp / warps), end = (int)((long long)m.tiles * (warp + 1) / warps);

    int sum = 0, x[4] = {0, 0, 0, 0};
    uint2 v[kAhead];
    int2 f[kAhead];
    auto load = [&](int t0, int t1) {  // what lies behind t1 changes nothing
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            v[i] = make_uint2(0, 0);
            f[i] = make_int2(16384, 0);
            if (t0 + i < t1) {
                v[i] = tv[(size_t)(t0 + i) * step];
                f[i] = fsum[(size_t)(t0 + i) * 8];
            }
        }
    };
    // (one of a warp's lanes' factors stands for all of them)
    auto plain = [&]() {
        int all = 16384;
#pragma unroll
        for (int i = 0; i < kAhead; i++) all &= f[i].x;  // at most 16384: a factor below it has no bit 14
        return __any_sync(0xffffffffu, all == 16384) != 0;
    };
    auto add_all = [&](Stretch<kLong> &n, Four &p) {
        if constexpr (kLong) {
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                n.add(4 * f[i].y);
                p.e[0].add(add_low(v[i].x, 0) * 256);
                p.e[1].add(add_high(v[i].x, 0) * 256);
                p.e[2].add(add_low(v[i].y, 0) * 256);
                p.e[3].add(add_high(v[i].y, 0) * 256);
            }
        } else {
            int s = 0, y[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                s += f[i].y;
                y[0] = add_low(v[i].x, y[0]);
                y[1] = add_high(v[i].x, y[1]);
                y[2] = add_low(v[i].y, y[2]);
                y[3] = add_high(v[i].y, y[3]);
            }
            n.add(4 * s);
#pragma unroll
            for (int k = 0; k < 4; k++) p.e[k].add(256 * y[k]);
        }
    };
    auto add_one = [&](Stretch<kLong> &n, Four &p, uint2 w, int s) {
        n.add(4 * s);
        p.e[0].add(llmx::lo16(w.x) * 256);
        p.e[1].add(llmx::hi16(w.x) * 256);
        p.e[2].add(llmx::lo16(w.y) * 256);
        p.e[3].add(llmx::hi16(w.y) * 256);
    };
    auto factor = [&](int by) {  // a factor of 1 leaves everything as it is
        if (by == 16384) return;
        sum = times(sum, by);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = times(x[k], by);
    };
    auto apply = [&](const Stretch<kLong> &n, const Four &p) {
        sum = n.of(sum);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = p.e[k].of(x[k]);
    };
    auto clear = [&](Stretch<kLong> &n, Four &p) {
        n.start();
#pragma unroll
        for (int k = 0; k < 4; k++) p.e[k].start();
    };
    // tiles t0 .. t1 - 1 on top of (sum, x)
    auto replay = [&](int t0, int t1) {
        for (; t0 < t1; t0 += kAhead) {
            load(t0, t1);
            Stretch<kLong> n;
            Four p;
            clear(n, p);
            if (plain()) {
                add_all(n, p);
                apply(n, p);
                continue;
            }
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                factor(f[i].x);
                clear(n, p);
                add_one(n, p, v[i], f[i].y);
                apply(n, p);
            }
        }
    };
    if (warp == 0) {
        replay(first, end);
    } else {
        Stretch<kLong> n;
        Four p;
        clear(n, p);
        int f0 = 16384, count = 0, left = end;
        Four *mine = stretches + (size_t)(warp - 1) * kMaxStretches * quads + lane;
        auto close = [&]() {
            if (lane < quads) mine[count * quads] = p;
            if (lane == 0) {
                norms[warp][count] = n;
                factors[warp][count] = f0;
            }
            count++;
        };
        for (int t0 = first; t0 < end && left == end; t0 += kAhead) {
            load(t0, end);
            if (plain()) {
                add_all(n, p);
                continue;
            }
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                if (left != end) continue;
                if (f[i].x != 16384) {
                    if (t0 + i > first) {  // the stretch ends here
                        if (count + 1 == kMaxStretches) {
                            left = t0 + i;
                            continue;
                        }
                        close();
                        clear(n, p);
                    }
                    f0 = f[i].x;
                }
                add_one(n, p, v[i], f[i].y);
            }
        }
        if (first < end) close();
        if (lane == 0) {
            counts[warp] = count;
            rest[warp] = left;
        }
    }
    if (warps > 1) {
        __syncthreads();
        if (warp != 0) return;
        for (int w = 1; w < warps; w++) {
            for (int k = 0; k < counts[w]; k++) {
                factor(factors[w][k]);
                apply(norms[w][k], stretches[((size_t)(w - 1) * kMaxStretches + k) * quads + min(lane, quads - 1)]);
            }
            replay(rest[w], (int)((long long)m.tiles * (w + 1) / warps));
        }
    }
    if (lane >= quads) return;
    const long long inv = sat16(rnd((long long)llmx::recip_q16(sum < 16 ? 16 : sum), 8));
    auto last = [&](int y) { return (int)(((long long)y * inv + 32768) >> 16); };
    *reinterpret_cast<uint2 *>(c.out + (size_t)row * c.ld_out + (size_t)head * c.dim + 4 * lane) =
        make_uint2(pack_sat16(last(x[0]), last(x[1])), pack_sat16(last(x[2]), last(x[3])));
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
    int *error;
};

static __device__ __forceinline__ void turn2(uint32_t x0, uint32_t x1, uint32_t c, uint32_t s, uint32_t &y0, uint32_t &y1) {
    // products of 16-bit values, their sums in 64 bits: a table may hold any value
    auto one = [](long long a, int ca, long long b, int cb) { return sat16(rnd(a * ca + b * cb, 8)); };
    const int c0 = llmx::lo16(c), c1 = llmx::hi16(c), s0 = llmx::lo16(s), s1 = llmx::hi16(s);
    const int a0 = llmx::lo16(x0), a1 = llmx::hi16(x0), b0 = llmx::lo16(x1), b1 = llmx::hi16(x1);
    y0 = (uint32_t)(one(a0, c0, b0, -s0) & 0xffff) | (uint32_t)one(a1, c1, b1, -s1) << 16;
    y1 = (uint32_t)(one(b0, c0, a0, s0) & 0xffff) | (uint32_t)one(b1, c1, a1, s1) << 16;
}

// A CTA per row; a thread turns 8 pairs (i, i + dim/2) of a head, or copies 16 values.
__global__ void __launch_bounds__(256) k_append(const AppendCall c) {
    pdl_wait();
    pdl_trigger();
    const uint32_t r = blockIdx.x;
    const uint32_t b = request_of(c.offsets, c.requests, r);
    const uint32_t first = c.offsets[b], last = c.offsets[b + 1];
    if (r < first || r >= last) return;  // of no request
    const long long position = (long long)c.lengths[b] - (long long)(last - first) + (r - first);
    if (position < 0) return;  // in front of the sequence
    const long long at = position / c.page_len;
    if (position >= c.positions || at >= (long long)c.ld_table) {
        if (threadIdx.x == 0) atomicOr(c.error, kErrRequest);
        return;
    }
    const uint32_t page = (uint32_t)c.table[(size_t)b * c.ld_table + at];
    if (page >= c.pages) {
        if (threadIdx.x == 0) atomicOr(c.error, kErrPage);
        return;
    }
    const size_t inside = (size_t)(position - at * c.page_len);
    const int parts = c.dim >> 4, half = c.dim >> 1;  // 16 values each
    const int16_t *turn = c.rope + (size_t)position * c.dim;
    for (int i = threadIdx.x; i < (c.heads + 2 * c.kv) * parts; i += blockDim.x) {
        const int head = i / parts, part = i - head * parts;
        const int16_t *src = c.qkv + (size_t)r * c.ld_qkv + (size_t)head * c.dim;
        if (head < c.heads + c.kv) {
            const uint4 x0 = *reinterpret_cast<const uint4 *>(src + 8 * part), x1 = *reinterpret_cast<const uint4 *>(src + half + 8 * part);
            const uint4 cs = *reinterpret_cast<const uint4 *>(turn + 8 * part), sn = *reinterpret_cast<const uint4 *>(turn + half + 8 * part);
            uint4 y0, y1;
            turn2(x0.x, x1.x, cs.x, sn.x, y0.x, y1.x);
            turn2(x0.y, x1.y, cs.y, sn.y, y0.y, y1.y);
            turn2(x0.z, x1.z, cs.z, sn.z, y0.z, y1.z);
            turn2(x0.w, x1.w, cs.w, sn.w, y0.w, y1.w);
            int16_t *dst = head < c.heads ? c.q + (size_t)r * c.ld_q + (size_t)head * c.dim
                                          : c.k + (((size_t)page * c.kv + (head - c.heads)) * c.page_len + inside) * c.dim;
            *reinterpret_cast<uint4 *>(dst + 8 * part) = y0;
            *reinterpret_cast<uint4 *>(dst + half + 8 * part) = y1;
        } else {
            const uint4 *from = reinterpret_cast<const uint4 *>(src) + 2 * part;
            uint4 *to = reinterpret_cast<uint4 *>(c.v + (((size_t)page * c.kv + (head - c.heads - c.kv)) * c.page_len + inside) * c.dim) + 2 * part;
            const uint4 a = from[0], d = from[1];
            to[0] = a;
            to[1] = d;
        }
    }
}

}  // namespace

struct llmx_paged {
    int dev = 0, sms = 0;
    int heads = 0, kv = 0, dim = 0, page_len = 0;
    uint32_t max_requests = 0, max_block = 0, max_length = 0;
    long long capacity = 0;  // (key head, tile) items of a call
    size_t scores_smem = 0, values_smem = 0;
    int scores_ctas = 0, values_ctas = 0;  // that are on the device at once
    unsigned char *memory = nullptr;
    Meta *meta = nullptr;
    int16_t *score = nullptr, *top = nullptr, *tv = nullptr, *exps = nullptr;
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

const void *scores_kernel(int dim) {
    switch ((dim + 31) / 32) {
        case 1: return (const void *)k_scores<1>;
        case 2: return (const void *)k_scores<2>;
        case 3: return (const void *)k_scores<3>;
        default: return (const void *)k_scores<4>;
    }
}

template <class T>
cudaError_t launch(const void *fn, unsigned grid, int threads, size_t smem, const T &call, cudaStream_t s) {
    T copy = call;
    void *args[] = {&copy};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
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
    p->capacity = (long long)(tiles * kv_heads);
    size_t at = 0;
    auto place = [&](size_t n) {
        const size_t was = at;
        at += (n + 255) / 256 * 256;
        return was;
    };
    const size_t error_at = place(4), exps_at = place(kExpWords * 4), meta_at = place(max_requests * sizeof(Meta)),
                 score_at = place(slots * 8 * kTile * 2), top_at = place(slots * 16), tv_at = place(slots * 8 * head_dim * 2),
                 fsum_at = place(slots * 64);
    p->bytes = at;
    p->scores_smem = 2 * blocks * ((head_dim + 31) / 32) * 512 + (size_t)max_requests * sizeof(Meta);
    p->values_smem = (size_t)kStages * stage_bytes((int)blocks) + blocks * 1024 + kExpWords * 4 +
                     (6 + kWarps) * blocks * 32 + (size_t)max_requests * sizeof(Meta);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int16_t e16[2049], host[kExpWords * 2] = {};
    llmx::build_exp_tables(e16, host);
    cudaError_t e;
    if ((e = cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, device)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(scores_kernel(p->dim), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaFuncSetAttribute((const void *)k_values, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaFuncSetAttribute((const void *)k_join<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) != cudaSuccess ||
        (e = cudaMalloc(reinterpret_cast<void **>(&p->memory), at)) != cudaSuccess ||
        (e = cudaMemsetAsync(p->memory + error_at, 0, 4, s)) != cudaSuccess ||
        (e = cudaMemcpyAsync(p->memory + exps_at, host, sizeof(host), cudaMemcpyHostToDevice, s)) != cudaSuccess ||
        (e = cudaStreamSynchronize(s)) != cudaSuccess) {
        release(p);
        return cuda_fail("create", e);
    }
    int per_sm[2] = {0, 0};
    if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm[0], scores_kernel(p->dim), kThreads, p->scores_smem)) != cudaSuccess ||
        (e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm[1], (const void *)k_values, kThreads, p->values_smem)) != cudaSuccess) {
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
    const uint64_t items = (uint64_t)requests * p->kv * ((longest + kTile - 1) / kTile);
    auto grid = [&](int ctas) { return (unsigned)std::min<uint64_t>(items, (uint64_t)ctas); };
    cudaError_t e = launch(scores_kernel(p->dim), grid(p->scores_ctas), kThreads, p->scores_smem, c, s);
    if (e == cudaSuccess) e = launch((const void *)k_values, grid(p->values_ctas), kThreads, p->values_smem, c, s);
    if (e == cudaSuccess) {
        const int tiles = (int)((longest + kTile - 1) / kTile);
        // few columns: a warp per kAhead tiles, for latency; many: no more warps than fill the SMs
        const uint64_t columns = (uint64_t)rows * p->heads;
        const int warps = (int)std::max<uint64_t>(1, std::min<uint64_t>({kMaxJoinWarps, (uint64_t)(tiles + kAhead - 1) / kAhead, (uint64_t)p->sms * 32 / columns}));
        const bool far = tiles > kShortTiles;
        const size_t smem = (size_t)(warps - 1) * kMaxStretches * p->dim * (far ? sizeof(Stretch<true>) : sizeof(Stretch<false>));
        e = launch(far ? (const void *)k_join<true> : (const void *)k_join<false>, rows * (unsigned)p->heads, 32 * warps, smem, c, s);
    }
    return e == cudaSuccess ? LLMX_OK : cuda_fail("attention", e);
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
