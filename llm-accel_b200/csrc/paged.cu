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
    int scale8;                   // fm(1/sqrt(dim)), Q8.8
    long long capacity;           // (key head, tile) items
    // workspace
    Meta *meta;          // [requests]
    int16_t *score;      // [slot][8 columns][64 positions]
    int16_t *top;        // [slot][8] maxima
    int16_t *tv;         // [slot][8][dim]
    int32_t *psum;       // [slot][4 blocks of 16 positions][8] sums of P
    int32_t *factor;     // [slot][8] P(m_before - m)
    const int16_t *exps; // [2049]
    int *error;
};

// ---- small pieces -------------------------------------------------------------------
static __device__ __forceinline__ uint32_t div_page(const Call &c, uint32_t p8) {
    return c.page8 == 1 ? p8 : __umulhi(p8, c.page8_magic);
}
// First row of 8 positions 8 p8 .. 8 p8 + 7 of key head h (page lengths are multiples of 8).
static __device__ __forceinline__ const int16_t *rows_at(const Call &c, const int16_t *cache, const int32_t *table, uint32_t p8, int h) {
    const uint32_t at = div_page(c, p8);
    uint32_t page = (uint32_t)table[at];
    if (page >= c.pages) {
        atomicOr(c.error, kErrPage);
        page = 0;
    }
    return cache + (((size_t)page * c.kv + h) * c.page_len + (size_t)(p8 - at * c.page8) * 8) * c.dim;
}
// (not .nc: the launch before may still be writing the cache when this one starts)
static __device__ __forceinline__ uint4 ld16(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
static __device__ __forceinline__ uint2 ld8(const void *p) {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
    return v;
}
static __device__ __forceinline__ uint32_t min16x2(uint32_t a, uint32_t b) { return __vmins2(a, b); }
static __device__ __forceinline__ uint32_t max16x2(uint32_t a, uint32_t b) { return __vmaxs2(a, b); }
static __device__ __forceinline__ uint32_t limit2(uint32_t v) { return max16x2(min16x2(v, 0x08000800u), 0xf800f800u); }
// Of four high bytes: 0xff.. where one is not in [-8, 7] (bits 3 to 7 differ).
static __device__ __forceinline__ uint32_t beyond(uint32_t h) { return (h ^ (h << 1)) & 0xf0f0f0f0u; }
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
LLMX_MMA(mma_ss, "s8", "s8")
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

static __device__ __forceinline__ int score_of(int total, int scale8) {
    const int v = (int)(((long long)total * scale8 + 128) >> 8);
    return sat16((v + 128) >> 8);
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
    int b, h, t;      // request, key head, tile
    Meta m;
    int length;
    const int32_t *table;

    __device__ void enter(const Call &c, const Meta *meta, int request) {
        b = request;
        m = meta[b];
        length = (int)c.lengths[b];
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
        enter(c, meta, lo);
        h = (item - m.item) / m.tiles;
        t = item - m.item - h * m.tiles;
    }
    // The next item, which there is.  Returns whether it is of another request or key head.
    __device__ bool next(const Call &c, const Meta *meta) {
        if (++t < m.tiles) return false;
        t = 0;
        if (++h == c.kv) {
            h = 0;
            int r = b + 1;
            while (meta[r].tiles == 0) r++;
            enter(c, meta, r);
        }
        return true;
    }
    __device__ int columns(const Call &c) const { return m.rows * c.group; }
    // Slot of this tile in column block nb.
    __device__ size_t slot(const Call &c, int nb) const {
        const int blocks = (columns(c) + 7) / 8;
        return (size_t)m.slot + (size_t)(h * blocks + nb) * m.tiles + t;
    }
    // Positions that column col sees.
    __device__ int seen(const Call &c, int col) const { return length - m.rows + 1 + col / c.group; }
};

static __device__ __forceinline__ void range_of(int items, int &first, int &end) {
    const int each = (int)(((long long)items + gridDim.x - 1) / gridDim.x);
    first = (int)min((long long)blockIdx.x * each, (long long)items);
    end = min(first + each, items);
}

// ---- scores -------------------------------------------------------------------------
// A warp scores 16 positions against 8 columns (query rows) at a time: the positions are
// the rows of A, and a lane's 16-byte load of a key row's 8 dimensions is, split into
// bytes, its share of A for both byte planes; no shared memory is passed through.
template <int KS>  // steps of 32 dimensions
__global__ void __launch_bounds__(kThreads, 4) k_scores(const Call c) {
    extern __shared__ Meta meta[];
    __shared__ int tops[2][kMaxColumns];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    for (int i = threadIdx.x; i < 2 * (int)kMaxColumns; i += kThreads) tops[i / kMaxColumns][i % kMaxColumns] = -32768;
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
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int p = p0 + 8 * r;
            const bool any = p < u.length;
            const int16_t *row = any ? rows_at(c, c.k, u.table, (uint32_t)p >> 3, u.h) + (size_t)g * c.dim : nullptr;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const int e = 32 * s + 8 * t4;
                raw[r][s] = p + g < u.length && e < c.dim ? ld16(row + e) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    load(cur);
    uint32_t qh[KS][2], ql[KS][2];  // this lane's share of B: column g
    bool held = false;              // the registers hold the only column block of (b, h)
    uint32_t wide = 0;
    for (int item = first; item < end; item++) {
        const int buf = item & 1;
        const int p0 = cur.t * kTile + warp * 16;
        const bool live = p0 < cur.length;
        // byte planes of the keys
        uint32_t kh[KS][4], kl[KS][4];
        uint32_t out = 0;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                kl[s][r] = low4(raw[r][s].x, raw[r][s].y);
                kl[s][r + 2] = low4(raw[r][s].z, raw[r][s].w);
                kh[s][r] = high4(raw[r][s].x, raw[r][s].y);
                kh[s][r + 2] = high4(raw[r][s].z, raw[r][s].w);
                out |= beyond(kh[s][r]) | beyond(kh[s][r + 2]);
            }
        const bool limit = __any_sync(0xffffffffu, out != 0);
        if (limit) {
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const uint4 w = make_uint4(limit2(raw[r][s].x), limit2(raw[r][s].y), limit2(raw[r][s].z), limit2(raw[r][s].w));
                    kl[s][r] = low4(w.x, w.y);
                    kl[s][r + 2] = low4(w.z, w.w);
                    kh[s][r] = high4(w.x, w.y);
                    kh[s][r + 2] = high4(w.z, w.w);
                }
        }
        // the next item's keys are on their way while this one's are used
        Cursor now = cur;
        const bool more = item + 1 < end;
        bool moved = false;
        if (more) {
            moved = cur.next(c, meta);
            load(cur);
        }
        const int columns = now.columns(c), blocks = (columns + 7) / 8;
        for (int nb = 0; live && nb < blocks; nb++) {
            const int col = nb * 8 + g;
            const int head = now.h * c.group + col % c.group;
            const int16_t *qrow = c.q + (size_t)(c.offsets[now.b] + col / c.group) * c.ld_q + (size_t)head * c.dim;
            if (!held) {
                uint32_t most = 0;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    const int e = 32 * s + 8 * t4;
                    const uint4 w = col < columns && e < c.dim ? *reinterpret_cast<const uint4 *>(qrow + e) : make_uint4(0, 0, 0, 0);
                    ql[s][0] = low4(w.x, w.y);
                    ql[s][1] = low4(w.z, w.w);
                    qh[s][0] = high4(w.x, w.y);
                    qh[s][1] = high4(w.z, w.w);
                    // |q| above 8192: the top three bits of a high byte differ
                    most |= (qh[s][0] ^ (qh[s][0] << 1)) | (qh[s][1] ^ (qh[s][1] << 1)) | (qh[s][0] ^ (qh[s][0] << 2)) | (qh[s][1] ^ (qh[s][1] << 2));
                }
                // (the sum reaches 2^31 only where every q is -8192, the first one too)
                const bool lowest = t4 == 0 && (qh[0][0] & 0xffu) == 0xe0u && (ql[0][0] & 0xffu) == 0;
                wide = __ballot_sync(0xffffffffu, (most & 0x80808080u) != 0 || lowest);
            }
            held = blocks == 1;
            int hh[4] = {0, 0, 0, 0}, mid[4] = {0, 0, 0, 0}, ll[4] = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                mma_ss(hh, kh[s][0], kh[s][1], kh[s][2], kh[s][3], qh[s][0], qh[s][1]);
                mma_su(mid, kh[s][0], kh[s][1], kh[s][2], kh[s][3], ql[s][0], ql[s][1]);
                mma_uu(ll, kl[s][0], kl[s][1], kl[s][2], kl[s][3], ql[s][0], ql[s][1]);
                mma_us(mid, kl[s][0], kl[s][1], kl[s][2], kl[s][3], qh[s][0], qh[s][1]);
            }
            if (limit) {
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    uint32_t m[4], r[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) m[i] = at_limit(kh[s][i]);
#pragma unroll
                    for (int i = 0; i < 2; i++) {  // (8 - q) >> 4, from the bytes of q
                        r[2 * i] = rest2(__byte_perm(ql[s][i], qh[s][i], 0x5140));
                        r[2 * i + 1] = rest2(__byte_perm(ql[s][i], qh[s][i], 0x7362));
                    }
                    mma_us(mid, m[0], m[1], m[2], m[3], high4(r[0], r[1]), high4(r[2], r[3]));
                    mma_uu(ll, m[0], m[1], m[2], m[3], low4(r[0], r[1]), low4(r[2], r[3]));
                }
            }
            int sc[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                sc[i] = score_of((int)(((uint32_t)hh[i] << 16) + ((uint32_t)mid[i] << 8) + (uint32_t)ll[i]), c.scale8);
            if (wide) {
#pragma unroll 1
                for (int i = 0; i < 4; i++) {
                    const int col1 = 2 * t4 + (i & 1), p = p0 + g + (i >> 1) * 8;
                    if ((wide >> (4 * col1) & 15u) == 0 || p >= now.length || nb * 8 + col1 >= columns) continue;
                    const int cc = nb * 8 + col1;
                    const int16_t *q1 = c.q + (size_t)(c.offsets[now.b] + cc / c.group) * c.ld_q + (size_t)(now.h * c.group + cc % c.group) * c.dim;
                    sc[i] = score_exact(q1, rows_at(c, c.k, now.table, (uint32_t)p >> 3, now.h) + (size_t)(p & 7) * c.dim, c.dim, c.scale8);
                }
            }
            // column g, positions 2 t4, 2 t4 + 1 (and + 8) after the transposition
            const uint32_t w0 = transpose8((uint32_t)(sc[0] & 0xffff) | ((uint32_t)sc[1] << 16));
            const uint32_t w1 = transpose8((uint32_t)(sc[2] & 0xffff) | ((uint32_t)sc[3] << 16));
            const size_t slot = now.slot(c, nb);
            uint32_t *dst = reinterpret_cast<uint32_t *>(c.score + (slot * 8 + g) * kTile + warp * 16 + 2 * t4);
            dst[0] = w0;
            dst[4] = w1;
            const int seen = now.seen(c, col) - (p0 + 2 * t4);
            int top = -32768;
            if (seen > 0) top = llmx::lo16(w0);
            if (seen > 1) top = max(top, llmx::hi16(w0));
            if (seen > 8) top = max(top, llmx::lo16(w1));
            if (seen > 9) top = max(top, llmx::hi16(w1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (t4 == 0) atomicMax(&tops[buf][col], top);
        }
        if (moved) held = false;
        __syncthreads();
        // (the other buffer is in use until every thread is here again)
        for (int col = threadIdx.x; col < blocks * 8; col += kThreads) {
            c.top[now.slot(c, col >> 3) * 8 + (col & 7)] = (int16_t)tops[buf][col];
            tops[buf][col] = -32768;
        }
    }
}

// ---- values -------------------------------------------------------------------------
constexpr int kExpWords = 1028;  // 2049 entries of 16 bits, rounded up to 16 bytes

// A warp forms 32 of a tile's elements: the elements are the rows of A, so that a lane needs
// the bytes of four positions in a word, a 4 x 4 transposition of bytes in its
// registers.  A tile's probabilities are formed once, by all warps, and pass
// through shared memory in the order of B.
__global__ void __launch_bounds__(kThreads, 4) k_values(const Call c) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const int warps = blockDim.x >> 5;
    const int most = (c.max_block * c.group + 7) / 8;  // column blocks
    uint32_t *exps_w = reinterpret_cast<uint32_t *>(dynamic);
    const int16_t *exps = reinterpret_cast<const int16_t *>(dynamic) + 2048;  // of differences <= 0
    uint4 *prob = reinterpret_cast<uint4 *>(dynamic + kExpWords * 4);         // [2][most][2 steps][32 lanes]
    int *before = reinterpret_cast<int *>(prob + 2 * most * 64) + warp * most * 8;  // this warp's running maxima
    Meta *meta = reinterpret_cast<Meta *>(reinterpret_cast<int *>(prob + 2 * most * 64) + kWarps * most * 8);
    for (int i = threadIdx.x; i < kExpWords; i += blockDim.x) exps_w[i] = reinterpret_cast<const uint32_t *>(c.exps)[i];
    pdl_wait();
    pdl_trigger();
    for (uint32_t b = threadIdx.x; b < c.requests; b += blockDim.x) meta[b] = c.meta[b];
    __syncthreads();
    const Meta last = meta[c.requests - 1];
    // void requests have no items but their place in the order
    const int items = last.item + c.kv * last.tiles;
    int first, end;
    range_of(items, first, end);
    if (first >= end) return;
    const int e0 = warp * 32 + g * 4;  // this lane's elements: e0 .. e0 + 3
    const bool mine = e0 < c.dim;

    Cursor cur;
    cur.start(c, meta, first);
    uint2 raw[2][8];  // positions 32 s + 8 t4 + i, elements e0 .. e0 + 3
    auto load = [&](const Cursor &u) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int p = u.t * kTile + 32 * s + 8 * t4;
            const bool any = p < u.length;
            const int16_t *row = any ? rows_at(c, c.v, u.table, (uint32_t)p >> 3, u.h) + e0 : nullptr;
#pragma unroll
            for (int i = 0; i < 8; i++) raw[s][i] = mine && p + i < u.length ? ld8(row + (size_t)i * c.dim) : make_uint2(0, 0);
        }
    };
    load(cur);
    bool moved = true;
    for (int item = first; item < end; item++) {
        const int columns = cur.columns(c), blocks = (columns + 7) / 8;
        uint4 *pb = prob + (item & 1) * most * 64;
        if (moved) {  // the maxima of the tiles before
            for (int nb = 0; nb < blocks; nb++) {
                const uint4 *tops = reinterpret_cast<const uint4 *>(c.top + (cur.slot(c, nb) - cur.t) * 8);
                uint4 m = make_uint4(0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u);
                for (int i = lane; i < cur.t; i += 32) {
                    const uint4 w = tops[i];
                    m.x = max16x2(m.x, w.x);
                    m.y = max16x2(m.y, w.y);
                    m.z = max16x2(m.z, w.z);
                    m.w = max16x2(m.w, w.w);
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
            __syncwarp();
        }
        // probabilities: 16 positions a warp at a time, lane: column g, 4 positions
        for (int nb = 0; nb < blocks; nb++) {
            const size_t slot = cur.slot(c, nb);
            const int col = nb * 8 + g;
            const int was = before[col];
            const int m = max(was, (int)c.top[slot * 8 + g]);
            for (int blk = warp; blk < 4; blk += warps) {
                const uint2 w = *reinterpret_cast<const uint2 *>(c.score + (slot * 8 + g) * kTile + blk * 16 + 4 * t4);
                const int seen = col < columns ? cur.seen(c, col) - (cur.t * kTile + blk * 16 + 4 * t4) : 0;
                const int s[4] = {llmx::lo16(w.x), llmx::hi16(w.x), llmx::lo16(w.y), llmx::hi16(w.y)};
                int p[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // (what lies behind the last position that is seen may hold anything)
                    p[i] = i < seen ? exps[min(max(s[i] - m, -2048), 0)] : 0;
                    sum += p[i];
                }
                const uint32_t w0 = (uint32_t)p[0] | (uint32_t)p[1] << 16, w1 = (uint32_t)p[2] | (uint32_t)p[3] << 16;
                uint32_t *dst = reinterpret_cast<uint32_t *>(pb + nb * 64 + (blk >> 1) * 32 + g * 4 + 2 * (blk & 1) + (t4 >> 1));
                dst[t4 & 1] = low4(w0, w1);
                dst[2 + (t4 & 1)] = high4(w0, w1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (t4 == 0) {
                    c.psum[(slot * 4 + blk) * 8 + g] = sum;
                    if (blk == 0) c.factor[slot * 8 + g] = exps[max(was - m, -2048)];
                }
            }
            __syncwarp();
            if (t4 == 0) before[col] = m;
            __syncwarp();
        }
        // byte planes of the values: [step][element pair][row or row + 8, positions 0-3 or 4-7]
        uint32_t vh[2][2][4], vl[2][2][4];
        uint32_t out = 0;
        auto planes = [&]() {
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int mb = 0; mb < 2; mb++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) w[i] = mb ? raw[s][4 * half + i].y : raw[s][4 * half + i].x;
                        const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
                        const uint32_t d = __byte_perm(w[0], w[1], 0x7362), e = __byte_perm(w[2], w[3], 0x7362);
                        vl[s][mb][2 * half] = __byte_perm(a, b, 0x5410);
                        vh[s][mb][2 * half] = __byte_perm(a, b, 0x7632);
                        vl[s][mb][2 * half + 1] = __byte_perm(d, e, 0x5410);
                        vh[s][mb][2 * half + 1] = __byte_perm(d, e, 0x7632);
                        out |= beyond(vh[s][mb][2 * half]) | beyond(vh[s][mb][2 * half + 1]);
                    }
        };
        planes();
        const bool limit = __any_sync(0xffffffffu, out != 0);
        if (limit) {
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) raw[s][i] = make_uint2(limit2(raw[s][i].x), limit2(raw[s][i].y));
            planes();
        }
        const Cursor now = cur;
        if (item + 1 < end) {
            moved = cur.next(c, meta);
            load(cur);
        }
        __syncthreads();
        for (int nb = 0; nb < blocks; nb++) {
            const uint4 b0 = pb[nb * 64 + lane], b1 = pb[nb * 64 + 32 + lane];  // {low, low, high, high}
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
                    const int r6 = ((ts >> 5) + 1) >> 1;  // rnd6, in 32 bits
                    y[i] = sat16((r6 + 128) >> 8);
                }
                tv[0][mb] = (uint32_t)(y[0] & 0xffff) | (uint32_t)y[2] << 16;
                tv[1][mb] = (uint32_t)(y[1] & 0xffff) | (uint32_t)y[3] << 16;
            }
            if (mine) {
                int16_t *dst = c.tv + (now.slot(c, nb) * 8 + 2 * t4) * c.dim + e0;
                *reinterpret_cast<uint2 *>(dst) = make_uint2(tv[0][0], tv[0][1]);
                *reinterpret_cast<uint2 *>(dst + c.dim) = make_uint2(tv[1][0], tv[1][1]);
            }
        }
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

// A thread carries two elements of one query head's row through its tiles in order.
__global__ void __launch_bounds__(kThreads) k_join(const Call c) {
    const int pairs = c.dim >> 1;  // threads of a head
    pdl_wait();
    pdl_trigger();
    const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
    const long long unit = id / pairs;  // (row, head)
    const uint32_t row = (uint32_t)min(unit / c.heads, (long long)c.rows - 1);
    // a warp may hold threads of two rows (pairs need not divide 32)
    const uint32_t row0 = __shfl_sync(0xffffffffu, row, 0), row1 = __shfl_sync(0xffffffffu, row, 31);
    uint32_t b = request_of(c.offsets, c.requests, row0);
    if (row1 != row0)
        for (uint32_t r = row0 + 1; r <= row1; r++) {
            const uint32_t n = request_of(c.offsets, c.requests, r);
            if (row == r) b = n;
        }
    if (unit / c.heads >= c.rows) return;
    const uint32_t first = c.offsets[b], last = c.offsets[b + 1];
    const Meta m = c.meta[b];
    if (row < first || row >= last || m.rows < 0) return;  // of no request, or of a void one
    const int head = (int)(unit % c.heads), e = 2 * (int)(id % pairs);
    const int h = head / c.group, col = (int)(row - first) * c.group + head % c.group;
    const int blocks = (m.rows * c.group + 7) / 8;
    const size_t slot = (size_t)m.slot + (size_t)(h * blocks + (col >> 3)) * m.tiles;
    const int lane8 = col & 7;
    const int16_t *tv = c.tv + (slot * 8 + lane8) * c.dim + e;
    const int32_t *psum = c.psum + slot * 32 + lane8, *factor = c.factor + slot * 8 + lane8;
    int sum = 0, a0 = 0, a1 = 0;
    constexpr int kAhead = 8;
    for (int t0 = 0; t0 < m.tiles; t0 += kAhead) {
        uint32_t v[kAhead];
        int f[kAhead], s[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int t = min(t0 + i, m.tiles - 1);
            v[i] = *reinterpret_cast<const uint32_t *>(tv + (size_t)t * 8 * c.dim);
            f[i] = factor[(size_t)t * 8];
            const int32_t *p = psum + (size_t)t * 32;
            s[i] = p[0] + p[8] + p[16] + p[24];
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (t0 + i >= m.tiles) break;
            if (f[i] != 16384) {  // a factor of 1 leaves everything as it is
                const long long o = (long long)f[i] * 4;  // Q2.14 -> Q16.16
                sum = (int)rnd((long long)sum * o, 16);   // o < 2^16: no saturation
                a0 = (int)rnd((long long)a0 * o, 16);
                a1 = (int)rnd((long long)a1 * o, 16);
            }
            sum = llmx::add_sat(sum, 4 * s[i]);
            a0 = llmx::add_sat(a0, llmx::lo16(v[i]) * 256);
            a1 = llmx::add_sat(a1, llmx::hi16(v[i]) * 256);
        }
    }
    const long long inv = sat16(rnd((long long)llmx::recip_q16(sum < 16 ? 16 : sum), 8));
    const int y0 = sat16(rnd((long long)a0 * inv, 16)), y1 = sat16(rnd((long long)a1 * inv, 16));
    *reinterpret_cast<uint32_t *>(c.out + (size_t)row * c.ld_out + (size_t)head * c.dim + e) =
        (uint32_t)(y0 & 0xffff) | (uint32_t)y1 << 16;
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
    size_t values_smem = 0;
    unsigned char *memory = nullptr;
    Meta *meta = nullptr;
    int16_t *score = nullptr, *top = nullptr, *tv = nullptr, *exps = nullptr;
    int32_t *psum = nullptr, *factor = nullptr;
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
                 psum_at = place(slots * 128), factor_at = place(slots * 32);
    p->bytes = at;
    p->values_smem = kExpWords * 4 + blocks * 2 * 64 * 16 + kWarps * blocks * 8 * 4 + (size_t)max_requests * sizeof(Meta);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int16_t e16[2049], host[kExpWords * 2] = {};
    llmx::build_exp_tables(e16, host);
    cudaError_t e;
    if ((e = cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, device)) != cudaSuccess ||
        (e = cudaFuncSetAttribute((const void *)k_values, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024)) != cudaSuccess ||
        (e = cudaMalloc(reinterpret_cast<void **>(&p->memory), at)) != cudaSuccess ||
        (e = cudaMemsetAsync(p->memory + error_at, 0, 4, s)) != cudaSuccess ||
        (e = cudaMemcpyAsync(p->memory + exps_at, host, sizeof(host), cudaMemcpyHostToDevice, s)) != cudaSuccess ||
        (e = cudaStreamSynchronize(s)) != cudaSuccess) {
        release(p);
        return cuda_fail("create", e);
    }
    auto as = [&](auto *&ptr, size_t where) { ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(p->memory + where); };
    as(p->error, error_at);
    as(p->exps, exps_at);
    as(p->meta, meta_at);
    as(p->score, score_at);
    as(p->top, top_at);
    as(p->tv, tv_at);
    as(p->psum, psum_at);
    as(p->factor, factor_at);
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
    c.scale8 = llmx::qk_scale_q1616(p->dim) >> 8;
    c.capacity = p->capacity;
    c.meta = p->meta;
    c.score = p->score;
    c.top = p->top;
    c.tv = p->tv;
    c.psum = p->psum;
    c.factor = p->factor;
    c.exps = p->exps;
    c.error = p->error;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint64_t items = (uint64_t)requests * p->kv * ((longest + kTile - 1) / kTile);
    const unsigned grid = (unsigned)std::min<uint64_t>(items, (uint64_t)p->sms * 4);
    cudaError_t e = launch(scores_kernel(p->dim), grid, kThreads, requests * sizeof(Meta), c, s);
    if (e == cudaSuccess) e = launch((const void *)k_values, grid, (p->dim + 31) / 32 * 32, p->values_smem, c, s);
    if (e == cudaSuccess) {
        const uint64_t threads = (uint64_t)rows * p->heads * (p->dim / 2);
        e = launch((const void *)k_join, (unsigned)((threads + kThreads - 1) / kThreads), kThreads, 0, c, s);
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
