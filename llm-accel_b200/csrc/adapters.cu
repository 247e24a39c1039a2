// A projection shared by many requests, with each row's own low-rank adapter
// beside it.
//
// No counterpart in the LLM-ACCEL tree, which serves one model's weights to one
// sequence.  The projection's arithmetic is that of golden_projection
// (host/host_qwen_8x64.cpp:3105-3142): an exact int16 x int16 sum, rounded once
// at the end; the adapter's product joins that sum before the rounding:
//
//   t[i][j] = sat16(rnd24(scale_a * sum_k down_a[j][k] x[i][k]))
//   y[i][n] = sum_k W[n][k] x[i][k] + sum_j up_a[n][j] t[i][j]
//
// t is kept in the Q8.8 of every activation between two projections of the
// path: with up_a in Q4.12 its product has the scale of W x, so the adapter is a
// longer sum over k and nothing is rounded in between.  Each t is off by up to 2^-9, so
// a result by up to 2^-9 sum |up|, in the root mean square 2^-8 / 12^(1/2) (rank)^(1/2) |up|:
// at rank 16 with up values of 0.05, 2e-4.  That is a twentieth of a Q8.8 result's step, but 15
// of a Q16.16 one's: an adapter's part in logits is good to t's step, not to the format's.  t
// saturates at +-128, and an adapter whose scaled down x stays below 2^-9 adds nothing.
//
// Tensor cores.  Both factors are split into bytes, as in mma_proj.cu: w = 256 wh
// + wl (wl unsigned), x = 256 xh + xs + 128 with xs = (x & 255) - 128, so that
// one tcgen05.mma of kind::i8 per weight plane multiplies it with the operand
// [xh rows | xs rows] (N = two planes of the row tile) and 128 * sum(w) is added per
// output at the end.  Four int32 sums (hh, hs, lh, ls) per result then give the
// exact int64 one: 65536 hh + 256 (hs + lh) + ls.  They cannot overflow for
// in_dim <= 32768 and rank <= 128: |ls| <= 2^15 * 255 * 128 + 128 * 255^2 < 2^31.
// An adapter is a longer k: its up matrix is a further operand of the same
// accumulators, against the t of its own rows and zeros in the other rows of the
// tile.  t is split with an unsigned low byte (its zero rows then are zero in
// both planes), which costs two MMAs of one plane each instead of one of both.
//
// Layouts.  k is cut into pieces of 16 (one 16-byte core-matrix column): a
// weight piece is [high | low][128 outputs][16 bytes] = 4 KiB, a row piece
// [high | low][row tile][16 bytes].  A stage of the ring is 8 pieces (4 for wide row
// tiles) of 128 outputs; an adapter of rank r has ceil(r / 16) pieces per 128
// outputs, so pieces of different adapters fill one 32-deep MMA step together and a
// rank of 16 wastes nothing.  All of it lands in shared memory by 1-D bulk copies.
//
// Two launches per call.  k_prepare splits the rows into pieces and forms t;
// k_project streams the stages of tiles of 128 outputs x up to 128 rows through one
// CTA per SM, and starts under k_prepare (dependent launch): its ring of weight
// stages fills while the rows are still being split.  Row tiles of the same outputs
// are neighbours, so a weight stage comes from HBM once.
//
// What bounds it (B200, in graphs of calls over three sets of weights, which thus come
// from HBM; bytes at 6.47 TB/s, exact products at a quarter of the int8 rate, which a
// loop of such MMAs measured as 4.5 P/s).  Up to about 64 rows the weight stream: LM
// head 151936 x 2048, 40 rows of 8 adapters, 110 to 116 us by machine (119 outside a graph, 0.86
// of the floor of 102; adapters of rank 8 are stored as pieces of 16: 20 MB more); Gate/Up
// 22016 x 2048, 16 rows of 16 adapters, 26.7 us against 16.9 (19.0 without adapters), of which
// 5 pass before k_prepare's t is there and the tail takes 2; 8 rows x 11008 -> 2048 15.3
// against 7.1 (13.6 without adapters): 5 until t, 5 of stages, 2.5 of adding parts up.
// 512 rows x 11008 x 2048 with rank 64: 57 us against 20.8 of products (47 without adapters):
// k_prepare 6, its end to the first product 5, then two whole tiles of 128 rows and a part of
// one: stages 0.72 us per 128 inputs (by calculation shared memory: 48 KB read by the MMAs and 32 KB
// written per 64 inputs, at 128 bytes a cycle; the tensor pipe is active half the time) and
// the results 3.5 a tile.  One row x 2560 x 2048: 9.2 us, the two kernels' latencies (8.0
// without an adapter).
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
#include "cluster.cuh"
#include "gemv_common.cuh"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace {

using namespace llmx;

constexpr uint32_t kMaxIn = 32768, kMaxOut = 1u << 22, kMaxSlots = 65536, kMaxRank = 128, kMaxCallRows = 65536;
constexpr int kOutTile = 128;             // outputs per tile (TMEM lanes) and inputs per item
constexpr int kRowTile = 128;          // most rows per tile: 4 sums x 128 rows = all 512 TMEM columns
constexpr int kPiece = 2 * kOutTile * 16; // bytes of a weight piece: two planes of 128 x 16
constexpr int kProjectSmem = 221 * 1024, kBesideSmem = 190 * 1024;  // alone on an SM, beside a block of k_prepare
// TMEM + products, loads, and warps of results: 8, or 16 for wide row tiles, whose
// accumulators fill the tensor memory, so that the next tile waits for the results
__host__ __device__ constexpr int result_threads(int depth) { return depth == 4 ? 512 : 256; }
__host__ __device__ constexpr int project_threads(int depth) { return 64 + result_threads(depth); }
constexpr int kHeader = 16 * 16 + 32 + 16 + 64 + 16;  // barriers and flags at the start of shared memory, then the row-tile tables
constexpr int kMaxRing = 16;
constexpr int kMoreTiles = 3;          // row tiles beyond the fewest that a call may take
// Measured, in us: a stage of 128 inputs at least and per row of its tile, adding a cut tile
// up and per row, and the later start that it has where there are several row tiles,
// the results per row.  77 rows x 1096 -> 4999: cut in three 23, whole 15.6, whole in
// three row tiles 13.1; 40 rows x 2048 -> 2560: cut in seven 13.6, whole in three row
// tiles 14.9; 100 rows x 2048 -> 2560: whole 20.1, in four row tiles 15.7.
constexpr double kStageUs = 0.5, kStageRowUs = 0.0056, kAddUs = 2.0, kAddRowUs = 0.085, kLateUs = 1.5, kResultRowUs = 0.03;
constexpr int kGroup = 8;              // rows of one adapter that share a pass over its down matrix

// What the kernels need of a handle and a call.
struct Call {
    const int16_t *x;
    size_t ld_x;
    const int32_t *slot;  // NULL: no adapters
    void *out;
    size_t ld_out;
    uint32_t rows;
    int wide;
    int K, P, T, N;       // inputs, pieces of 16 (a multiple of 8), tiles of 128 outputs, outputs
    int D, C;             // pieces per ring stage, stages of a tile's weight
    int NT, RT;           // rows per row tile (a multiple of 16), row tiles
    int slots, Q;         // pieces reserved per adapter
    int max_pieces;       // adapter pieces of one row tile at most
    int span, ksplit;     // k_prepare: rows per block of t, blocks of a cluster that share k
    int steps;            // of 32 inputs
    const uint8_t *weight; // pieces [T][P]
    const int32_t *wsum;   // [T * 128] sums of the weights of an output
    const uint8_t *up;     // pieces [slots][T][Q]
    const uint4 *down;     // [slots][Q][steps][2][32] operands of t's products: see k_pack_down
    const int32_t *rank, *scale;
    uint8_t *xp;           // row pieces [RT][P]
    uint8_t *tp;           // t pieces [RT][NT first rows][Q]
    const uint8_t *zero;   // a piece of zeros
    int2 *list;            // [RT][max_pieces] {slot * Q + piece, first row * Q + piece}
    int32_t *count;        // [RT] pieces
    int64_t *acc;          // [grid][NT][128] sums of tiles cut between CTAs, zero between calls
    int32_t *arrived;      // [grid]
    int *error;
    uint32_t polls;        // of a wait, except for what has to land before a CTA ends
    int ring, buffers;     // ring stages, accumulator sets
    int shared_tiles;      // tiles whose stages are shared by several CTAs
    int sharers;           // CTAs that share them
};

// Results are many and their arithmetic is all that the result warps do, so it is kept
// short: sums by 64-bit multiply-adds, each rounding in the width that holds it.
static __device__ __forceinline__ int64_t mad_wide(int32_t a, int32_t b, int64_t c) {
    int64_t r;
    asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(r) : "r"(a), "r"(b), "l"(c));
    return r;
}
// sat32(rnd4(s - 8)): the 8 of the rounding is in the sum already.
static __device__ __forceinline__ int32_t to_q16(int64_t s) {
    const uint32_t lo = (uint32_t)s;
    const int32_t hi = (int32_t)(s >> 32), v = (int32_t)__funnelshift_r(lo, (uint32_t)hi, 4);
    return (hi >> 4) == (v >> 31) ? v : (hi >> 31) ^ 0x7fffffff;
}
// sat16(rnd8(v)), without the carry out of 32 bits.
static __device__ __forceinline__ int32_t to_q8(int32_t v) {
    v = (v >> 8) + ((v >> 7) & 1);
    return min(max(v, -32768), 32767);
}

static __device__ __forceinline__ int slot_of(const Call &c, uint32_t row) {
    if (!c.slot || row >= c.rows) return -1;
    const int a = c.slot[row];
    return a >= 0 && a < c.slots && c.rank[a] > 0 ? a : -1;
}
static __device__ __forceinline__ int pieces_of(const Call &c, int a) { return a >= 0 ? (c.rank[a] + 15) >> 4 : 0; }

// The rows of tile rt that have slot a, as a bit per row, in every lane of a warp.
struct RowMask {
    uint32_t w[kRowTile / 32];
    __device__ __forceinline__ int first() const {
        for (int k = 0; k < kRowTile / 32; k++)
            if (w[k]) return k * 32 + __ffs((int)w[k]) - 1;
        return -1;
    }
    __device__ __forceinline__ int before(int at) const {  // rows of the mask below row at
        int n = 0;
#pragma unroll
        for (int k = 0; k < kRowTile / 32; k++) {
            const int top = at - k * 32;
            n += __popc(top >= 32 ? w[k] : top > 0 ? w[k] & ((1u << top) - 1) : 0u);
        }
        return n;
    }
};
static __device__ __forceinline__ RowMask rows_of_slot(const Call &c, int rt, int a) {
    const int lane = threadIdx.x & 31;
    int32_t v[kRowTile / 32];
#pragma unroll
    for (int k = 0; k < kRowTile / 32; k++) {
        const uint32_t row = (uint32_t)rt * c.NT + k * 32 + lane;
        v[k] = k * 32 + lane < c.NT && row < c.rows ? c.slot[row] : -1;
    }
    RowMask m;
#pragma unroll
    for (int k = 0; k < kRowTile / 32; k++) m.w[k] = __ballot_sync(~0u, v[k] == a);
    return m;
}

// The adapters of one row tile, by a block of at least 128 threads.  Thread t <
// 128 stands for row t: whether it is the first row of its adapter, and where
// that adapter's pieces start in the tile's list.  total: pieces of the tile.
struct TileSlots {
    int4 slot[kRowTile / 4];
    int32_t warp_sum[4];
};
struct RowSlot {
    int slot, base, total;
    bool first;
};
static __device__ RowSlot tile_slots(const Call &c, int rt, TileSlots &s) {
    const int t = threadIdx.x, lane = t & 31;
    RowSlot r{-1, 0, 0, false};
    int own = 0, scan = 0;
    if (t < kRowTile) {
        r.slot = t < c.NT ? slot_of(c, (uint32_t)rt * c.NT + t) : -1;
        reinterpret_cast<int32_t *>(s.slot)[t] = r.slot;
        own = pieces_of(c, r.slot);
    }
    __syncthreads();
    if (t < kRowTile) {
        bool seen = r.slot < 0;
        for (int u = 0; u < c.NT; u += 4) {
            const int4 v = s.slot[u >> 2];
            seen |= (v.x == r.slot && u < t) | (v.y == r.slot && u + 1 < t) | (v.z == r.slot && u + 2 < t) |
                    (v.w == r.slot && u + 3 < t);
        }
        r.first = !seen;
        if (seen) own = 0;
        scan = own;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) s.warp_sum[t >> 5] = scan;
    }
    __syncthreads();
    if (t < kRowTile) {
        for (int w = 0; w < (t >> 5); w++) r.base += s.warp_sum[w];
        r.base += scan - own;
    }
    r.total = s.warp_sum[0] + s.warp_sum[1] + s.warp_sum[2] + s.warp_sum[3];
    return r;
}

// ---------------------------------------------------------------------------
// rows -> byte planes, t -> byte planes, the lists of adapter pieces
// ---------------------------------------------------------------------------
static __device__ void split_item(const Call &c, int item) {
    const int chunks = c.P >> 3, rt = item / chunks, chunk = item - rt * chunks;
    uint8_t *dst = c.xp + (size_t)item * 8 * c.NT * 32;
    for (int u = threadIdx.x; u < c.NT * 8; u += blockDim.x) {
        const int kc = u / c.NT, r = u - kc * c.NT;
        const uint32_t row = (uint32_t)rt * c.NT + r;
        const int col = chunk * kOutTile + kc * 16;
        uint4 v[2];
#pragma unroll
        for (int h = 0; h < 2; h++)  // K is a multiple of 8: a piece is whole, half or not there
            v[h] = row < c.rows && col + 8 * h < c.K
                       ? *reinterpret_cast<const uint4 *>(c.x + row * c.ld_x + col + 8 * h)
                       : make_uint4(0, 0, 0, 0);
        uint4 hi, lo;
        hi.x = __byte_perm(v[0].x, v[0].y, 0x7531);
        hi.y = __byte_perm(v[0].z, v[0].w, 0x7531);
        hi.z = __byte_perm(v[1].x, v[1].y, 0x7531);
        hi.w = __byte_perm(v[1].z, v[1].w, 0x7531);
        lo.x = __byte_perm(v[0].x, v[0].y, 0x6420) ^ 0x80808080u;
        lo.y = __byte_perm(v[0].z, v[0].w, 0x6420) ^ 0x80808080u;
        lo.z = __byte_perm(v[1].x, v[1].y, 0x6420) ^ 0x80808080u;
        lo.w = __byte_perm(v[1].z, v[1].w, 0x6420) ^ 0x80808080u;
        uint8_t *p = dst + (size_t)kc * c.NT * 32 + r * 16;
        *reinterpret_cast<uint4 *>(p) = hi;
        *reinterpret_cast<uint4 *>(p + c.NT * 16) = lo;
    }
}

constexpr int kPrepareThreads = 256, kMaxSplit = 8, kSplitInputs = 2048;

// d += 16 ranks x 8 rows over 32 inputs; each side's bytes signed or not.
#define LLMX_MMA_BYTES(name, at, bt)                                                                                    \
    static __device__ __forceinline__ void name(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {        \
        asm("mma.sync.aligned.m16n8k32.row.col.s32." at "." bt ".s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "    \
            "{%0, %1, %2, %3};"                                                                                         \
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])                                                            \
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                                            \
    }
LLMX_MMA_BYTES(mma_ss, "s8", "s8")
LLMX_MMA_BYTES(mma_su, "s8", "u8")
LLMX_MMA_BYTES(mma_us, "u8", "s8")
LLMX_MMA_BYTES(mma_uu, "u8", "u8")
#undef LLMX_MMA_BYTES

// Sums over steps [from, to) of 32 inputs of the products of 16 down rows with 8 rows:
// v[0..3] are those of down rows lane / 4 (v[0], v[1]) and lane / 4 + 8 with rows
// 2 (lane % 4) and the next.  x: row lane / 4.  A lane takes 8 inputs of each, whatever
// places they have among the 32: both sides of a product agree.  int32 holds every
// sum: 2 * 2^16 * 4128 inputs.
static __device__ __forceinline__ void down_products(const uint4 *d, const uint4 *x, int from, int to, int vectors, int lane,
                                                     int64_t (&v)[4]) {
    constexpr int U = 4;  // steps in flight
    const uint4 none = make_uint4(0, 0, 0, 0);
    int hh[4] = {}, mid[4] = {}, ll[4] = {};
#pragma unroll 1
    for (int s = from; s < to; s += U) {
        uint4 w[U], w8[U], r[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = (s + u) * 4 + (lane & 3);
            const bool in = s + u < to;
            w[u] = in ? __ldg(d + (s + u) * 64 + lane) : none;
            w8[u] = in ? __ldg(d + (s + u) * 64 + 32 + lane) : none;
            r[u] = in && at < vectors ? __ldg(x + at) : none;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t low[4] = {w[u].x, w8[u].x, w[u].y, w8[u].y}, high[4] = {w[u].z, w8[u].z, w[u].w, w8[u].w};
            const uint32_t xl0 = __byte_perm(r[u].x, r[u].y, 0x6420), xl1 = __byte_perm(r[u].z, r[u].w, 0x6420);
            const uint32_t xh0 = __byte_perm(r[u].x, r[u].y, 0x7531), xh1 = __byte_perm(r[u].z, r[u].w, 0x7531);
            mma_ss(hh, high, xh0, xh1);
            mma_uu(ll, low, xl0, xl1);
            mma_su(mid, high, xl0, xl1);
            mma_us(mid, low, xh0, xh1);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = ((int64_t)hh[i] << 16) + ((int64_t)mid[i] << 8) + ll[i];
}

// t of rows [row0, row0 + span) for ranks 16 q to 16 q + 15 of their adapters, a pass per
// group of up to 8 rows of one adapter (the group that starts at a row of the span).
// The warps of a block, times the blocks of its cluster, share k.  Every thread of
// the cluster takes the same path: it depends on the row, q and the slots alone.
static __device__ void form_t(const Call &c, uint32_t row0, int q, int share) {
    constexpr int kWarps = kPrepareThreads / 32, kSums = 16 * kGroup;
    __shared__ __align__(16) int64_t sum_s[kWarps][kSums];  // [rank][row] of each warp
    __shared__ int64_t part_s[kMaxSplit][kSums];            // of each block, in the cluster's first
    __shared__ uint64_t part_bar;
    __shared__ __align__(16) int16_t t_s[kGroup][16];       // read as 32-bit words
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int vectors = c.K >> 3, all = kWarps * c.ksplit, part = share * kWarps + warp;
    const int from = c.steps * part / all, to = c.steps * (part + 1) / all;
    bool came = true;    // the other blocks' sums
    uint32_t taken = 0;  // rows of the span that are members of a group of it (a group's first row aside)
    for (uint32_t row = row0; row < min(row0 + c.span, c.rows); row++) {
        if ((taken >> (row - row0)) & 1u) continue;
        const int rt = row / c.NT, at = row - rt * c.NT;
        const int a = c.slot[row];
        if (a < 0 || a >= c.slots) continue;
        const int rank = c.rank[a], scale = c.scale[a];
        const RowMask mask = rows_of_slot(c, rt, a);
        const int order = mask.before(at);
        if (order % kGroup != 0) continue;
        // (the first piece does not wait for the rank: an empty slot's t is formed and never read)
        if (q > 0 && q * 16 >= rank) continue;
        if (c.ksplit > 1) {  // (a block then has one row, so one group at most)
            if (threadIdx.x == 0) {
                mbar_init(&part_bar, 1);
                asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
                mbar_expect_tx(&part_bar, c.ksplit * kSums * 8);
            }
            __syncwarp();
            cluster_arrive();
        }
        // members: the next 8 rows of the mask from this one on
        int member[kGroup], members = 0;
        {
            int next = at;
#pragma unroll
            for (int g = 0; g < kGroup; g++) {
                member[g] = at;  // absent members repeat the first: never stored
                int k = next >> 5;
                uint32_t w = k < kRowTile / 32 ? mask.w[k] & (~0u << (next & 31)) : 0u;
                while (w == 0 && ++k < kRowTile / 32) w = mask.w[k];
                if (k < kRowTile / 32 && w) {
                    member[g] = k * 32 + __ffs((int)w) - 1;
                    members = g + 1;
                    next = member[g] + 1;
                    const uint32_t of_span = row + member[g] - at - row0;
                    if (of_span < 32) taken |= 1u << of_span;
                } else {
                    next = kRowTile;
                }
            }
        }
        auto row_of = [&](int g) {  // member[] stays in registers
            int r = member[0];
#pragma unroll
            for (int u = 1; u < kGroup; u++)
                if (g == u) r = member[u];
            return r;
        };
        const int16_t *x = c.x + ((size_t)rt * c.NT + row_of(lane >> 2)) * c.ld_x;
        int64_t v[4];
        down_products(c.down + ((size_t)a * c.Q + q) * c.steps * 64, reinterpret_cast<const uint4 *>(x), from, to, vectors, lane,
                      v);
        *reinterpret_cast<longlong2 *>(&sum_s[warp][2 * lane]) = make_longlong2(v[0], v[1]);
        *reinterpret_cast<longlong2 *>(&sum_s[warp][2 * lane + 8 * kGroup]) = make_longlong2(v[2], v[3]);
        if (c.ksplit > 1) {
            __syncwarp();
            cluster_wait();
        }
        __syncthreads();  // (also between this wait and the next arrival)
        int64_t sum = 0;
        if (threadIdx.x < kSums)
#pragma unroll
            for (int w = 0; w < kWarps; w++) sum += sum_s[w][threadIdx.x];
        if (c.ksplit > 1) {
            if (threadIdx.x < kSums)
                st_async(remote(&part_s[share][threadIdx.x], 0), (uint64_t)sum, remote(&part_bar, 0));
            __syncwarp();
            cluster_arrive();  // nothing more is sent
            if (share != 0) {
                cluster_leave(true);
                return;
            }
            came = mbar_wait_cluster(&part_bar, 0, c.polls);
            if (!came) atomicExch(c.error, 3);
            sum = 0;
            if (threadIdx.x < kSums)
                for (int p = 0; p < c.ksplit; p++) sum += part_s[p][threadIdx.x];
        }
        if (threadIdx.x < kSums) {
            const int j = threadIdx.x / kGroup, g = threadIdx.x % kGroup;
            t_s[g][j] = q * 16 + j < rank ? (int16_t)sat16(rnd(sum * scale, 24)) : (int16_t)0;
        }
        __syncthreads();
        uint8_t *dst = c.tp + (((size_t)rt * c.NT + mask.first()) * c.Q + q) * c.NT * 32;
        const int g = threadIdx.x / 4, w4 = threadIdx.x % 4;  // 4 ranks per thread
        if (g < members) {
            const uint32_t *t = reinterpret_cast<const uint32_t *>(&t_s[g][4 * w4]);
            uint8_t *p = dst + row_of(g) * 16 + 4 * w4;
            *reinterpret_cast<uint32_t *>(p) = __byte_perm(t[0], t[1], 0x7531);
            *reinterpret_cast<uint32_t *>(p + c.NT * 16) = __byte_perm(t[0], t[1], 0x6420);
        }
        // zeros of the tile's other rows, by the adapter's first group
        if (order == 0)
            for (int u = threadIdx.x; u < c.NT * 4; u += kPrepareThreads) {
                const int r = u / 4, w = u % 4;
                if ((mask.w[r >> 5] >> (r & 31)) & 1u) continue;
                *reinterpret_cast<uint32_t *>(dst + r * 16 + 4 * w) = 0;
                *reinterpret_cast<uint32_t *>(dst + c.NT * 16 + r * 16 + 4 * w) = 0;
            }
        if (c.ksplit > 1) cluster_leave(came);
    }
}

// Blocks (x, share): per x first t, then the rows' pieces and the lists of the row tiles'
// adapters.  Bound by latency: slots 0.7 us, then ranks and the rows of the adapter,
// then products 2 us (one row: 4 KiB of a row, 64 KiB of a rank-16 down matrix) and their
// sums 0.4, or 0.75 across a cluster.  t on the legacy matrix instructions, whose 16 x 8
// tile is 16 ranks of 8 rows, took 512 rows of rank 64 from 65 to 59.5 us against
// dp2a products, whose pipe took 9 us of that; tcgen05 would need the operands in shared
// memory and 128 ranks or rows a tile.
__global__ void __launch_bounds__(kPrepareThreads, 2) k_prepare(const Call c) {
    __shared__ TileSlots ts;
    pdl_wait();     // the caller's rows, and the last call's reads of the workspace
    pdl_trigger();
    const int share = blockIdx.y;
    int b = blockIdx.x;
    const int forms = c.slot ? (int)((c.rows + c.span - 1) / c.span) * c.Q : 0;
    if (b < forms) {
        form_t(c, (uint32_t)(b / c.Q) * c.span, b % c.Q, share);
        return;
    }
    b -= forms;
    const int items = c.RT * (c.P >> 3), splits = (items + c.ksplit - 1) / c.ksplit;
    if (b < splits) {
        if (b * c.ksplit + share < items) split_item(c, b * c.ksplit + share);
        return;
    }
    b -= splits;
    if (share != 0) return;
    const RowSlot r = tile_slots(c, b, ts);  // the list of the row tile's adapter pieces
    if (r.first)
        for (int q = 0; q < pieces_of(c, r.slot); q++)
            c.list[(size_t)b * c.max_pieces + r.base + q] = make_int2(r.slot * c.Q + q, (int)threadIdx.x * c.Q + q);
    if (threadIdx.x == 0) c.count[b] = r.total;
}

// ---------------------------------------------------------------------------
// the projection
// ---------------------------------------------------------------------------
static __host__ __device__ __forceinline__ int header_bytes(int RT) { return (kHeader + (2 * RT + 1) * 4 + 127) / 128 * 128; }
// Shared stages are those of fewer tiles than there are SMs: 32 bits hold them times the CTAs.
static __device__ __forceinline__ int range_begin(int b, int stages, int grid) { return stages * b / grid; }
static __device__ __forceinline__ int cta_of(int i, int stages, int grid) {
    int b = i * grid / stages;
    while (b + 1 < grid && range_begin(b + 1, stages, grid) <= i) b++;
    while (b > 0 && range_begin(b, stages, grid) > i) b--;
    return b;
}
// Stages before shared tile t in the line of all of them (row tiles of the same outputs
// are neighbours); pre[rt]: stages of the row tiles before rt.
static __device__ __forceinline__ int line_at(int t, const int32_t *pre, int RT) {
    return RT == 1 ? t * pre[1] : t / RT * pre[RT] + pre[t % RT];
}

// A CTA's way through the tiles: its run of the stages of the first `shared`
// tiles, then every grid-th of the tiles after them, whole.  A step is the run of
// a tile's stages [begin, end) that the CTA takes: of the weight's (below C), then
// of the adapters'.
struct Walk {
    int tile, ft, rt;     // tile, its outputs and its row tile
    int begin, end, len;  // stages of this step, stages of the tile
    int left;             // stages left in the shared run, this step's included

    __device__ __forceinline__ void set(const Call &c, const int32_t *pre, int t, int stage) {
        tile = t;
        ft = c.RT == 1 ? t : t / c.RT;
        rt = t - ft * c.RT;
        len = pre[rt + 1] - pre[rt];
        begin = stage;
        end = left > 0 ? min(len, begin + left) : len;
    }
    __device__ __forceinline__ void start(const Call &c, const int32_t *pre, int w0, int w1) {
        left = w1 - w0;
        if (left == 0) {
            set(c, pre, c.shared_tiles + blockIdx.x, 0);
            return;
        }
        const int per = pre[c.RT];
        const int f = w0 / per, rem = w0 - f * per;
        int r = 0;
        while (r + 1 < c.RT && pre[r + 1] <= rem) r++;
        set(c, pre, f * c.RT + r, rem - pre[r]);
    }
    __device__ __forceinline__ bool more(const Call &c) const { return left > 0 || tile < c.T * c.RT; }
    __device__ __forceinline__ void next(const Call &c, const int32_t *pre) {
        if (left > 0) {
            left -= end - begin;
            set(c, pre, left > 0 ? tile + 1 : c.shared_tiles + blockIdx.x, 0);
        } else {
            set(c, pre, tile + gridDim.x, 0);
        }
    }
};

// Warp roles: 0 tensor memory and products, 1 loads, the others results.  The issuing
// lanes' instructions pace a stage (an MMA of 32 columns takes 41 cycles, one whose
// descriptors are computed anew 190), so each loop over stages has little more
// than its wait, its issue and its commit: LM head 40 rows 132 -> 111 us.  Result code is
// small for the same reason (it runs a few times per CTA, from a cold instruction
// cache): one body instead of two took 77 rows x 1096 -> 4999 from 31 to 23 us.
// D: pieces per ring stage.  With 8 (narrow row tiles) at most 96 registers a thread
// and kBesideSmem bytes of shared memory: a block of k_prepare then fits beside it, so
// that neither waits for the other's SM.
template <int D>
__global__ void __launch_bounds__(project_threads(D), D == 8 ? 2 : 1) k_project(const Call c) {
    constexpr int kResultThreads = result_threads(D), kResultWarps = kResultThreads / 32;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(smem);  // [kMaxRing] stage loaded
    uint64_t *empty = full + kMaxRing;                    // [kMaxRing] stage consumed
    uint64_t *tfull = empty + kMaxRing;                   // [2] accumulator set complete
    uint64_t *tempty = tfull + 2;                         // [2] accumulator set read out
    uint64_t *done = tempty + 2;                          // every MMA of the CTA complete
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    int *last_s = reinterpret_cast<int *>(tmem_slot + 1);
    int *fail_s = last_s + 1;                             // [16] wait outcome of each result warp
    int32_t *pre = fail_s + 16;                           // [RT + 1] stages before each row tile
    int32_t *pieces = pre + c.RT + 1;                     // [RT] adapter pieces of each row tile
    uint8_t *ring = smem + header_bytes(c.RT);
    const int NT = c.NT, C = c.C, S = c.ring;
    
    const int w_bytes = D * kPiece, x_bytes = D * NT * 32, stage = w_bytes + x_bytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t columns = 32;
    while (columns < (uint32_t)(4 * NT * c.buffers)) columns <<= 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(tfull + b, 1);
            mbar_init(tempty + b, kResultThreads);
        }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // Stages of each row tile.  Where the CTA meets one row tile only, its adapters are
    // counted here, from the slots themselves (k_prepare passed its wait before this
    // kernel could start, so they are final), and the weights can be fetched before
    // k_prepare ends; with more, k_prepare's counts are waited for.
    const bool waits = c.slot && c.RT > 1 && (c.shared_tiles != 0 || c.T * c.RT > (int)gridDim.x);
    if (c.slot && !waits) {
        TileSlots &ts = *reinterpret_cast<TileSlots *>(ring);
        const int own = blockIdx.x % c.RT;
        const RowSlot r = tile_slots(c, own, ts);
        if (threadIdx.x == 0) {
            pieces[own] = r.total;
            for (int rt = 0; rt <= c.RT; rt++) pre[rt] = rt <= own ? 0 : C + (r.total + D - 1) / D;
        }
        // the ring takes this memory over for bulk copies
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    } else {
        if (waits) pdl_wait();
        for (int rt = threadIdx.x; rt < c.RT; rt += blockDim.x) pieces[rt] = c.slot ? __ldcg(c.count + rt) : 0;
        __syncthreads();
        if (threadIdx.x == 0) {
            int n = 0;
            for (int rt = 0; rt < c.RT; rt++) {
                pre[rt] = n;
                n += C + (pieces[rt] + D - 1) / D;
            }
            pre[c.RT] = n;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int line = line_at(c.shared_tiles, pre, c.RT);  // stages that are shared out one by one
    // no more sharers than stages: every CTA between a tile's first and last takes a part in it
    const int sharers = min(c.sharers, max(line, 1)), me = min((int)blockIdx.x, sharers);
    Walk k;
    k.start(c, pre, range_begin(me, line, sharers), range_begin(min(me + 1, sharers), line, sharers));

    if (warp == 1) {  // ---- loads ---------------------------------------------------
        // Lane 0 loads the weight's stages: few instructions per stage, since one
        // thread's latency is all that paces them.  In an adapter stage lanes 0-7 load
        // its pieces and lanes 8-15 their t.
        const uint64_t policy = evict_first_policy();
        auto load_weight = [&](const uint8_t *src, int s) {  // announces the whole stage
            mbar_expect_tx(full + s, stage);
            if (c.RT == 1) bulk_g2s_hint(ring + s * stage, src, w_bytes, full + s, policy);  // read once
            else bulk_g2s(ring + s * stage, src, w_bytes, full + s);
        };
        auto weight_of = [&](const Walk &w, int i) { return c.weight + ((size_t)w.ft * c.P + (size_t)i * D) * kPiece; };
        auto rows_of = [&](const Walk &w, int i) { return c.xp + ((size_t)w.rt * c.P + (size_t)i * D) * NT * 32; };
        // weights of the first stages before k_prepare has finished (unless that has
        // been waited for), up to the first adapter stage, whose list it writes
        Walk w = k;
        int early = 0;
        for (bool go = !waits; go && early < S && w.more(c); w.next(c, pre)) {
            for (int i = w.begin; i < w.end && early < S; i++) {
                if (i >= C) {
                    go = false;
                    break;
                }
                if (lane == 0) load_weight(weight_of(w, i), early);
                early++;
            }
        }
        pdl_wait();
        asm volatile("fence.proxy.async.global;" ::: "memory");  // k_prepare's stores before the bulk reads
        bool ok = true;
        int s = 0, phase = 1, issued = 0;  // phase: of the last use of stage s
        for (; ok && k.more(c); k.next(c, pre)) {
            const int bound = min(k.end, C), first = k.begin;
            if (lane == 0 && first < bound) {
                const uint8_t *src = weight_of(k, first), *rows = rows_of(k, first);
                for (int i = first; i < bound; i++) {
                    if (issued >= S && !mbar_wait(empty + s, phase, c.polls)) {
                        ok = false;
                        break;
                    }
                    if (issued >= early) load_weight(src, s);
                    bulk_g2s(ring + s * stage + w_bytes, rows, x_bytes, full + s);
                    src += w_bytes;
                    rows += x_bytes;
                    issued++;
                    if (++s == S) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
            ok = __shfl_sync(~0u, ok, 0);
            s = __shfl_sync(~0u, s, 0);
            phase = __shfl_sync(~0u, phase, 0);
            issued = __shfl_sync(~0u, issued, 0);
            for (int i = max(first, C); ok && i < k.end; i++) {
                const int p0 = (i - C) * D, np = min(D, pieces[k.rt] - p0);
                const int2 mine = (lane & 7) < np ? __ldcg(c.list + (size_t)k.rt * c.max_pieces + p0 + (lane & 7)) : make_int2(0, 0);
                if (issued >= S) {
                    ok = mbar_wait(empty + s, phase, c.polls);
                    ok = __all_sync(~0u, ok);
                    if (!ok) break;
                }
                uint8_t *dst = ring + s * stage;
                if (lane == 0) mbar_expect_tx(full + s, np * kPiece + ((np + 1) & ~1) * NT * 32);
                __syncwarp();
                if (lane < np) {
                    const int a = mine.x / c.Q, q = mine.x - a * c.Q;
                    bulk_g2s(dst + lane * kPiece, c.up + (((size_t)a * c.T + k.ft) * c.Q + q) * kPiece, kPiece, full + s);
                }
                const int p = lane - 8;  // an odd last piece is paired with one of zeros
                if (p >= 0 && p < ((np + 1) & ~1))
                    bulk_g2s(dst + w_bytes + p * NT * 32,
                             p < np ? c.tp + ((size_t)k.rt * NT * c.Q + mine.y) * NT * 32 : c.zero, NT * 32, full + s);
                issued++;
                if (++s == S) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        if (!ok && lane == 0) atomicExch(c.error, 1);
        // The copies in flight land before the CTA ends, also where the warp that waits for them
        // has given up.  (Every announced stage was issued whole: the first S need no wait.)
        for (int q = 0; lane == 0 && q < S && q < issued; q++) {
            const int last = q + ((issued - 1 - q) / S) * S;
            (void)mbar_wait(full + q, (last / S) & 1);
        }
        __syncwarp();
    } else if (warp == 0) {  // ---- products ---------------------------------------
        // One lane issues.  Descriptors are a stage's first one plus constants: their
        // arithmetic is what limits narrow row tiles (a step of 32 columns takes
        // the tensor cores 41 cycles).
        if (lane == 0) {
            const uint32_t ss2 = umma_idesc_i8(1, 1, 2 * NT), us2 = umma_idesc_i8(0, 1, 2 * NT);  // [xh | xs] of NT rows each
            const uint32_t ss = umma_idesc_i8(1, 1, NT), su = umma_idesc_i8(1, 0, NT), us = umma_idesc_i8(0, 1, NT),
                           uu = umma_idesc_i8(0, 0, NT);  // t's planes one by one, the low one unsigned
            const uint64_t wd0 = umma_desc(smem_u32(ring), kPiece, 128), xd0 = umma_desc(smem_u32(ring) + w_bytes, NT * 32, 128);
            const uint32_t step = (uint32_t)(2 * NT * 32) >> 4;  // two row pieces, in descriptor units
            constexpr uint32_t kStep = 2 * kPiece >> 4, kLow = kPiece / 2 >> 4;
            int tiles = 0, s = 0, phase = 0;
            uint64_t wd = wd0, xd = xd0;
            bool ok = true;
            auto advance = [&] {
                umma_commit(empty + s);
                wd += (uint32_t)stage >> 4;
                xd += (uint32_t)stage >> 4;
                if (++s == S) {
                    s = 0;
                    phase ^= 1;
                    wd = wd0;
                    xd = xd0;
                }
            };
            for (; k.more(c); k.next(c, pre), tiles++) {
                const int b = c.buffers == 2 ? tiles & 1 : 0, use = c.buffers == 2 ? tiles >> 1 : tiles;
                if (use > 0 && !mbar_wait(tempty + b, (use - 1) & 1, c.polls)) ok = false;
                const uint32_t dh = tmem + (uint32_t)(b * 4 * NT), dl = dh + 2 * NT;
                const int bound = min(k.end, C);
                uint32_t more = 0;  // the first product of the step overwrites
                for (int i = k.begin; ok && i < bound; i++) {
                    if (!mbar_wait(full + s, phase, c.polls)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    umma_i8(dh, wd, xd, ss2, more);
                    umma_i8(dl, wd + kLow, xd, us2, more);
#pragma unroll
                    for (int q = 1; q < D / 2; q++) {  // 32-deep steps: two pieces
                        umma_i8(dh, wd + q * kStep, xd + q * step, ss2, 1u);
                        umma_i8(dl, wd + q * kStep + kLow, xd + q * step, us2, 1u);
                    }
                    more = 1;
                    advance();
                }
                for (int i = max(k.begin, C); ok && i < k.end; i++) {
                    if (!mbar_wait(full + s, phase, c.polls)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const int np = min(D, pieces[k.rt] - (i - C) * D);
                    const uint32_t low = (uint32_t)(NT * 16) >> 4;
                    for (int q = 0; 2 * q < np; q++) {
                        const uint64_t wh = wd + q * kStep, th = xd + q * step;
                        umma_i8(dh, wh, th, ss, more);
                        umma_i8(dh + NT, wh, th + low, su, more);
                        umma_i8(dl, wh + kLow, th, us, more);
                        umma_i8(dl + NT, wh + kLow, th + low, uu, more);
                        more = 1;
                    }
                    advance();
                }
                if (!ok) break;
                umma_commit(tfull + b);
            }
            if (!ok) atomicExch(c.error, 2);
            umma_commit(done);  // the accumulators are released only after every MMA
            if (!mbar_wait(done, 0)) atomicExch(c.error, 2);
        }
        __syncwarp();
    } else {  // ---- results: a thread per output of the tile and a half or a quarter of its rows ----
        const int q4 = warp & 3, m = q4 * 32 + lane;   // TMEM lanes of this warp, output of this thread
        const int part = (warp - 2) >> 2;              // rows 8 (i kResultWarps / 4 + part) .. + 7
        for (int tiles = 0; k.more(c); tiles++, k.next(c, pre)) {
            const int b = c.buffers == 2 ? tiles & 1 : 0, use = c.buffers == 2 ? tiles >> 1 : tiles;
            const bool whole = k.begin == 0 && k.end == k.len;
            const int o = k.ft * kOutTile + m;
            const bool live = o < c.N;
            const int64_t corr = k.begin == 0 ? 128 * (int64_t)c.wsum[o] + 8 : 0;  // and half of a Q16.16 step, for the rounding
            const int rows = min(NT, (int)c.rows - k.rt * NT);
            int b_lo = 0, b_hi = 0;
            if (!whole) {
                const int at = line_at(k.tile, pre, c.RT);
                b_lo = cta_of(at, line, sharers);
                b_hi = cta_of(at + k.len - 1, line, sharers);
            }
            unsigned long long *acc = reinterpret_cast<unsigned long long *>(c.acc) + (size_t)b_lo * NT * kOutTile + m;
            const bool okw = mbar_wait_err(tfull + b, use & 1, c.error, c.polls);
            if (lane == 0) fail_s[warp - 2] = okw ? 0 : 1;
            named_sync(3, kResultThreads);
            int failed = 0;
#pragma unroll
            for (int w = 0; w < kResultWarps; w++) failed |= fail_s[w];
            named_sync(3, kResultThreads);  // read by all before the next tile writes it
            if (failed) {
                if (threadIdx.x == 64) atomicCAS(c.error, 0, 3);
                break;
            }
            tc_fence_after();
            const uint32_t t0 = tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(b * 4 * NT);
            // 8 rows at a time: sums from the accumulators, or (a shared tile's last CTA) from
            // memory, into the results or added to memory.  One body for all three
            // keeps the code small: it runs once or twice per CTA, mostly uncached.
            auto rows8 = [&](bool summed, bool add) {
#pragma unroll 1
                for (int r0 = 8 * part; r0 < rows; r0 += 2 * kResultWarps) {
                    int64_t sum[8];
                    unsigned long long *at = acc + (size_t)r0 * kOutTile;
                    const int n = min(8, rows - r0);
                    if (summed) {
#pragma unroll
                        for (int r = 0; r < 8; r++) sum[r] = r < n ? (int64_t)__ldcg(at + r * kOutTile) : 0;
                    } else {
                        uint32_t v[32];
                        tmem_ld4x8(t0 + r0, t0 + NT + r0, t0 + 2 * NT + r0, t0 + 3 * NT + r0, v);
#pragma unroll
                        for (int r = 0; r < 8; r++)
                            // hs + lh <= 2^15 * (2^14 + 255 * 2^7) < 2^31
                            sum[r] = mad_wide((int32_t)v[r], 65536,
                                              mad_wide((int32_t)(v[8 + r] + v[16 + r]), 256, mad_wide((int32_t)v[24 + r], 1, corr)));
                    }
                    if (add) {
#pragma unroll
                        for (int r = 0; r < 8; r++)
                            if (r < n) atomicAdd(at + r * kOutTile, (unsigned long long)sum[r]);
                        continue;
                    }
                    if (summed) {
#pragma unroll
                        for (int r = 0; r < 8; r++)
                            if (r < n) at[r * kOutTile] = 0;  // ready for the next call
                    }
                    const size_t first = ((size_t)k.rt * NT + r0) * c.ld_out + o;
                    if (!live) {
                    } else if (c.wide) {
                        int32_t *out = static_cast<int32_t *>(c.out) + first;
#pragma unroll
                        for (int r = 0; r < 8; r++, out += c.ld_out)
                            if (r < n) *out = to_q16(sum[r]);
                    } else {
                        int16_t *out = static_cast<int16_t *>(c.out) + first;
#pragma unroll
                        for (int r = 0; r < 8; r++, out += c.ld_out)
                            if (r < n) *out = (int16_t)to_q8(to_q16(sum[r]));
                    }
                    __syncwarp();  // the next loads from tensor memory are the whole warp's
                }
            };
            rows8(false, !whole);
            tc_fence_before();
            mbar_arrive(tempty + b);
            if (!whole) {
                named_sync(3, kResultThreads);  // every thread's additions before the release below
                if (threadIdx.x == 64) {
                    int old;
                    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;"
                                 : "=r"(old)
                                 : "l"(c.arrived + b_lo)
                                 : "memory");
                    *last_s = old == b_hi - b_lo;
                }
                named_sync(3, kResultThreads);
                if (*last_s) {
                    rows8(true, false);
                    if (threadIdx.x == 64) c.arrived[b_lo] = 0;
                }
            }
        }
    }
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    }
}

// ---------------------------------------------------------------------------
// layouts
// ---------------------------------------------------------------------------
// Pieces of a dense [rows][ld] matrix: tile t, piece p (columns 16 p .. 16 p + 15) at
// dst + (t * stride_pieces + p) * kPiece as [plane][row][16 bytes], zeros past the matrix.
// kWide: rows of 16-byte aligned vectors of 8 (the weight); else one by one (up matrices).
template <bool kWide>
__global__ void __launch_bounds__(256) k_pack_pieces(const int16_t *__restrict__ src, uint32_t rows, uint32_t cols, uint32_t pieces,
                                                     uint32_t stride_pieces, uint32_t tiles, uint8_t *__restrict__ dst) {
    const uint64_t total = (uint64_t)tiles * pieces * kOutTile;
    for (uint64_t g = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; g < total; g += (uint64_t)gridDim.x * blockDim.x) {
        // 8 rows x 4 pieces per warp: whole sectors are read, core matrices written
        const uint32_t in = (uint32_t)(g % (kOutTile * 4)), m = (in >> 5) * 8 + (in & 7), quad = (in >> 3) & 3;
        const uint64_t rest = g / (kOutTile * 4);
        const uint32_t quads = pieces / 4;
        uint32_t p, t;
        if (kWide) {
            t = (uint32_t)(rest / quads);
            p = (uint32_t)(rest % quads) * 4 + quad;
        } else {
            const uint64_t lin = g / kOutTile;
            t = (uint32_t)(lin / pieces);
            p = (uint32_t)(lin % pieces);
        }
        const uint32_t mm = kWide ? m : (uint32_t)(g % kOutTile), row = t * kOutTile + mm;
        uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (row < rows) {
            if (kWide) {
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (p * 16 + h * 8 < cols)
                        v[h] = *reinterpret_cast<const uint4 *>(src + (size_t)row * cols + p * 16 + h * 8);
            } else {
                uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (p * 16 + e < cols) w[e >> 1] |= (uint32_t)(uint16_t)src[(size_t)row * cols + p * 16 + e] << (16 * (e & 1));
                v[0] = make_uint4(w[0], w[1], w[2], w[3]);
                v[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
        uint8_t *d = dst + ((size_t)t * stride_pieces + p) * kPiece + mm * 16;
        *reinterpret_cast<uint4 *>(d) = make_uint4(__byte_perm(v[0].x, v[0].y, 0x7531), __byte_perm(v[0].z, v[0].w, 0x7531),
                                                   __byte_perm(v[1].x, v[1].y, 0x7531), __byte_perm(v[1].z, v[1].w, 0x7531));
        *reinterpret_cast<uint4 *>(d + kPiece / 2) =
            make_uint4(__byte_perm(v[0].x, v[0].y, 0x6420), __byte_perm(v[0].z, v[0].w, 0x6420),
                       __byte_perm(v[1].x, v[1].y, 0x6420), __byte_perm(v[1].z, v[1].w, 0x6420));
    }
}
// Sum of every output's weights (|sum| <= 2^15 * 32768: 32 bits hold it), 0 past the last output.
__global__ void __launch_bounds__(256) k_weight_sums(const int16_t *__restrict__ src, uint32_t rows, uint32_t cols,
                                                     uint32_t padded, int32_t *__restrict__ sums) {
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= padded) return;
    int32_t s = 0;
    if (row < rows) {
        const uint4 *p = reinterpret_cast<const uint4 *>(src + (size_t)row * cols);
        for (uint32_t k = lane; k < cols / 8; k += 32) {
            const uint4 v = p[k];
            s += lo16(v.x) + hi16(v.x) + lo16(v.y) + hi16(v.y) + lo16(v.z) + hi16(v.z) + lo16(v.w) + hi16(v.w);
        }
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (lane == 0) sums[row] = s;
}
// down [rank][K] -> [rank / 16][step of 32 inputs][half][lane]: the operands of t's products
// as their lanes take them, 8 inputs of a rank's row as {low bytes, high bytes}, so that
// a warp reads 512 bytes in a row; zeros past the last rank and input
__global__ void k_pack_down(const int16_t *__restrict__ src, uint32_t rank, uint32_t cols, uint32_t steps,
                            uint4 *__restrict__ dst) {
    const uint32_t n = (rank + 15) / 16 * steps * 64;
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
        const uint32_t lane = i & 31, step = i / 64 % steps, row = i / 64 / steps * 16 + (i >> 5 & 1) * 8 + lane / 4;
        const uint32_t col = (step * 4 + lane % 4) * 8;
        const uint4 v = row < rank && col < cols ? *reinterpret_cast<const uint4 *>(src + (size_t)row * cols + col)
                                                 : make_uint4(0, 0, 0, 0);
        dst[i] = make_uint4(__byte_perm(v.x, v.y, 0x6420), __byte_perm(v.z, v.w, 0x6420), __byte_perm(v.x, v.y, 0x7531),
                            __byte_perm(v.z, v.w, 0x7531));
    }
}
__global__ void k_set_slot(int32_t *ranks, int32_t *scales, uint32_t slot, int32_t rank, int32_t scale) {
    ranks[slot] = rank;
    scales[slot] = scale;
}

// Rows per tile when a call's rows are spread over rt row tiles, in steps of 16
// (the MMA's column granularity).
int rows_per_tile(uint32_t rows, int rt) { return (int)(((rows + rt - 1) / rt + 15) / 16 * 16); }
int row_tiles(uint32_t rows) { return (int)((rows + kRowTile - 1) / kRowTile); }

// Tiles whose stages are shared out one by one: all when there are fewer tiles
// than CTAs, else what is left after whole tiles for every CTA -- unless that is
// nearly another one for each, which then costs less than adding up shared tiles.
int shared_tiles(int64_t tiles, int ctas) {
    if (tiles < ctas) return (int)tiles;
    const int rest = (int)(tiles % ctas);
    return 4 * rest >= 3 * ctas ? 0 : rest;
}

}  // namespace

struct llmx_adapters {
    int dev = 0, sms = 0;
    uint32_t in_dim = 0, out_dim = 0, slots = 0, max_rank = 0, max_rows = 0;
    int P = 0, T = 0, Q = 0, row_cap = 0;  // row_cap: most rows per row tile of any call
    uint8_t *memory = nullptr;   // the one allocation
    uint8_t *weight = nullptr;   // pieces [T][P]
    int32_t *wsum = nullptr;     // [T * 128]
    uint4 *down = nullptr;    // [slots][Q][steps of 32 inputs][2][32]
    uint8_t *up = nullptr;       // pieces [slots][T][Q]
    int32_t *rank = nullptr, *scale = nullptr;  // [slots]
    uint8_t *xp = nullptr, *tp = nullptr, *zero = nullptr;  // row and t pieces of a call, a piece of zeros
    int2 *list = nullptr;                       // adapter pieces of its row tiles
    int32_t *count = nullptr;
    int64_t *acc = nullptr;
    int32_t *arrived = nullptr;
    int *error = nullptr;
    uint64_t bytes = 0;

    size_t max_pieces(int nt) const { return std::min<size_t>((size_t)nt, slots) * Q; }  // of one row tile
    size_t acc_bytes() const { return (size_t)sms * row_cap * kOutTile * 8; }
};

namespace {

int fail(int code, const std::string &msg) {
    set_last_error("adapters: " + msg);
    return code;
}
// The runtime keeps a failed call's code for the thread's next check of a launch, of any
// operator: it is reported here, and only here.
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

void release(llmx_adapters *h) {
    cudaFree(h->memory);
    delete h;
}

cudaError_t launch(const void *fn, dim3 grid, int cluster_y, int threads, size_t smem, const Call &c, cudaStream_t s) {
    Call copy = c;
    void *args[] = {&copy};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = (unsigned)cluster_y;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster_y > 1 ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace

extern "C" int llmx_adapters_create(int device, uint32_t in_dim, uint32_t out_dim, const int16_t *weight,
                                    uint32_t slots, uint32_t max_rank, uint32_t max_rows, void *stream,
                                    llmx_adapters **out) {
    if (!weight || !out) return fail(LLMX_ERR_ARG, "null pointer");
    *out = nullptr;
    if (in_dim == 0 || in_dim % 8 != 0 || in_dim > kMaxIn)
        return fail(LLMX_ERR_ARG, "in_dim must be a multiple of 8 up to 32768, got " + std::to_string(in_dim));
    if (out_dim == 0 || out_dim > kMaxOut)
        return fail(LLMX_ERR_ARG, "out_dim must be 1..2^22, got " + std::to_string(out_dim));
    if (slots > kMaxSlots) return fail(LLMX_ERR_ARG, "slots must be at most 65536, got " + std::to_string(slots));
    if (slots && (max_rank == 0 || max_rank > kMaxRank))
        return fail(LLMX_ERR_ARG, "max_rank must be 1..128, got " + std::to_string(max_rank));
    if (max_rows == 0 || max_rows > kMaxCallRows)
        return fail(LLMX_ERR_ARG, "max_rows must be 1..65536, got " + std::to_string(max_rows));
    if ((uintptr_t)weight & 15u) return fail(LLMX_ERR_ARG, "weight must be 16-byte aligned");
    DeviceScope scope(device);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    llmx_adapters *h = new (std::nothrow) llmx_adapters;
    if (!h) return fail(LLMX_ERR_NOMEM, "host allocation failed");
    h->dev = device;
    h->in_dim = in_dim;
    h->out_dim = out_dim;
    h->slots = slots;
    h->max_rank = slots ? max_rank : 0;
    h->max_rows = max_rows;
    h->P = (int)((in_dim + 127) / 128 * 8);
    h->T = (int)((out_dim + kOutTile - 1) / kOutTile);
    h->Q = (int)((h->max_rank + 15) / 16);
    h->row_cap = max_rows > kRowTile ? kRowTile : rows_per_tile(max_rows, 1);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if ((e = cudaDeviceGetAttribute(&h->sms, cudaDevAttrMultiProcessorCount, device)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(k_project<8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kProjectSmem)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(k_project<4>, cudaFuncAttributeMaxDynamicSharedMemorySize, kProjectSmem)) != cudaSuccess ||
        // an SM changes its division into L1 and shared memory only when it is empty: with
        // k_prepare's default one k_project would wait for its blocks to end
        (e = cudaFuncSetAttribute(k_prepare, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared)) !=
            cudaSuccess) {
        release(h);
        return cuda_fail("create", e);
    }
    const size_t rt = (size_t)row_tiles(max_rows) + (max_rows > kRowTile || 2 * (int64_t)h->T <= h->sms ? kMoreTiles : 0);
    const size_t xt = rt == 1 ? (size_t)h->row_cap : max_rows + 16 * rt;  // rows of all row tiles
    const size_t pieces = h->max_pieces(h->row_cap);
    // one allocation; what has to start as zeros lies at its front
    size_t at = 0;
    auto place = [&](size_t n) {
        const size_t was = at;
        at += (n + 255) / 256 * 256;
        return was;
    };
    const size_t rank_at = place((size_t)slots * 4), zero_at = place((size_t)h->row_cap * 32), acc_at = place(h->acc_bytes()),
                 arrived_at = place((size_t)h->sms * 4), error_at = place(4),
                 // ranks of a slot that no adapter fills are multiplied by nothing, but read
                 down_at = place((size_t)slots * h->Q * ((in_dim + 31) / 32) * 64 * sizeof(uint4)), zeros = at, scale_at = place((size_t)slots * 4),
                 wsum_at = place((size_t)h->T * kOutTile * 4), xp_at = place(xt * h->P * 32),
                 tp_at = place(xt * h->Q * h->row_cap * 32), list_at = place(rt * pieces * 8), count_at = place(rt * 4),
                 up_at = place((size_t)slots * h->T * h->Q * kPiece), weight_at = place((size_t)h->T * h->P * kPiece);
    h->bytes = at;
    if ((e = cudaMalloc(reinterpret_cast<void **>(&h->memory), at)) != cudaSuccess ||
        (e = cudaMemsetAsync(h->memory, 0, zeros, s)) != cudaSuccess) {
        release(h);
        return cuda_fail("create", e);
    }
    auto as = [&](auto *&p, size_t where) { p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(h->memory + where); };
    as(h->rank, rank_at);
    as(h->zero, zero_at);
    as(h->acc, acc_at);
    as(h->arrived, arrived_at);
    as(h->error, error_at);
    as(h->down, down_at);
    as(h->scale, scale_at);
    as(h->wsum, wsum_at);
    as(h->xp, xp_at);
    as(h->tp, tp_at);
    as(h->list, list_at);
    as(h->count, count_at);
    as(h->up, up_at);
    as(h->weight, weight_at);
    k_pack_pieces<true><<<h->sms * 8, 256, 0, s>>>(weight, out_dim, in_dim, h->P, h->P, h->T, h->weight);
    k_weight_sums<<<h->T * (kOutTile / 8), 256, 0, s>>>(weight, out_dim, in_dim, h->T * kOutTile, h->wsum);
    if ((e = cudaGetLastError()) != cudaSuccess) {
        release(h);
        return cuda_fail("create", e);
    }
    *out = h;
    return LLMX_OK;
}

extern "C" int llmx_adapters_destroy(llmx_adapters *h) {
    if (!h) return LLMX_OK;
    DeviceScope scope(h->dev);
    release(h);
    return LLMX_OK;
}

extern "C" int llmx_adapters_set(llmx_adapters *h, uint32_t slot, uint32_t rank, int16_t scale, const int16_t *down,
                                 const int16_t *up, void *stream) {
    if (!h) return fail(LLMX_ERR_ARG, "null handle");
    if (slot >= h->slots)
        return fail(LLMX_ERR_ARG, "slot " + std::to_string(slot) + " of " + std::to_string(h->slots));
    if (rank > h->max_rank)
        return fail(LLMX_ERR_ARG, "rank " + std::to_string(rank) + " above max_rank " + std::to_string(h->max_rank));
    if (rank && (!down || !up)) return fail(LLMX_ERR_ARG, "null adapter matrix");
    if (rank && (((uintptr_t)down & 15u) || ((uintptr_t)up & 1u)))
        return fail(LLMX_ERR_ARG, "down must be 16-byte aligned, up 2-byte aligned");
    DeviceScope scope(h->dev);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rank) {
        const uint32_t used = (rank + 15) / 16, steps = (h->in_dim + 31) / 32;
        k_pack_down<<<256, 256, 0, s>>>(down, rank, h->in_dim, steps, h->down + (size_t)slot * h->Q * steps * 64);
        k_pack_pieces<false><<<h->sms * 4, 256, 0, s>>>(up, h->out_dim, rank, used, h->Q, h->T,
                                                        h->up + (size_t)slot * h->T * h->Q * kPiece);
    }
    k_set_slot<<<1, 1, 0, s>>>(h->rank, h->scale, slot, (int32_t)rank, scale);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LLMX_OK : cuda_fail("set", e);
}

extern "C" int llmx_adapters_project(llmx_adapters *h, const int16_t *x, uint32_t rows, size_t ld_x,
                                     const int32_t *slot, void *out, int out_format, size_t ld_out, void *stream) {
    if (!h) return fail(LLMX_ERR_ARG, "null handle");
    if (out_format != LLMX_OUT_Q8_8 && out_format != LLMX_OUT_Q16_16)
        return fail(LLMX_ERR_ARG, "out_format must be LLMX_OUT_Q8_8 or LLMX_OUT_Q16_16");
    if (rows > h->max_rows)
        return fail(LLMX_ERR_ARG, "rows " + std::to_string(rows) + " above max_rows " + std::to_string(h->max_rows));
    if (ld_x == 0) ld_x = h->in_dim;
    if (ld_out == 0) ld_out = h->out_dim;
    if (ld_x < h->in_dim || ld_x % 8 != 0) return fail(LLMX_ERR_ARG, "ld_x must be a multiple of 8 not below in_dim");
    if (ld_out < h->out_dim) return fail(LLMX_ERR_ARG, "ld_out is below out_dim");
    if (rows == 0) return LLMX_OK;
    if (!x || !out) return fail(LLMX_ERR_ARG, "null pointer");
    const bool wide = out_format == LLMX_OUT_Q16_16;
    if (((uintptr_t)x & 15u) || ((uintptr_t)out & (wide ? 3u : 1u)) || ((uintptr_t)slot & 3u))
        return fail(LLMX_ERR_ARG, "x must be 16-byte aligned, out and slot aligned to their elements");
    DeviceScope scope(h->dev);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Call c{};
    c.x = x;
    c.ld_x = ld_x;
    c.slot = h->slots ? slot : nullptr;
    c.out = out;
    c.ld_out = ld_out;
    c.rows = rows;
    c.wide = wide;
    c.K = (int)h->in_dim;
    c.P = h->P;
    c.T = h->T;
    c.N = (int)h->out_dim;
    // Row tiles: the fewest, or a few more where narrower tiles fill the CTAs' turns better.
    // A stage's time goes as its bytes, 128 outputs and NT rows wide.
    double best = 0;
    for (int rt = row_tiles(rows); rt <= row_tiles(rows) + (rows > kRowTile ? kMoreTiles : 0); rt++) {
        const int nt = rows_per_tile(rows, rt), shared = shared_tiles((int64_t)h->T * rt, h->sms);
        const double turns = (double)(((int64_t)h->T * rt - shared + h->sms - 1) / h->sms) + (double)shared / h->sms;
        if (c.RT == 0 || turns * (kOutTile + nt) < best) {
            best = turns * (kOutTile + nt);
            c.RT = rt;
            c.NT = nt;
            c.shared_tiles = shared;
        }
    }
    // Fewer tiles than CTAs: a tile's stages of 128 inputs, one after another or shared
    // out and then added up, and its results.  More row tiles make both shorter.
    auto tile_us = [&](int rt, int nt, bool cut) {
        const double depth = std::max(kStageUs, kStageRowUs * nt) * (h->P / 8);
        const double adding = kAddUs + kAddRowUs * std::min<int>((int)rows, nt) + (rt > 1 ? kLateUs : 0);
        return (cut ? depth * ((double)h->T * rt / h->sms) + adding : depth) + kResultRowUs * nt;
    };
    const int fewest = row_tiles(rows);
    for (int rt = fewest; rt <= fewest + kMoreTiles && (int64_t)h->T * rt <= h->sms; rt++) {
        const int nt = rows_per_tile(rows, rt);
        const bool cut = tile_us(rt, nt, true) < tile_us(rt, nt, false);
        const double us = tile_us(rt, nt, cut);
        if (rt > fewest && ((uint32_t)((rt - 1) * nt) >= rows || us >= best)) continue;
        best = us;
        c.RT = rt;
        c.NT = nt;
        c.shared_tiles = cut ? h->T * rt : 0;
    }
    c.slots = (int)h->slots;
    c.Q = h->Q;
    c.max_pieces = (int)h->max_pieces(c.NT);
    c.steps = (int)((h->in_dim + 31) / 32);
    c.weight = h->weight;
    c.wsum = h->wsum;
    c.up = h->up;
    c.down = h->down;
    c.rank = h->rank;
    c.scale = h->scale;
    c.xp = h->xp;
    c.tp = h->tp;
    c.zero = h->zero;
    c.list = h->list;
    c.count = h->count;
    c.acc = h->acc;
    c.arrived = h->arrived;
    c.error = h->error;
    c.polls = serving_wait_polls();
    c.buffers = c.NT <= 64 ? 2 : 1;  // 4 sums x NT columns each, 512 in all
    c.D = c.NT < 96 ? 8 : 4;
    c.C = c.P / c.D;
    const int stage = c.D * (kPiece + c.NT * 32), header = header_bytes(c.RT);
    c.ring = std::min(kMaxRing, ((c.NT <= 64 ? kBesideSmem : kProjectSmem) - header) / stage);
    const int grid = (int)std::min<int64_t>(h->sms, (int64_t)c.T * c.RT * c.C);
    // A shared tile is cut into equal parts where that leaves at most a quarter of the CTAs
    // without one (every part then belongs to one tile only), else the line of all
    // their stages is cut evenly.
    const int parts = c.shared_tiles ? grid / c.shared_tiles : 0;
    c.sharers = 4 * parts * c.shared_tiles >= 3 * grid ? parts * c.shared_tiles : grid;
    // t: a block per row and 16 ranks while that is few blocks or few rows (most end at once:
    // the first row of 8 of an adapter does the work), else per 8 rows.  Few blocks cut k
    // beyond their warps, over up to 8 of a cluster, in runs of more than 2048 inputs: the
    // exchange costs 1 to 2 us (16 rows x 2048 cut in two 26.2 -> 28.6).
    const bool few = c.slot && (int64_t)rows * c.Q <= h->sms;
    c.span = few || rows <= kRowTile ? 1 : kGroup;
    const int forms = c.slot ? (int)((rows + c.span - 1) / c.span) * c.Q : 0;
    c.ksplit = 1;
    while (few && c.ksplit < kMaxSplit && c.K > kSplitInputs * c.ksplit) c.ksplit *= 2;
    const dim3 blocks((unsigned)(forms + (c.RT * (c.P / 8) + c.ksplit - 1) / c.ksplit + (c.slot ? c.RT : 0)), (unsigned)c.ksplit);
    cudaError_t e = launch((const void *)k_prepare, blocks, c.ksplit, kPrepareThreads, 0, c, s);
    if (e == cudaSuccess)
        e = launch(c.D == 8 ? (const void *)k_project<8> : (const void *)k_project<4>, dim3((unsigned)grid), 1, project_threads(c.D),
                   header + (size_t)c.ring * stage, c, s);
    return e == cudaSuccess ? LLMX_OK : cuda_fail("project", e);
}

extern "C" int llmx_adapters_error(llmx_adapters *h, void *stream) {
    if (!h) return fail(LLMX_ERR_ARG, "null handle");
    DeviceScope scope(h->dev);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int word = 0;
    cudaError_t e = cudaMemcpyAsync(&word, h->error, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && word) {  // what a call that gave up left behind
        e = cudaMemsetAsync(h->error, 0, 4, s);
        if (e == cudaSuccess) e = cudaMemsetAsync(h->acc, 0, h->acc_bytes(), s);
        if (e == cudaSuccess) e = cudaMemsetAsync(h->arrived, 0, (size_t)h->sms * 4, s);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    }
    if (e != cudaSuccess) return cuda_fail("error", e);
    return word ? fail(LLMX_ERR_TIMEOUT, "a kernel's bounded wait expired (code " + std::to_string(word) + ")") : LLMX_OK;
}

extern "C" uint64_t llmx_adapters_device_bytes(const llmx_adapters *h) { return h ? h->bytes : 0; }
