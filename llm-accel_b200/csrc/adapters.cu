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
// longer sum over k and nothing is rounded in between.  A row of rank 16 with
// up values of 0.05 then differs by about 16^(1/2) * 0.05 * 2^-9 = 4e-4 from
// one with unrounded t, a tenth of the Q8.8 result's own step.
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
// [high | low][row tile][16 bytes].  Eight weight pieces in a row are an item of 128 outputs x
// 128 inputs; an adapter of rank r has ceil(r / 16) pieces per 128 outputs, so
// pieces of different adapters fill one 32-deep MMA step together and a rank of 16
// wastes nothing.  All of it lands in shared memory by 1-D bulk copies.
//
// Two launches per call.  k_prepare splits the rows into pieces and forms t (a
// block per 16 ranks and up to 8 rows of one adapter in one row tile, so that
// an adapter's down matrix is read once for 8 rows).  k_project streams the
// items: tiles of 128 outputs x up to 128 rows, the items of all tiles in one
// line cut evenly over one CTA per SM (a tile cut between CTAs is summed in
// int64 atomics, which no order changes, and finished by the last to arrive);
// row tiles of the same outputs are neighbours in that line, so a weight item
// comes from HBM once.  k_project starts under k_prepare (dependent launch): its
// ring of weight items fills while the rows are still being split.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <new>
#include <string>

#include "llmx.h"
#include "device_util.cuh"
#include "fixed.cuh"
#include "gemv_common.cuh"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace {

using namespace llmx;

constexpr uint32_t kMaxIn = 32768, kMaxOut = 1u << 22, kMaxSlots = 65536, kMaxRank = 128, kMaxCallRows = 65536;
constexpr int kOutTile = 128;             // outputs per tile (TMEM lanes) and inputs per item
constexpr int kRowTile = 128;          // most rows per tile: 4 sums x 128 rows = all 512 TMEM columns
constexpr int kPiece = 2 * kOutTile * 16; // bytes of a weight piece: two planes of 128 x 16
constexpr int kItem = 8 * kPiece;
constexpr int kProjectThreads = 6 * 32;
constexpr int kHeader = 3072;          // barriers, flags, row-tile table at the start of shared memory
constexpr int kMaxRing = 8;
static_assert(192 + (kMaxCallRows / kRowTile + 1) * 4 <= kHeader, "the row-tile table lies in the header");
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
    int K, C, T, N;       // inputs, chunks of 128, tiles of 128 outputs, outputs
    int NT, RT;           // rows per row tile (a multiple of 16), row tiles
    int slots, Q;         // pieces reserved per adapter
    int max_pieces;       // adapter pieces of one row tile at most (even)
    int down_words;       // 32-bit words of one down row
    const uint8_t *weight; // items [T][C]
    const int32_t *wsum;   // [T * 128] sums of the weights of an output
    const uint8_t *up;     // pieces [slots][T][Q]
    const uint32_t *down;  // [slots][16 Q][K / 2] words {lo(w0), lo(w1), hi(w0), hi(w1)}
    const int32_t *rank, *scale;
    uint8_t *xp;           // row pieces [RT][C][8]
    uint8_t *tp;           // t pieces [RT][max_pieces]
    int32_t *list;         // [RT][max_pieces] slot * Q + piece
    int32_t *count;        // [RT] pieces
    int64_t *acc;          // [grid][NT][128] sums of tiles cut between CTAs, zero between calls
    int32_t *arrived;      // [grid]
    int *error;
    int ring, buffers;     // ring stages, accumulator sets
};

static __device__ __forceinline__ int slot_of(const Call &c, uint32_t row) {
    if (!c.slot || row >= c.rows) return -1;
    const int a = c.slot[row];
    return a >= 0 && a < c.slots && c.rank[a] > 0 ? a : -1;
}
static __device__ __forceinline__ int pieces_of(const Call &c, int a) { return a >= 0 ? (c.rank[a] + 15) >> 4 : 0; }

// The adapters of one row tile.  Thread t < 128 stands for row t of the tile:
// its slot, its place among the rows of that slot, and where that adapter's
// pieces start in the tile's list (adapters in the order of their first rows).
struct TileSlots {
    int32_t slot[kRowTile], base[kRowTile];
    int32_t warp_sum[4];
};
struct RowSlot {
    int slot, order, base, total;
};
static __device__ RowSlot tile_slots(const Call &c, int rt, TileSlots &s) {
    const int t = threadIdx.x, lane = t & 31;
    RowSlot r{-1, 0, 0, 0};
    if (t < kRowTile) {
        r.slot = t < c.NT ? slot_of(c, (uint32_t)rt * c.NT + t) : -1;
        s.slot[t] = r.slot;
    }
    __syncthreads();
    int leader = t, scan = 0, own = 0;
    if (t < kRowTile) {
        if (r.slot >= 0)
            for (int u = 0; u < t; u++)
                if (s.slot[u] == r.slot) {
                    if (r.order == 0) leader = u;
                    r.order++;
                }
        own = r.order == 0 ? pieces_of(c, r.slot) : 0;
        scan = own;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) s.warp_sum[t >> 5] = scan;
    }
    __syncthreads();
    if (t < kRowTile) {
        int before = 0;
        for (int w = 0; w < (t >> 5); w++) before += s.warp_sum[w];
        s.base[t] = before + scan - own;
    }
    __syncthreads();
    if (t < kRowTile) r.base = s.base[leader];
    r.total = s.warp_sum[0] + s.warp_sum[1] + s.warp_sum[2] + s.warp_sum[3];
    return r;
}

// ---------------------------------------------------------------------------
// rows -> byte planes, t -> byte planes, the lists of adapter pieces
// ---------------------------------------------------------------------------
static __device__ void split_item(const Call &c, int item) {
    const int rt = item / c.C, chunk = item - rt * c.C;
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

constexpr int kPrepareThreads = 256;

// t of up to 8 rows of one adapter for 16 of its ranks, and the zeros of the
// tile's other rows (by the adapter's first group).
static __device__ void form_t(const Call &c, uint32_t row, int q, TileSlots &ts) {
    __shared__ int32_t member_s[kGroup];
    __shared__ int32_t me_s[2];  // order and base of this block's row
    __shared__ int16_t t_s[kGroup][16];
    const int a = slot_of(c, row);
    if (a < 0 || q >= pieces_of(c, a)) return;
    const int rt = row / c.NT, at = row - rt * c.NT;
    const int rank = c.rank[a], scale = c.scale[a];
    const RowSlot r = tile_slots(c, rt, ts);
    if (threadIdx.x < kGroup) member_s[threadIdx.x] = -1;
    if ((int)threadIdx.x == at) {
        me_s[0] = r.order;
        me_s[1] = r.base;
    }
    __syncthreads();
    const int order = me_s[0], base = me_s[1] + q;
    if (order % kGroup != 0) return;
    if (r.slot == a && r.order >= order && r.order < order + kGroup) member_s[r.order - order] = threadIdx.x;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int j0 = q * 16 + warp * 2;  // two ranks per warp
    const int16_t *xr[kGroup];
#pragma unroll
    for (int g = 0; g < kGroup; g++)  // absent members repeat the first: loaded, not stored
        xr[g] = c.x + ((size_t)rt * c.NT + (member_s[g] >= 0 ? member_s[g] : at)) * c.ld_x;
    const uint32_t *d0 = c.down + ((size_t)a * c.Q * 16 + j0) * c.down_words, *d1 = d0 + c.down_words;
    const int members = 1 + (member_s[1] >= 0) + (member_s[2] >= 0) + (member_s[3] >= 0) + (member_s[4] >= 0) +
                        (member_s[5] >= 0) + (member_s[6] >= 0) + (member_s[7] >= 0);
    int64_t sum[2 * kGroup];
#pragma unroll
    for (int g = 0; g < 2 * kGroup; g++) sum[g] = 0;
    const int vectors = c.K >> 3;
    for (int v0 = 0; v0 < vectors; v0 += 32 * 16) {
        // 16 vectors of 8 products per lane between flushes: |lo| <= 128 * 255 * 2^15 < 2^30
        int lo[2 * kGroup], hi[2 * kGroup];
#pragma unroll
        for (int g = 0; g < 2 * kGroup; g++) lo[g] = hi[g] = 0;
#pragma unroll 2
        for (int k = 0; k < 16; k++) {
            const int v = v0 + k * 32 + lane;
            if (v >= vectors) break;
            const uint4 w0 = __ldg(reinterpret_cast<const uint4 *>(d0) + v), w1 = __ldg(reinterpret_cast<const uint4 *>(d1) + v);
#pragma unroll
            for (int g = 0; g < kGroup; g++) {
                if (g >= members) break;
                const uint4 x = __ldg(reinterpret_cast<const uint4 *>(xr[g]) + v);
                lo[2 * g] = dp2a_lo_su(x.x, w0.x, lo[2 * g]);
                hi[2 * g] = dp2a_hi_ss(x.x, w0.x, hi[2 * g]);
                lo[2 * g] = dp2a_lo_su(x.y, w0.y, lo[2 * g]);
                hi[2 * g] = dp2a_hi_ss(x.y, w0.y, hi[2 * g]);
                lo[2 * g] = dp2a_lo_su(x.z, w0.z, lo[2 * g]);
                hi[2 * g] = dp2a_hi_ss(x.z, w0.z, hi[2 * g]);
                lo[2 * g] = dp2a_lo_su(x.w, w0.w, lo[2 * g]);
                hi[2 * g] = dp2a_hi_ss(x.w, w0.w, hi[2 * g]);
                lo[2 * g + 1] = dp2a_lo_su(x.x, w1.x, lo[2 * g + 1]);
                hi[2 * g + 1] = dp2a_hi_ss(x.x, w1.x, hi[2 * g + 1]);
                lo[2 * g + 1] = dp2a_lo_su(x.y, w1.y, lo[2 * g + 1]);
                hi[2 * g + 1] = dp2a_hi_ss(x.y, w1.y, hi[2 * g + 1]);
                lo[2 * g + 1] = dp2a_lo_su(x.z, w1.z, lo[2 * g + 1]);
                hi[2 * g + 1] = dp2a_hi_ss(x.z, w1.z, hi[2 * g + 1]);
                lo[2 * g + 1] = dp2a_lo_su(x.w, w1.w, lo[2 * g + 1]);
                hi[2 * g + 1] = dp2a_hi_ss(x.w, w1.w, hi[2 * g + 1]);
            }
        }
#pragma unroll
        for (int g = 0; g < 2 * kGroup; g++) sum[g] += (int64_t)hi[g] * 256 + lo[g];
    }
    int idx;
    const int64_t s = warp_reduce_n<2 * kGroup>(sum, lane, idx);
    if ((lane & 1) == 0) {  // two lanes hold each sum
        const int j = j0 + (idx & 1);
        t_s[idx >> 1][warp * 2 + (idx & 1)] = j < rank ? (int16_t)sat16(rnd(s * scale, 24)) : (int16_t)0;
    }
    __syncthreads();
    uint8_t *dst = c.tp + ((size_t)rt * c.max_pieces + base) * c.NT * 32;
    if (threadIdx.x < kGroup && member_s[threadIdx.x] >= 0) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t *p = reinterpret_cast<const uint32_t *>(&t_s[threadIdx.x][4 * k]);
            hi[k] = __byte_perm(p[0], p[1], 0x7531);
            lo[k] = __byte_perm(p[0], p[1], 0x6420);
        }
        uint8_t *p = dst + member_s[threadIdx.x] * 16;
        *reinterpret_cast<uint4 *>(p) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(p + c.NT * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if (order == 0 && (int)threadIdx.x < c.NT && r.slot != a) {
        *reinterpret_cast<uint4 *>(dst + threadIdx.x * 16) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4 *>(dst + c.NT * 16 + threadIdx.x * 16) = make_uint4(0, 0, 0, 0);
    }
}

__global__ void __launch_bounds__(kPrepareThreads) k_prepare(const Call c) {
    __shared__ TileSlots ts;
    pdl_wait();     // the caller's rows, and the last call's reads of the workspace
    pdl_trigger();
    const int splits = c.RT * c.C;
    int b = blockIdx.x;
    if (b < splits) {
        split_item(c, b);
        return;
    }
    b -= splits;
    if (b < c.RT) {  // the list of the row tile's adapter pieces
        const RowSlot r = tile_slots(c, b, ts);
        if (r.slot >= 0 && r.order == 0)
            for (int q = 0; q < pieces_of(c, r.slot); q++) c.list[(size_t)b * c.max_pieces + r.base + q] = r.slot * c.Q + q;
        if (threadIdx.x == 0) c.count[b] = r.total;
        if (r.total & 1) {  // the second half of the last MMA step: zeros
            uint4 *z = reinterpret_cast<uint4 *>(c.tp + ((size_t)b * c.max_pieces + r.total) * c.NT * 32);
            for (int u = threadIdx.x; u < c.NT * 2; u += blockDim.x) z[u] = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    b -= c.RT;
    form_t(c, (uint32_t)(b / c.Q), b % c.Q, ts);
}

// ---------------------------------------------------------------------------
// the projection
// ---------------------------------------------------------------------------
static __device__ __forceinline__ int64_t range_begin(int b, int64_t items, int grid) { return items * b / grid; }
static __device__ __forceinline__ int cta_of(int64_t i, int64_t items, int grid) {
    int b = (int)(i * grid / items);
    while (b + 1 < grid && range_begin(b + 1, items, grid) <= i) b++;
    while (b > 0 && range_begin(b, items, grid) > i) b--;
    return b;
}

// A place in the line of items: outputs tile ft, row tile rt, item i of the
// `len` of that tile (C chunks of the weight, then stages of 8 adapter pieces).
struct Cursor {
    int ft, rt, i, len;
    int64_t tile0;  // line position of the tile's first item
};
static __device__ __forceinline__ Cursor cursor_at(int64_t w, const int32_t *pre, int RT) {
    Cursor k;
    const int per = pre[RT];
    k.ft = (int)(w / per);
    const int rem = (int)(w - (int64_t)k.ft * per);
    k.rt = 0;
    while (k.rt + 1 < RT && pre[k.rt + 1] <= rem) k.rt++;
    k.i = rem - pre[k.rt];
    k.len = pre[k.rt + 1] - pre[k.rt];
    k.tile0 = w - k.i;
    return k;
}
static __device__ __forceinline__ void next_tile(Cursor &k, const int32_t *pre, int RT) {
    k.tile0 += k.len;
    k.i = 0;
    if (++k.rt == RT) {
        k.rt = 0;
        k.ft++;
    }
    k.len = pre[k.rt + 1] - pre[k.rt];
}

__global__ void __launch_bounds__(kProjectThreads, 1) k_project(const Call c) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(smem);  // [kMaxRing] stage loaded
    uint64_t *empty = full + kMaxRing;                    // [kMaxRing] stage consumed
    uint64_t *tfull = empty + kMaxRing;                   // [2] accumulator set complete
    uint64_t *tempty = tfull + 2;                         // [2] accumulator set read out
    uint64_t *done = tempty + 2;                          // every MMA of the CTA complete
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    int *last_s = reinterpret_cast<int *>(tmem_slot + 1);
    int *fail_s = last_s + 1;                             // [4] wait outcome of each epilogue warp
    int32_t *pre = fail_s + 4;                            // [RT + 1] items before each row tile
    uint8_t *ring = smem + kHeader;
    const int NT = c.NT, C = c.C, S = c.ring;
    const int x_bytes = NT * 256, stage = kItem + x_bytes;
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
            mbar_init(tempty + b, 128);
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
    // Items of each row tile.  With one row tile its adapters are counted here,
    // from the slots themselves (k_prepare passed its wait before this kernel
    // could start, so they are final), and the weights can be fetched before
    // k_prepare ends; with more, k_prepare's counts are waited for.
    if (c.slot && c.RT == 1) {
        TileSlots &ts = *reinterpret_cast<TileSlots *>(ring);
        const RowSlot r = tile_slots(c, 0, ts);
        if (threadIdx.x == 0) {
            pre[0] = 0;
            pre[1] = C + (r.total + 7) / 8;
        }
        // the ring takes this memory over for bulk copies
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    } else {
        if (c.slot) pdl_wait();
        if (threadIdx.x == 0) {
            int n = 0;
            for (int rt = 0; rt < c.RT; rt++) {
                pre[rt] = n;
                n += C + (c.slot ? (__ldcg(c.count + rt) + 7) / 8 : 0);
            }
            pre[c.RT] = n;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int64_t items = (int64_t)c.T * pre[c.RT];
    const int64_t w0 = range_begin(blockIdx.x, items, gridDim.x), w1 = range_begin(blockIdx.x + 1, items, gridDim.x);
    const int n = (int)(w1 - w0);
    const Cursor start = cursor_at(n > 0 ? w0 : 0, pre, c.RT);

    if (warp == 1) {  // ---- loads ---------------------------------------------------
        if (lane == 0) {
            const uint64_t policy = evict_first_policy();
            auto load_weight = [&](const Cursor &k, int s) {  // announces the whole stage
                uint8_t *dst = ring + (size_t)s * stage;
                if (k.i < C) {
                    mbar_expect_tx(full + s, kItem + x_bytes);
                    const uint8_t *src = c.weight + ((size_t)k.ft * C + k.i) * kItem;
                    if (c.RT == 1) bulk_g2s_hint(dst, src, kItem, full + s, policy);  // read once
                    else bulk_g2s(dst, src, kItem, full + s);
                } else {
                    const int p0 = (k.i - C) * 8, np = min(8, __ldcg(c.count + k.rt) - p0);
                    mbar_expect_tx(full + s, np * kPiece + ((np + 1) & ~1) * NT * 32);
                    for (int p = 0; p < np; p++) {
                        const int e = __ldcg(c.list + (size_t)k.rt * c.max_pieces + p0 + p), a = e / c.Q, q = e - a * c.Q;
                        bulk_g2s(dst + p * kPiece, c.up + (((size_t)a * c.T + k.ft) * c.Q + q) * kPiece, kPiece, full + s);
                    }
                }
            };
            auto load_rows = [&](const Cursor &k, int s) {
                uint8_t *dst = ring + (size_t)s * stage + kItem;
                if (k.i < C) {
                    bulk_g2s(dst, c.xp + ((size_t)k.rt * C + k.i) * x_bytes, x_bytes, full + s);
                } else {
                    const int p0 = (k.i - C) * 8, np = min(8, __ldcg(c.count + k.rt) - p0);
                    bulk_g2s(dst, c.tp + ((size_t)k.rt * c.max_pieces + p0) * NT * 32, ((np + 1) & ~1) * NT * 32, full + s);
                }
            };
            // weights of the first stages before k_prepare has finished; adapter
            // stages wait for its lists
            Cursor k = start, kr = start;
            int early = 0;
            while (early < n && early < S && k.i < C) {
                load_weight(k, early);
                early++;
                if (++k.i == k.len) next_tile(k, pre, c.RT);
            }
            pdl_wait();
            asm volatile("fence.proxy.async.global;" ::: "memory");  // k_prepare's stores before the bulk reads
            for (int j = 0; j < early; j++) {
                load_rows(kr, j);
                if (++kr.i == kr.len) next_tile(kr, pre, c.RT);
            }
            bool ok = true;
            int issued = early;
            for (int j = early; j < n; j++) {
                const int s = j % S;
                if (j >= S && !mbar_wait(empty + s, ((j / S) - 1) & 1)) {
                    ok = false;
                    break;
                }
                load_weight(k, s);
                load_rows(k, s);
                issued = j + 1;
                if (++k.i == k.len) next_tile(k, pre, c.RT);
            }
            if (!ok) {
                atomicExch(c.error, 1);
                for (int s = 0; s < S && s < issued; s++) {  // the copies in flight land before the CTA ends
                    const int last = s + ((issued - 1 - s) / S) * S;
                    (void)mbar_wait(full + s, (last / S) & 1);
                }
            }
        }
        __syncwarp();
    } else if (warp == 0) {  // ---- products ---------------------------------------
        if (lane == 0) {
            // [xh | xs] of NT rows each: signed; t's planes one by one, the low one unsigned
            const uint32_t ss2 = umma_idesc_i8(1, 1, 2 * NT), us2 = umma_idesc_i8(0, 1, 2 * NT);
            const uint32_t ss = umma_idesc_i8(1, 1, NT), su = umma_idesc_i8(1, 0, NT), us = umma_idesc_i8(0, 1, NT),
                           uu = umma_idesc_i8(0, 0, NT);
            const uint32_t lbo = NT * 32;
            pdl_wait();  // k_prepare's counts
            Cursor k = start;
            int tiles = 0;
            bool ok = true;
            for (int j = 0; j < n; j++) {
                const bool first = j == 0 || k.i == 0, last = j == n - 1 || k.i == k.len - 1;
                const int b = c.buffers == 2 ? tiles & 1 : 0, use = c.buffers == 2 ? tiles >> 1 : tiles;
                if (first && use > 0 && !mbar_wait(tempty + b, (use - 1) & 1)) ok = false;
                if (ok && !mbar_wait(full + j % S, (j / S) & 1)) ok = false;
                if (!ok) break;
                tc_fence_after();
                const uint32_t wa = smem_u32(ring + (size_t)(j % S) * stage), xa = wa + kItem;
                const uint32_t dh = tmem + (uint32_t)(b * 4 * NT), dl = dh + 2 * NT;
                if (k.i < C) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {  // 32-deep steps: two pieces
                        const uint32_t acc = (first && q == 0) ? 0u : 1u;
                        const uint64_t wh = umma_desc(wa + q * 2 * kPiece, kPiece, 128);
                        const uint64_t wl = umma_desc(wa + q * 2 * kPiece + kPiece / 2, kPiece, 128);
                        const uint64_t x2 = umma_desc(xa + q * 2 * lbo, lbo, 128);
                        umma_i8(dh, wh, x2, ss2, acc);
                        umma_i8(dl, wl, x2, us2, acc);
                    }
                } else {
                    const int np = min(8, __ldcg(c.count + k.rt) - (k.i - C) * 8);
                    for (int q = 0; 2 * q < np; q++) {
                        const uint32_t acc = (first && q == 0) ? 0u : 1u;
                        const uint64_t wh = umma_desc(wa + q * 2 * kPiece, kPiece, 128);
                        const uint64_t wl = umma_desc(wa + q * 2 * kPiece + kPiece / 2, kPiece, 128);
                        const uint64_t th = umma_desc(xa + q * 2 * lbo, lbo, 128);
                        const uint64_t tl = umma_desc(xa + q * 2 * lbo + NT * 16, lbo, 128);
                        umma_i8(dh, wh, th, ss, acc);
                        umma_i8(dh + NT, wh, tl, su, acc);
                        umma_i8(dl, wl, th, us, acc);
                        umma_i8(dl + NT, wl, tl, uu, acc);
                    }
                }
                umma_commit(empty + j % S);
                if (last) {
                    umma_commit(tfull + b);
                    tiles++;
                }
                if (++k.i == k.len) next_tile(k, pre, c.RT);
            }
            if (!ok) atomicExch(c.error, 2);
            umma_commit(done);  // the accumulators are released only after every MMA
            if (!mbar_wait(done, 0)) atomicExch(c.error, 2);
        }
        __syncwarp();
    } else {  // ---- results: warps 2-5, thread m = output m of the tile ---------------------
        const int q4 = warp & 3, m = q4 * 32 + lane;
        Cursor k = start;
        int64_t w = w0;
        for (int tiles = 0; w < w1; tiles++) {
            const int b = c.buffers == 2 ? tiles & 1 : 0, use = c.buffers == 2 ? tiles >> 1 : tiles;
            const int64_t seg1 = min(w1, k.tile0 + k.len);
            const bool whole = w == k.tile0 && seg1 == k.tile0 + k.len;
            const int o = k.ft * kOutTile + m;
            const bool live = o < c.N;
            const int64_t corr = w == k.tile0 ? 128 * (int64_t)c.wsum[o] : 0;
            const int rows = min(NT, (int)c.rows - k.rt * NT);
            const bool okw = mbar_wait_err(tfull + b, use & 1, c.error);
            if (lane == 0) fail_s[q4] = okw ? 0 : 1;
            named_sync(3, 128);
            const int failed = fail_s[0] | fail_s[1] | fail_s[2] | fail_s[3];
            named_sync(3, 128);  // read by all before the next tile writes it
            if (failed) {
                if (m == 0) atomicCAS(c.error, 0, 3);
                break;
            }
            tc_fence_after();
            const uint32_t t0 = tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(b * 4 * NT);
            auto put = [&](int r, int64_t s) {
                const int32_t v = sat32(rnd(s, 4));
                const size_t at = ((size_t)k.rt * NT + r) * c.ld_out + o;
                if (c.wide) static_cast<int32_t *>(c.out)[at] = v;
                else static_cast<int16_t *>(c.out)[at] = (int16_t)sat16(rnd(v, 8));
            };
            int b_lo = 0, b_hi = 0;
            unsigned long long *acc = nullptr;
            if (!whole) {
                b_lo = cta_of(k.tile0, items, gridDim.x);
                b_hi = cta_of(k.tile0 + k.len - 1, items, gridDim.x);
                acc = reinterpret_cast<unsigned long long *>(c.acc) + (size_t)b_lo * NT * kOutTile + m;
            }
            for (int r0 = 0; r0 < rows; r0 += 8) {
                uint32_t v[32];
                tmem_ld4x8(t0 + r0, t0 + NT + r0, t0 + 2 * NT + r0, t0 + 3 * NT + r0, v);
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    if (r0 + r >= rows) break;
                    const int64_t s = (int64_t)(int32_t)v[r] * 65536 +
                                      ((int64_t)(int32_t)v[8 + r] + (int64_t)(int32_t)v[16 + r]) * 256 +
                                      (int64_t)(int32_t)v[24 + r] + corr;
                    if (!whole) atomicAdd(acc + (size_t)(r0 + r) * kOutTile, (unsigned long long)s);
                    else if (live) put(r0 + r, s);
                }
            }
            tc_fence_before();
            mbar_arrive(tempty + b);
            if (!whole) {
                named_sync(3, 128);  // every thread's additions before thread 0's release
                if (m == 0) {
                    int old;
                    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;"
                                 : "=r"(old)
                                 : "l"(c.arrived + b_lo)
                                 : "memory");
                    *last_s = old == b_hi - b_lo;
                }
                named_sync(3, 128);
                const int finish = *last_s;
                if (finish) {
                    for (int r0 = 0; r0 < rows; r0 += 8) {
                        int64_t s[8];
#pragma unroll
                        for (int r = 0; r < 8; r++)
                            s[r] = r0 + r < rows ? (int64_t)__ldcg(acc + (size_t)(r0 + r) * kOutTile) : 0;
#pragma unroll
                        for (int r = 0; r < 8; r++) {
                            if (r0 + r >= rows) break;
                            acc[(size_t)(r0 + r) * kOutTile] = 0;  // ready for the next call
                            if (live) put(r0 + r, s[r]);
                        }
                    }
                    if (m == 0) c.arrived[b_lo] = 0;
                }
            }
            w = seg1;
            next_tile(k, pre, c.RT);
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
// dst + (t * pieces + p) * kPiece as [plane][row][16 bytes], zeros past the matrix.
__global__ void k_pack_pieces(const int16_t *__restrict__ src, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t pieces,
                              uint32_t stride_pieces, uint32_t tiles, uint8_t *__restrict__ dst) {
    const uint64_t total = (uint64_t)tiles * pieces * kOutTile;
    for (uint64_t g = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; g < total; g += (uint64_t)gridDim.x * blockDim.x) {
        const uint32_t m = (uint32_t)(g % kOutTile);
        const uint64_t rest = g / kOutTile;
        const uint32_t p = (uint32_t)(rest % pieces), t = (uint32_t)(rest / pieces), row = t * kOutTile + m;
        uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
        if (row < rows)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t col = p * 16 + e;
                const uint32_t v = col < cols ? (uint16_t)src[(size_t)row * ld + col] : 0u;
                hi[e >> 2] |= (v >> 8) << (8 * (e & 3));
                lo[e >> 2] |= (v & 255u) << (8 * (e & 3));
            }
        uint8_t *d = dst + ((size_t)t * stride_pieces + p) * kPiece + m * 16;
        *reinterpret_cast<uint4 *>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(d + kPiece / 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}
// Sum of every output's weights (|sum| <= 2^15 * 32768: 32 bits hold it), 0 past the last output.
__global__ void __launch_bounds__(256) k_weight_sums(const int16_t *__restrict__ src, uint32_t rows, uint32_t cols,
                                                     uint32_t padded, int32_t *__restrict__ sums) {
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= padded) return;
    int32_t s = 0;
    if (row < rows)
        for (uint32_t k = lane; k < cols; k += 32) s += src[(size_t)row * cols + k];
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (lane == 0) sums[row] = s;
}
// down [rank][K] -> words {lo(w0), lo(w1), hi(w0), hi(w1)} for the dp2a products
__global__ void k_pack_down(const uint32_t *__restrict__ src, uint32_t words, uint32_t *__restrict__ dst) {
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < words; i += gridDim.x * blockDim.x)
        dst[i] = __byte_perm(src[i], 0, 0x3120);
}
__global__ void k_set_slot(int32_t *ranks, int32_t *scales, uint32_t slot, int32_t rank, int32_t scale) {
    ranks[slot] = rank;
    scales[slot] = scale;
}

// Rows per row tile of a call: as few row tiles as 128 rows each allow, evenly
// filled, in steps of 16 (the MMA's column granularity).
int row_tiles(uint32_t rows) { return (int)((rows + kRowTile - 1) / kRowTile); }
int rows_per_tile(uint32_t rows) {
    const uint32_t rt = (uint32_t)row_tiles(rows);
    return (int)(((rows + rt - 1) / rt + 15) / 16 * 16);
}

}  // namespace

struct llmx_adapters {
    int dev = 0, sms = 0, smem = 0;
    uint32_t in_dim = 0, out_dim = 0, slots = 0, max_rank = 0, max_rows = 0;
    int C = 0, T = 0, Q = 0, row_cap = 0;  // row_cap: most rows per row tile of any call
    uint8_t *weight = nullptr;   // items [T][C]
    int32_t *wsum = nullptr;     // [T * 128]
    uint32_t *down = nullptr;    // [slots][16 Q][in_dim / 2]
    uint8_t *up = nullptr;       // pieces [slots][T][Q]
    int32_t *rank = nullptr, *scale = nullptr;  // [slots]
    uint8_t *xp = nullptr, *tp = nullptr;       // row and t pieces of a call
    int32_t *list = nullptr, *count = nullptr;  // adapter pieces of its row tiles
    int64_t *acc = nullptr;
    int32_t *arrived = nullptr;
    int *error = nullptr;
    uint64_t bytes = 0;

    size_t max_pieces(int nt) const {  // of one row tile, even
        const size_t n = std::min<size_t>((size_t)nt, slots) * Q;
        return (n + 1) / 2 * 2;
    }
    size_t acc_bytes() const { return (size_t)sms * row_cap * kOutTile * 8; }
};

namespace {

int fail(int code, const std::string &msg) {
    set_last_error("adapters: " + msg);
    return code;
}
int cuda_fail(const char *what, cudaError_t e) {
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
    for (void *p : {(void *)h->weight, (void *)h->wsum, (void *)h->down, (void *)h->up, (void *)h->rank, (void *)h->scale,
                    (void *)h->xp, (void *)h->tp, (void *)h->list, (void *)h->count, (void *)h->acc, (void *)h->arrived,
                    (void *)h->error})
        cudaFree(p);
    delete h;
}

cudaError_t launch(const void *fn, int grid, int threads, size_t smem, const Call &c, cudaStream_t s) {
    Call copy = c;
    void *args[] = {&copy};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
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
    h->C = (int)((in_dim + kOutTile - 1) / kOutTile);
    h->T = (int)((out_dim + kOutTile - 1) / kOutTile);
    h->Q = (int)((h->max_rank + 15) / 16);
    h->row_cap = max_rows > kRowTile ? kRowTile : rows_per_tile(max_rows);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto get = [&](auto **p, size_t n) {
        n = std::max<size_t>(n, 16);
        h->bytes += n;
        return cudaMalloc(reinterpret_cast<void **>(p), n);
    };
    const size_t rt = (size_t)row_tiles(max_rows), up_bytes = (size_t)slots * h->T * h->Q * kPiece;
    const size_t pieces = h->max_pieces(h->row_cap);
    cudaError_t e;
    if ((e = cudaDeviceGetAttribute(&h->sms, cudaDevAttrMultiProcessorCount, device)) != cudaSuccess ||
        (e = cudaDeviceGetAttribute(&h->smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, device)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(k_project, cudaFuncAttributeMaxDynamicSharedMemorySize, h->smem)) != cudaSuccess ||
        (e = get(&h->weight, (size_t)h->T * h->C * kItem)) != cudaSuccess ||
        (e = get(&h->wsum, (size_t)h->T * kOutTile * 4)) != cudaSuccess ||
        (e = get(&h->down, (size_t)slots * h->Q * 16 * in_dim * 2)) != cudaSuccess ||
        (e = get(&h->up, up_bytes)) != cudaSuccess || (e = get(&h->rank, (size_t)slots * 4)) != cudaSuccess ||
        (e = get(&h->scale, (size_t)slots * 4)) != cudaSuccess ||
        (e = get(&h->xp, rt * h->C * h->row_cap * 256)) != cudaSuccess ||
        (e = get(&h->tp, rt * pieces * h->row_cap * 32)) != cudaSuccess || (e = get(&h->list, rt * pieces * 4)) != cudaSuccess ||
        (e = get(&h->count, rt * 4)) != cudaSuccess || (e = get(&h->acc, h->acc_bytes())) != cudaSuccess ||
        (e = get(&h->arrived, (size_t)h->sms * 4)) != cudaSuccess || (e = get(&h->error, 4)) != cudaSuccess ||
        (e = cudaMemsetAsync(h->rank, 0, (size_t)slots * 4, s)) != cudaSuccess ||
        // the last ranks of a slot that no adapter fills are multiplied by nothing, but read
        (e = cudaMemsetAsync(h->down, 0, (size_t)slots * h->Q * 16 * in_dim * 2, s)) != cudaSuccess ||
        (e = cudaMemsetAsync(h->acc, 0, h->acc_bytes(), s)) != cudaSuccess ||
        (e = cudaMemsetAsync(h->arrived, 0, (size_t)h->sms * 4, s)) != cudaSuccess ||
        (e = cudaMemsetAsync(h->error, 0, 4, s)) != cudaSuccess) {
        release(h);
        return cuda_fail("create", e);
    }
    k_pack_pieces<<<h->sms * 8, 256, 0, s>>>(weight, out_dim, in_dim, in_dim, h->C * 8, h->C * 8, h->T, h->weight);
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
        const uint32_t words = rank * h->in_dim / 2, used = (rank + 15) / 16;
        k_pack_down<<<256, 256, 0, s>>>(reinterpret_cast<const uint32_t *>(down), words,
                                        h->down + (size_t)slot * h->Q * 16 * (h->in_dim / 2));
        k_pack_pieces<<<h->sms * 4, 256, 0, s>>>(up, h->out_dim, rank, rank, used, h->Q, h->T,
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
    c.C = h->C;
    c.T = h->T;
    c.N = (int)h->out_dim;
    c.RT = row_tiles(rows);
    c.NT = rows_per_tile(rows);
    c.slots = (int)h->slots;
    c.Q = h->Q;
    c.max_pieces = (int)h->max_pieces(c.NT);
    c.down_words = (int)(h->in_dim / 2);
    c.weight = h->weight;
    c.wsum = h->wsum;
    c.up = h->up;
    c.down = h->down;
    c.rank = h->rank;
    c.scale = h->scale;
    c.xp = h->xp;
    c.tp = h->tp;
    c.list = h->list;
    c.count = h->count;
    c.acc = h->acc;
    c.arrived = h->arrived;
    c.error = h->error;
    c.buffers = c.NT <= 64 ? 2 : 1;  // 4 sums x NT columns each, 512 in all
    const int stage = kItem + c.NT * 256;
    c.ring = std::min(kMaxRing, (h->smem - kHeader) / stage);
    const int grid = (int)std::min<int64_t>(h->sms, (int64_t)c.T * c.RT * c.C);
    const int64_t blocks = (int64_t)c.RT * c.C + (c.slot ? c.RT + (int64_t)rows * c.Q : 0);
    cudaError_t e = launch((const void *)k_prepare, (int)blocks, kPrepareThreads, 0, c, s);
    if (e == cudaSuccess)
        e = launch((const void *)k_project, grid, kProjectThreads, kHeader + (size_t)c.ring * stage, c, s);
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
