// Verification of drafted tokens against the target's probabilities, from
// random numbers that the caller gives.
//
// No counterpart in the LLM-ACCEL tree: its host decodes greedily
// (lm_head_argmax, host/host_qwen_8x64.cpp:937-977) and never forms
// probabilities.  The arithmetic follows the path's rule that a result is a
// whole number which no order of summation can change: a logit becomes a
// 32-bit weight, sums of weights are 64-bit integers, probabilities are Q0.40
// integers, and both the accept test and the draw compare integers.
//
// Two launches.  k_mass reduces every row of logits to its maximum and its
// sum of weights.  A weight depends on the row's maximum, so a row is read
// twice, by a cluster of CTAs that exchange their maxima through shared memory.  With
// few rows, for latency, a cluster is so large that it holds a row in
// shared memory between the passes.  With many it is small, and some of its warps
// take the rows' first passes while the others follow a row or two behind with the
// second, whose chunks come again, mostly from L2: neither waits for an exchange or for
// the other's loads.  k_draw tests the drafts of a request and draws its last
// token, a cluster per request.
//
// What bounds it (B200, vocabulary of 151936, in graphs of calls over three sets of
// inputs; 156 to 164 us for the first by machine).  64 requests x 7 drafts with draft rows, 960 rows,
// 583 MB: 156 us against 90 for the bytes; k_mass 120 (0.6 GB read: second loads leave the L2
// first; 19 instructions a logit of both passes, 0.68 a cycle and scheduler), k_draw 32 to 40 (70
// MB, 0.60 instructions a cycle).  64 requests without drafts: 36.8 us against 6, three passes over
// a row, none of them at a limit of the machine (under ncu 20.5 in k_mass and 24.5 in
// k_draw, 0.48 and 0.57 instructions a cycle, DRAM at a fifth).  One request with 4 copied
// drafts: 11.6 us, latency: 4.8 in k_mass, then accept tests 1.5, sums 2.9, cluster totals
// 0.6, the token 1.0, the cluster's end 0.3.  Simple kernels, a block per row and per request, took 862 and 194 us.
//
// Waits are bounded.  A warp that gives one up takes part in nothing after it: no maximum, sum or
// slot is passed on from it, so whatever needs them gives up as well, and a row or
// request is either exact or marked.  CTAs end when their copies have landed and their cluster
// sends nothing more (0.3 to 0.9 us of a call).
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <mutex>
#include <string>
#include <type_traits>

#include "llmx.h"
#include "device_util.cuh"
#include "cluster.cuh"
#include "gemv_common.cuh"
#include "kernels.cuh"

namespace {

using llmx::arrive_remote;
using llmx::bulk_g2s;
using llmx::bulk_g2s_hint;
using llmx::cluster_arrive;
using llmx::cluster_leave;
using llmx::cluster_rank;
using llmx::cluster_wait;
using llmx::let_land;
using llmx::mbar_arrive;
using llmx::mbar_expect_tx;
using llmx::mbar_init;
using llmx::mbar_test_cluster;
using llmx::mbar_wait;
using llmx::mbar_wait_cluster;
using llmx::pdl_trigger;
using llmx::pdl_wait;
using llmx::remote;
using llmx::smem_u32;
using llmx::st_async;

constexpr int kExcluded = INT_MIN;
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr uint32_t kMaxVocab = 1u << 22, kMaxRequests = 65535, kMaxDrafts = 1023, kMaxTotal = 1u << 24;
constexpr float kMinTemperature = 1e-6f;     // at or below: greedy
constexpr float kLog2e16 = 0x1.715476p-16f;  // log2(e) / 2^16: Q16.16 differences to octaves
constexpr int kMaxCluster = 16;

// What a row of logits is reduced to, as k_mass leaves it: every CTA of the
// row's cluster writes its part, the sum of its weights or (greedy) the first
// position of the maximum in its share (kNoToken: not there).
constexpr unsigned long long kGaveUp = ~1ull;   // a wait of the CTA ran out
struct RowPart {
    int32_t top;
    float scale;  // log2(e) / 2^16 / T; negative: greedy
    unsigned long long pad;
    unsigned long long part[kMaxCluster];
};

struct Args {
    const int32_t *target, *draft;
    size_t ld_target, ld_draft;
    uint32_t vocab, requests, drafts, max_drafts;
    const uint32_t *draft_tokens, *offsets;
    const float *temperature;
    const uint32_t *accept_u, *sample_u;
    uint32_t *tokens, *accepted;
    uint64_t *probs;
    RowPart *rows;   // [drafts + requests] target rows, then [drafts] draft rows
    uint32_t total;  // rows
    int split;       // CTAs per row (k_mass), and of a cluster there
    int ring;        // chunks of shared memory per CTA
    int resident;    // the ring holds a CTA's share of a row: it is loaded once
    uint32_t polls;  // of a wait, except for what has to land before a CTA ends
};

// ---- arithmetic -------------------------------------------------------------------
// Offsets of request b; false when they are not a range of at most max_drafts
// within [0, drafts].
static __device__ __forceinline__ bool request_range(const Args &a, uint32_t b, uint32_t &begin, uint32_t &count) {
    begin = a.offsets[b];
    const uint32_t end = a.offsets[b + 1];
    count = end - begin;
    return begin <= end && end <= a.drafts && count <= a.max_drafts;
}
static __device__ __forceinline__ float row_scale(float temperature) {
    return temperature > kMinTemperature ? __fdiv_rn(kLog2e16, temperature) : -1.0f;
}

using f32x2 = unsigned long long;
static __device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
static __device__ __forceinline__ void unpack2(f32x2 v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
// Products of pairs one by one: a packed mul.rn is fused by the compiler with the packed
// addition that follows it, and the weights would differ in their last bits; a scalar
// product and a packed sum it cannot fuse. (A packed fma with a -0 that the compiler
// cannot see through is as exact: 64 requests x 7 drafts 162 us against 155.)
static __device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    float a0, a1, b0, b1;
    unpack2(a, a0, a1);
    unpack2(b, b0, b1);
    return pack2(__fmul_rn(a0, b0), __fmul_rn(a1, b1));
}
static __device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
static __device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// floor(2^31 * 2^-e), e = (top - z) * scale capped at 100, of the logits of one
// row.  Every float step of the definition is rounded on its own, so that the
// weight is the same integer wherever it is computed.
//   2^x = 2^round(x) 2^f, and 2^f on [-1/2, 1/2] is 1 + f q(f), q of degree 4 fitted
// to the relative error at Chebyshev points: below 2e-7 with the rounding of its
// steps.  Here x = -e; adding 1.5 * 2^23 rounds it to the nearest whole number
// (even at ties) and leaves that number in the low bits, from where one shifted
// addition puts it into the exponent.  The coefficients carry the 2^31.  Packed
// pairs halve the sums' instructions; a row's second pass spends most of its time on these steps.
//   The usual row (fast) needs no conversion to float: with d = top - z below
// 2^23, the bits of 2^23 + d are 0x4b000000 + d, and (2^23 + d) (-scale) + 2^23 scale in one
// fused step is d (-scale) rounded once (2^23 scale is exact).  A d of 32 / scale
// or more has a weight of 0, as has any larger one, so d is cut there in
// whole numbers; that needs 32 / scale < 2^23 (T below 5.7) and a maximum so low
// that 0x4b000000 + d cannot pass 2^32.  The other rows convert and cap as defined.
struct RowWeight {
    int32_t top;
    float scale;
    bool greedy, fast, test;  // test: an excluded logit is not far enough below the maximum to vanish by itself
    uint32_t base, most;      // fast: 0x4b000000 + top, 0x4b000000 + the largest d
    f32x2 minus_scale, shift;

    __device__ __forceinline__ void set(int32_t t, float s) {
        top = t;
        scale = s;
        greedy = s < 0.0f;
        test = !(__fmul_rn(__uint2float_rn((uint32_t)t - (uint32_t)kExcluded), s) >= 33.0f);
        const float limit = __fdiv_rn(32.0f, s);
        fast = !greedy && !test && limit < 8388000.0f && t < 889192448;
        base = 0x4b000000u + (uint32_t)t;
        most = 0x4b000000u + (fast ? __float2uint_ru(limit) : 0u);
        minus_scale = pack2(-s, -s);
        shift = pack2(8388608.0f * s, 8388608.0f * s);
    }
    // the second half, from x = -e
    __device__ __forceinline__ void finish(f32x2 x, uint32_t &w0, uint32_t &w1) const {
        const f32x2 magic = pack2(12582912.0f, 12582912.0f), minus_magic = pack2(-12582912.0f, -12582912.0f);
        const f32x2 m = add2(x, magic), f = fma2(add2(m, minus_magic), pack2(-1.0f, -1.0f), x);
        f32x2 p = add2(mul2(f, pack2(0x1.5bba12p21f, 0x1.5bba12p21f)), pack2(0x1.3cea88p24f, 0x1.3cea88p24f));
        p = add2(mul2(p, f), pack2(0x1.c6b752p26f, 0x1.c6b752p26f));
        p = add2(mul2(p, f), pack2(0x1.ebf9bcp28f, 0x1.ebf9bcp28f));
        p = add2(mul2(p, f), pack2(0x1.62e42ap30f, 0x1.62e42ap30f));
        p = add2(mul2(p, f), pack2(0x1p31f, 0x1p31f));
        float m0, m1, p0, p1;
        unpack2(m, m0, m1);
        unpack2(p, p0, p1);
        w0 = __float2uint_rz(__int_as_float(__float_as_int(p0) + (__float_as_int(m0) << 23)));
        w1 = __float2uint_rz(__int_as_float(__float_as_int(p1) + (__float_as_int(m1) << 23)));
    }
    __device__ __forceinline__ void fast2(int32_t z0, int32_t z1, uint32_t &w0, uint32_t &w1) const {
        const uint32_t d0 = min(base - (uint32_t)z0, most), d1 = min(base - (uint32_t)z1, most);
        finish(fma2(pack2(__uint_as_float(d0), __uint_as_float(d1)), minus_scale, shift), w0, w1);
    }
    __device__ __forceinline__ void slow2(int32_t z0, int32_t z1, uint32_t &w0, uint32_t &w1) const {
        float x0 = __uint2float_rn((uint32_t)top - (uint32_t)z0), x1 = __uint2float_rn((uint32_t)top - (uint32_t)z1);
        unpack2(mul2(pack2(x0, x1), minus_scale), x0, x1);
        finish(pack2(fmaxf(x0, -100.0f), fmaxf(x1, -100.0f)), w0, w1);
        w0 = z0 == kExcluded ? 0u : w0;
        w1 = z1 == kExcluded ? 0u : w1;
    }
};

// A row's numbers as k_draw uses them.
struct RowMass {
    int32_t top;
    float scale;
    uint32_t first;    // greedy: the maximum's first position
    uint32_t inverse;  // floor(2^62 / (S >> h)), 0 when nothing is left
    int32_t shift;     // 22 + h
    int ok;
};
// Sum over the warp, below 2^59: two 32-bit reductions take less than five rounds of
// 64-bit shuffles.
static __device__ __forceinline__ unsigned long long sum_lanes(unsigned long long v) {
    const uint32_t lo = __reduce_add_sync(~0u, (uint32_t)v & 0x7ffffffu), hi = __reduce_add_sync(~0u, (uint32_t)(v >> 27));
    return ((unsigned long long)hi << 27) + lo;
}
// From the parts of a row, by half a warp: its lanes hold a part each.
static __device__ RowMass load_row(const RowPart *rows, uint32_t row, int split) {
    const int i = threadIdx.x & (kMaxCluster - 1);
    const RowPart *p = rows + row;
    RowMass r;
    unsigned long long v = i < split ? p->part[i] : 0;
    r.top = p->top;
    r.scale = p->scale;
    const bool greedy = r.scale < 0.0f;
    r.ok = !(i < split && v == kGaveUp);
    uint32_t first = greedy && i < split ? (uint32_t)v : kNoToken;
    if (greedy) v = 0;
    for (int o = kMaxCluster / 2; o; o >>= 1) {
        v += __shfl_xor_sync(~0u, v, o);
        first = min(first, __shfl_xor_sync(~0u, first, o));
        r.ok &= __shfl_xor_sync(~0u, r.ok, o);
    }
    r.first = first;
    const unsigned long long sum = greedy ? (r.top != kExcluded && first != kNoToken ? 1ull << 31 : 0) : v;
    int h = 32 - __clzll((long long)sum);  // sum has 64 - clz bits; 32 remain
    h = h < 0 ? 0 : h;
    r.inverse = sum ? (uint32_t)((1ull << 62) / (sum >> h)) : 0u;
    r.shift = 22 + h;
    return r;
}
static __device__ __forceinline__ void row_weight2(const RowWeight &w, uint32_t first, int32_t z0, int32_t z1, uint32_t v0,
                                                   uint32_t v1, uint32_t &w0, uint32_t &w1) {
    if (w.fast) {
        w.fast2(z0, z1, w0, w1);
    } else if (w.greedy) {
        w0 = v0 == first && z0 != kExcluded ? 0x80000000u : 0u;
        w1 = v1 == first && z1 != kExcluded ? 0x80000000u : 0u;
    } else {
        w.slow2(z0, z1, w0, w1);
    }
}
static __device__ __forceinline__ uint64_t row_share(uint32_t w, const RowMass &r) {
    return ((uint64_t)w * r.inverse) >> r.shift;
}
// The same for shifts below 32 (a sum of weights below 2^42: the usual row).
static __device__ __forceinline__ uint64_t row_share_small(uint32_t w, const RowMass &r) {
    const uint64_t v = (uint64_t)w * r.inverse;
    const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    return ((uint64_t)(hi >> r.shift) << 32) | __funnelshift_r(lo, hi, r.shift);
}
// floor(a * u / 2^32)
static __device__ __forceinline__ uint64_t mul_frac(uint64_t a, uint32_t u) { return __umul64hi(a, (uint64_t)u << 32); }

// ---------------------------------------------------------------------------
// rows -> maxima and sums
// ---------------------------------------------------------------------------
constexpr int kMassWarps = 16;              // that sum
constexpr int kChunk = 4096;                // logits per chunk
constexpr int kChunkBytes = kChunk * 4;
constexpr int kMaxRing = 12, kFirstRing = 4;  // chunks in shared memory; of these the first pass's, where it has its own
constexpr int kFirstWarps = 4;              // of a first pass of its own
constexpr int kTops = 2;                    // rows whose maxima may be under way
static __host__ __device__ constexpr int mass_threads(bool twice) { return (kMassWarps + (twice ? kFirstWarps : 0) + 3) * 32; }

// A row's logits: a head of at most 3 up to a 16-byte boundary, vectors of 4, a
// tail of at most 3.  CTA `rank` of `split` takes an even share of the
// vectors; the first has the head too, the last the tail.
struct Row {
    const int32_t *z;
    uint32_t head, vectors, v0, v1;
    __device__ __forceinline__ Row(const Args &a, uint32_t row, int rank) {
        const uint32_t targets = a.drafts + a.requests;
        z = row < targets ? a.target + row * a.ld_target : a.draft + (row - targets) * a.ld_draft;
        head = min(a.vocab, (uint32_t)((16 - ((uintptr_t)z & 15)) & 15) >> 2);
        vectors = (a.vocab - head) >> 2;
        v0 = vectors * rank / a.split;  // below 2^20 * 16
        v1 = vectors * (rank + 1) / a.split;
    }
};

// The request that a row belongs to, by a warp: a 32-way search in the offsets,
// checked; where they are not in order, the first request that claims the row.
static __device__ uint32_t owner_of(const Args &a, uint32_t row) {
    const int lane = threadIdx.x & 31;
    const uint32_t targets = a.drafts + a.requests;
    const bool is_draft = row >= targets;
    if (is_draft) row -= targets;
    auto claims = [&](uint32_t b) {
        uint32_t begin, count;
        if (!request_range(a, b, begin, count)) return false;
        const uint32_t lo = is_draft ? begin : begin + b, n = is_draft ? count : count + 1;
        return row >= lo && row - lo < n;
    };
    // the last b whose first row is not above `row`: among equal starts (requests
    // without drafts have no draft rows) the last has the draft rows
    uint32_t lo = 0, n = a.requests;  // b in [lo, lo + n)
    while (n > 1) {
        const uint32_t step = (n + 31) / 32, b = lo + lane * step;
        const bool not_above = lane * step < n && (is_draft ? a.offsets[b] : a.offsets[b] + b) <= row;
        const unsigned m = __ballot_sync(~0u, not_above);
        const int last = m ? 31 - __clz(m) : 0;
        n = min(step, n - last * step);
        lo += last * step;
    }
    if (claims(lo)) return lo;
    for (uint32_t b0 = 0; b0 < a.requests; b0 += 32) {
        const unsigned m = __ballot_sync(~0u, b0 + lane < a.requests && claims(b0 + lane));
        if (m) return b0 + __ffs((int)m) - 1;
    }
    return kNoToken;
}

// A CTA's part in a row, and a thread's logit of its head or tail, if any.
struct Held {
    Row r;
    int chunks;
    uint32_t edge_at;
    int32_t edge;
    __device__ __forceinline__ Held(const Args &a, uint32_t row, int rank, int t) : r(a, row, rank) {
        chunks = (int)((r.v1 - r.v0 + kChunk / 4 - 1) / (kChunk / 4));
        edge_at = kNoToken;
        edge = kExcluded;
        const uint32_t tail = r.head + r.vectors * 4;
        if (t < 3 && rank == 0 && t < (int)r.head) edge_at = t;
        if (t >= 4 && t < 7 && rank == a.split - 1 && tail + t - 4 < a.vocab) edge_at = tail + t - 4;
        if (edge_at != kNoToken) edge = r.z[edge_at];
    }
};

// Warps of a CTA: the first kMassWarps sum; kTwice: kFirstWarps more take the
// maxima, through a ring of their own (slots [0, kFirstRing)), else the summing
// warps do, and a row stays in the one ring until it is summed; then two that load
// and one that finds the rows' temperatures.
// No barrier over the CTA: the last warp to add its maximum (or sum) passes
// the CTA's on.  The maxima of the cluster arrive in one of kTops places; a CTA
// sends row i + kTops's once every CTA of the cluster has summed row i (top_done),
// which also keeps the words that its warps share apart: they alternate between rows.
// A chunk is one group's of GW summing warps.
template <bool kTwice, int GW>
__global__ void __launch_bounds__(mass_threads(kTwice), 1) k_mass(const Args a) {
    constexpr int kGroups = kMassWarps / GW;
    constexpr int kMaxWarps = kTwice ? kFirstWarps : kMassWarps;  // that take maxima
    constexpr int kLoad = kMassWarps + (kTwice ? kFirstWarps : 0);
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t full[kMaxRing], empty[kMaxRing];
    __shared__ uint64_t info_full[2], info_empty[2];      // a row's temperature
    __shared__ uint64_t top_full[kTops], top_done[kTops]; // of every CTA: its maximum of the row is there, its sum done
    __shared__ float scale_s[2];
    __shared__ int32_t tops[kTops][kMaxCluster];
    __shared__ int32_t warp_top[2][kMassWarps];
    __shared__ unsigned long long warp_part[2][kMassWarps];
    __shared__ int top_count[2], part_count[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = a.split, rank = S > 1 ? (int)cluster_rank() : 0;
    const uint32_t group = blockIdx.x / S, groups = gridDim.x / S;
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.ring; i++) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, kTwice && i < kFirstRing ? kFirstWarps : GW);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(info_full + i, 1);
            mbar_init(info_empty + i, kMassWarps);
            top_count[i] = part_count[i] = 0;
        }
        for (int i = 0; i < kTops; i++) {
            mbar_init(top_full + i, 1);
            mbar_init(top_done + i, S);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (S > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    pdl_wait();
    // with many rows the draw's CTAs would only take room from the last of this kernel's
    if (!kTwice) pdl_trigger();

    // Every warp's end; true where a warp of the CTA gave up.  Where none did, all that was on its way
    // to the CTA has been waited for.
    auto leave = [&](bool came) {
        __syncwarp();
        const bool lost = __syncthreads_or(!came);
        if (S > 1) {
            cluster_arrive();
            cluster_leave(!lost);
        }
        return lost;
    };
    if (warp >= kLoad && warp < kLoad + 2) {  // ---- loads, of the first pass and of the second -----
        int base = 0, ring = 1, issued = 0;
        bool ok = true;
        if (lane == 0 && (kTwice || warp == kLoad)) {
            base = warp == kLoad ? 0 : kFirstRing;
            ring = !kTwice ? a.ring : warp == kLoad ? kFirstRing : a.ring - kFirstRing;
            const uint64_t policy = llmx::evict_first_policy();
            int s = 0, phase = 1;
            for (uint32_t row = group; ok && row < a.total; row += groups) {
                const Row r(a, row, rank);
                for (uint32_t v = r.v0; v < r.v1; v += kChunk / 4) {
                    const int at = base + s;
                    if (issued >= ring && !mbar_wait(empty + at, phase, a.polls)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bytes = min(r.v1 - v, (uint32_t)kChunk / 4) * 16;
                    mbar_expect_tx(full + at, bytes);
                    const int32_t *src = r.z + r.head + (size_t)v * 4;
                    if (base == 0) bulk_g2s(smem + at * kChunkBytes, src, bytes, full + at);
                    else bulk_g2s_hint(smem + at * kChunkBytes, src, bytes, full + at, policy);  // not needed again
                    issued++;
                    if (++s == ring) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        if (leave(ok))  // the copies in flight land before the CTA ends, which warp of it gave up ever
            for (int q = 0; q < ring && q < issued; q++) {
                const int last = q + ((issued - 1 - q) / ring) * ring;
                (void)mbar_wait(full + base + q, (last / ring) & 1);
            }
        return;
    }
    if (warp == kLoad + 2) {  // ---- the rows' temperatures --------------------------
        uint32_t i = 0;
        for (uint32_t row = group; row < a.total; row += groups, i++) {
            const uint32_t b = owner_of(a, row);
            const float scale = b == kNoToken ? -1.0f : row_scale(a.temperature[b]);
            if (i >= 2 && !__all_sync(~0u, mbar_wait(info_empty + (i & 1), ((i >> 1) - 1) & 1, a.polls))) break;
            if (lane == 0) {
                scale_s[i & 1] = scale;
                mbar_arrive(info_full + (i & 1));
            }
            __syncwarp();
        }
        leave(true);
        return;
    }

    // ---- maxima and sums ---------------------------------------------------------------
    bool ok = true;
    uint32_t row = group;
    // A place in a ring of n slots from slot `base` on, moved by chunks.  Slot s is always
    // group s mod kGroups's (n is a multiple of kGroups): a warp then meets every phase of the
    // barriers that it waits on, and cannot take an older phase for the one it needs.
    struct Place {
        int at, phase, base, n;
        __device__ __forceinline__ void move(int by) {
            at += by;
            while (at >= n) {
                at -= n;
                phase ^= 1;
            }
        }
        __device__ __forceinline__ int slot() const { return base + at; }
        // moves to the group's first chunk from here on, and says how far that is
        __device__ __forceinline__ int own(int group) {
            const int by = (group + kGroups - at % kGroups) % kGroups;
            move(by);
            return by;
        }
    };
    static_assert((kMaxRing - kFirstRing) % kGroups == 0 && kMaxRing % kGroups == 0, "a slot is one group's");
    // whether this warp, whose lane 0 has just written its word, is the last of n to
    // come here; it then sees the others' words
    auto last_of = [&](int *count, int n) {
        int old = 0;
        if (lane == 0) {
            asm volatile("atom.acq_rel.cta.shared::cta.add.s32 %0, [%1], 1;" : "=r"(old) : "r"(smem_u32(count)) : "memory");
            if (old == n - 1) *count = 0;
        }
        return __shfl_sync(~0u, old, 0) == n - 1;
    };
    auto arrive_all = [&](uint64_t *bar) {  // on this barrier of every CTA of the cluster
        if (lane < S) arrive_remote(remote(bar, lane));
    };
    // (a slot whose chunk was not waited for to the end stays this warp's: it may still be filled)
    auto release = [&](int at) {
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(empty + at);
    };
    int32_t top = kExcluded;  // of the row in its first pass
    // thread t of `stride` takes its vectors of a chunk
    auto first_chunk = [&](const Row &r, int at, int c, int t, auto stride) {
        constexpr int kStride = decltype(stride)::value, kVectors = kChunk / 4 / kStride;
        const int4 *p = reinterpret_cast<const int4 *>(smem + at * kChunkBytes) + t;
        const int n = (int)min(r.v1 - r.v0 - c * (kChunk / 4), (uint32_t)kChunk / 4) - t;
        auto most = [&](const int4 &q) { top = max(max(top, q.x), max(max(q.y, q.z), q.w)); };
        if ((kVectors - 1) * kStride < n) {
#pragma unroll
            for (int u = 0; u < kVectors; u++) most(p[u * kStride]);
        } else {
            for (int u = 0; u * kStride < n; u++) most(p[u * kStride]);
        }
    };
    // row number i's maximum, sent to every CTA of the cluster
    auto send_top = [&](uint32_t i, int32_t edge, int w) {
        top = __reduce_max_sync(~0u, max(top, edge));
        // every warp waits, not the last alone: else one could go on two rows and be counted
        // in a row that others have not reached
        if (i >= kTops) ok = ok && mbar_wait_cluster(top_done + i % kTops, (i / kTops - 1) & 1, a.polls);
        // a warp that gave up counts in nothing any more: what it has no part in is never sent, and
        // all that need it give up too
        ok = __all_sync(~0u, ok);
        if (!ok) return;
        if (lane == 0) warp_top[i & 1][w] = top;
        if (last_of(&top_count[i & 1], kMaxWarps)) {
            top = __reduce_max_sync(~0u, lane < kMaxWarps ? warp_top[i & 1][lane] : kExcluded);
            // (without a cluster there is no asynchronous store, not even to the CTA itself)
            if (S == 1) {
                if (lane == 0) {
                    tops[i % kTops][0] = top;
                    mbar_arrive(top_full + i % kTops);
                }
            } else if (lane == 0) {
                mbar_expect_tx(top_full + i % kTops, S * 4);
            }
            if (S > 1 && lane < S) st_async(remote(&tops[i % kTops][rank], lane), top, remote(top_full + i % kTops, lane));
        }
        top = kExcluded;
        __syncwarp();
    };
    if (kTwice && warp >= kMassWarps) {  // ---- first passes of their own ---------------------
        const int w = warp - kMassWarps, t = w * 32 + lane;
        Place p{0, 0, 0, kFirstRing};
        uint32_t i = 0;
        for (; ok && row < a.total; row += groups, i++) {
            const Held h(a, row, rank, t);
            for (int c = 0; c < h.chunks; c++, p.move(1)) {
                ok = ok && mbar_wait(full + p.slot(), p.phase, a.polls);
                first_chunk(h.r, p.slot(), c, t, std::integral_constant<int, kFirstWarps * 32>());
                release(p.slot());
            }
            send_top(i, h.edge, w);
            if (!ok) break;
        }
    } else {
        const int mine = warp / GW, gt = (warp % GW) * 32 + lane;
        const uint32_t count = group < a.total ? (a.total - group + groups - 1) / groups : 0;  // rows
        constexpr int kStride = GW * 32, kVectors = kChunk / 4 / kStride;
        RowWeight rw;
        unsigned long long sum = 0;
        uint32_t first = kNoToken;
        auto begin_second = [&](const Held &h, uint32_t i) {
            ok = ok && mbar_wait(info_full + (i & 1), (i >> 1) & 1, a.polls);
            const float scale = scale_s[i & 1];
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(info_empty + (i & 1));
            ok = ok && mbar_wait_cluster(top_full + i % kTops, (i / kTops) & 1, a.polls);
            const int32_t t = __reduce_max_sync(~0u, lane < S ? tops[i % kTops][lane] : kExcluded);
            rw.set(t, scale);
            sum = 0;
            first = kNoToken;
            if (h.edge_at != kNoToken) {
                uint32_t w, none;
                rw.slow2(h.edge, h.edge, w, none);
                sum = w;
                if (h.edge == rw.top) first = h.edge_at;
            }
        };
        auto second_chunk = [&](const Row &r, int at, int c) {
            const int4 *p = reinterpret_cast<const int4 *>(smem + at * kChunkBytes) + gt;
            const int n = (int)min(r.v1 - r.v0 - c * (kChunk / 4), (uint32_t)kChunk / 4) - gt;
            if (rw.fast) {
                auto add = [&](const int4 &q) {
                    uint32_t w0, w1, w2, w3;
                    rw.fast2(q.x, q.y, w0, w1);
                    rw.fast2(q.z, q.w, w2, w3);
                    sum += (unsigned long long)w0 + w1;
                    sum += (unsigned long long)w2 + w3;
                };
                if ((kVectors - 1) * kStride < n) {
#pragma unroll
                    for (int u = 0; u < kVectors; u++) add(p[u * kStride]);
                } else {
#pragma unroll 1
                    for (int u = 0; u * kStride < n; u++) add(p[u * kStride]);
                }
                return;
            }
#pragma unroll 1
            for (int u = 0; u * kStride < n; u++) {
                const int4 q = p[u * kStride];
                if (rw.greedy) {
                    const uint32_t e = r.head + (r.v0 + c * (kChunk / 4) + gt + u * kStride) * 4;
                    if (q.w == rw.top) first = min(first, e + 3);
                    if (q.z == rw.top) first = min(first, e + 2);
                    if (q.y == rw.top) first = min(first, e + 1);
                    if (q.x == rw.top) first = min(first, e);
                } else {
                    uint32_t w0, w1, w2, w3;
                    rw.slow2(q.x, q.y, w0, w1);
                    rw.slow2(q.z, q.w, w2, w3);
                    sum += (unsigned long long)w0 + w1;
                    sum += (unsigned long long)w2 + w3;
                }
            }
        };
        auto end_second = [&](uint32_t row, uint32_t i) {
            // sums (greedy: the smallest first position) of the warp, then of the CTA; nothing is
            // written for a row that a warp of the CTA gave up
            ok = __all_sync(~0u, ok);
            if (!ok) return;
            auto whole = [&](unsigned long long v) {
                if (rw.greedy) return (unsigned long long)__reduce_min_sync(~0u, (uint32_t)v);
                return sum_lanes(v);
            };
            sum = whole(rw.greedy ? first : sum);
            if (lane == 0) warp_part[i & 1][warp] = sum;
            if (last_of(&part_count[i & 1], kMassWarps)) {
                const unsigned long long part =
                    whole(lane < kMassWarps ? warp_part[i & 1][lane] : rw.greedy ? (unsigned long long)kNoToken : 0);
                if (lane == 0) {
                    RowPart *out = a.rows + row;
                    out->part[rank] = part;
                    if (rank == 0) {
                        out->top = rw.top;
                        out->scale = rw.scale;
                    }
                }
                // (nobody waits for the last rows', and their CTAs may be gone)
                if (i + kTops < count) arrive_all(top_done + i % kTops);
            }
            __syncwarp();
        };
        Place place{0, 0, kTwice ? kFirstRing : 0, kTwice ? a.ring - kFirstRing : a.ring};
        uint32_t i = 0;
        for (; ok && row < a.total; row += groups, i++) {
            const Held h(a, row, rank, (int)threadIdx.x);
            if (!kTwice) {
                Place p = place;
                for (int c = p.own(mine); c < h.chunks; c += kGroups, p.move(kGroups)) {
                    ok = ok && mbar_wait(full + p.slot(), p.phase, a.polls);
                    first_chunk(h.r, p.slot(), c, gt, std::integral_constant<int, kStride>());
                }
                send_top(i, h.edge, warp);
                if (!ok) break;
            }
            begin_second(h, i);
            Place q = place;
            for (int c = q.own(mine); c < h.chunks; c += kGroups, q.move(kGroups)) {
                if (kTwice) ok = ok && mbar_wait(full + q.slot(), q.phase, a.polls);
                second_chunk(h.r, q.slot(), c);
                release(q.slot());
            }
            end_second(row, i);
            if (!ok) break;
            place.move(h.chunks);
        }
    }
    // A wait ran out: from this row on the CTA has no parts, since none is written without every
    // warp, and the mark stays.
    if (!ok && lane == 0)
        for (; row < a.total; row += groups) a.rows[row].part[rank] = kGaveUp;
    leave(ok);
}

// ---------------------------------------------------------------------------
// accept tests and the drawn token, a cluster per request
// ---------------------------------------------------------------------------
constexpr int kDrawWarps = 16, kDrawThreads = kDrawWarps * 32;
constexpr int kRuns = 8;
constexpr uint32_t kKeep = 32;  // rows of a request whose numbers stay in shared memory
struct DrawArgs {
    Args a;
    int split;      // CTAs per request
    uint32_t lose;  // by rank in the cluster: CTAs that give the others' sums up at once
};

// kModel: drafts have a distribution of their own.
template <bool kModel>
__global__ void __launch_bounds__(kDrawThreads, 2) k_draw(const DrawArgs d) {
    const Args &a = d.a;
    __shared__ uint32_t first_s, bad_s, begin_s;
    __shared__ RowMass mass_s[kKeep][2], last_s[2];
    __shared__ unsigned long long warp_sum[kDrawWarps], cta_sum[2][kMaxCluster];
    __shared__ unsigned long long run_sum[kDrawWarps][kRuns];  // of up to kRuns runs of a warp's steps
    __shared__ uint64_t sums_full[2];                          // every CTA's sum of the round is there
    __shared__ uint64_t lost[kMaxCluster];                     // a CTA of the cluster, by rank, did not get them
    const int S = d.split, rank = S > 1 ? (int)cluster_rank() : 0;
    const uint32_t b = blockIdx.x / S;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (S > 1) {
        if (threadIdx.x == 0) {
            for (int i = 0; i < 2; i++) mbar_init(sums_full + i, 1);
            for (int i = 0; i < S; i++) mbar_init(lost + i, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            for (int i = 0; i < 2; i++) mbar_expect_tx(sums_full + i, S * 8);
        }
        __syncwarp();
        cluster_arrive();  // waited for before the first sums are sent
    }
    pdl_wait();
    pdl_trigger();
    uint32_t begin, count;
    const bool valid = request_range(a, b, begin, count);
    if (!valid) begin = count = 0;
    if (threadIdx.x == 0) {
        first_s = count;
        bad_s = valid ? 0u : 1u;
        begin_s = begin;
    }
    __syncthreads();
    const uint32_t targets = a.drafts + a.requests;
    // a warp per row: its lower half has the target's, its upper half the draft's;
    // j = count is the row after the last draft
    for (uint32_t j = warp; valid && j <= count; j += kDrawWarps) {
        const uint32_t e = begin + j;
        const bool is_draft = lane >= 16, has = j < count, there = is_draft ? has && kModel : true;
        const RowMass m = load_row(a.rows, there && is_draft ? targets + e : e + b, a.split);
        if (!m.ok && (lane & 15) == 0) bad_s = 1;
        if ((lane & 15) == 0 && j < kKeep) mass_s[j][lane >> 4] = m;
        const uint32_t x = has ? a.draft_tokens[e] : kNoToken;
        uint64_t share = 0;
        if (x < a.vocab && there) {
            const int32_t z = is_draft ? a.draft[e * a.ld_draft + x] : a.target[(e + b) * a.ld_target + x];
            RowWeight rw;
            rw.set(m.top, m.scale);
            uint32_t w, none;
            row_weight2(rw, m.first, z, z, x, x, w, none);
            share = row_share(w, m);
        }
        if (is_draft && !kModel) share = 1ull << 40;
        const uint64_t p = __shfl_sync(~0u, share, 0), q = __shfl_sync(~0u, share, 16);
        if (has && lane == 0) {
            if (a.probs && rank == 0) {
                a.probs[2 * (size_t)e] = p;
                a.probs[2 * (size_t)e + 1] = q;
            }
            if (mul_frac(q, a.accept_u[e]) >= p) atomicMin(&first_s, j);
        }
    }
    __syncthreads();
    const uint32_t n = first_s;
    const bool rejected = n < count, both = kModel && rejected;
    const uint32_t trow = begin + b + n, drow = begin + n;
    if (n >= kKeep && warp == 0) {
        const RowMass m = load_row(a.rows, lane >= 16 && both ? targets + drow : trow, a.split);
        if ((lane & 15) == 0) last_s[lane >> 4] = m;
    }
    if (n >= kKeep) __syncthreads();
    const RowMass mt = n < kKeep ? mass_s[n][0] : last_s[0], md = n < kKeep ? mass_s[n][1] : last_s[1];
    // one path for the whole cluster from here: all of it depends on the request alone
    uint32_t drawn = kNoToken;
    bool bad = bad_s != 0, none = false;  // none: no token can be drawn
    if (S > 1) cluster_wait();
    if (!bad) {
        RowWeight wt, wd;
        wt.set(mt.top, mt.scale);
        if (kModel) wd.set(md.top, md.scale);
        const int32_t *zt = a.target + trow * a.ld_target, *zd = both ? a.draft + drow * a.ld_draft : zt;
        const uint32_t x = rejected ? a.draft_tokens[drow] : kNoToken;
        // a CTA has a run of the vocabulary, a warp a run of that, in steps of 128
        const uint32_t steps = (a.vocab + 127) / 128, parts = S * kDrawWarps, part = rank * kDrawWarps + warp;
        const uint32_t v0 = (uint32_t)((uint64_t)steps * part / parts) * 128,
                       v1 = min(a.vocab, (uint32_t)((uint64_t)steps * (part + 1) / parts) * 128);
        const uint32_t run = ((v1 - v0 + 127) / 128 + kRuns - 1) / kRuns * 128;  // logits per run
        // logits v + lane + 32 u of both rows, and what is drawn from there
        struct Four {
            int32_t t[4], q[kModel ? 4 : 1];
        };
        auto fetch = [&](uint32_t v, bool rest, Four &z) {
            const int32_t *pt = zt + v + lane, *pq = zd + v + lane;
            if (v + 128 <= v1) {
#pragma unroll
                for (int u = 0; u < 4; u++) z.t[u] = pt[32 * u];
                if (kModel && both && rest)
#pragma unroll
                    for (int u = 0; u < 4; u++) z.q[kModel ? u : 0] = pq[32 * u];
            } else {
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const bool in = v + lane + 32 * u < v1;
                    z.t[u] = in ? pt[32 * u] : kExcluded;
                    if (kModel) z.q[kModel ? u : 0] = both && rest && in ? pq[32 * u] : kExcluded;
                }
            }
        };
        // Q0.40 probabilities of four logits of a row
        auto shares = [&](const RowWeight &w, const RowMass &row, bool usual, uint32_t v, const int32_t *z, uint64_t (&m)[4]) {
            uint32_t x0, x1, x2, x3;
            if (usual) {
                w.fast2(z[0], z[1], x0, x1);
                w.fast2(z[2], z[3], x2, x3);
                m[0] = row_share_small(x0, row);
                m[1] = row_share_small(x1, row);
                m[2] = row_share_small(x2, row);
                m[3] = row_share_small(x3, row);
            } else {
                const uint32_t at = v + lane;
                row_weight2(w, row.first, z[0], z[1], at, at + 32, x0, x1);
                row_weight2(w, row.first, z[2], z[3], at + 64, at + 96, x2, x3);
                m[0] = row_share(x0, row);
                m[1] = row_share(x1, row);
                m[2] = row_share(x2, row);
                m[3] = row_share(x3, row);
            }
        };
        const bool usual_t = wt.fast && mt.shift < 32, usual_q = kModel && wd.fast && md.shift < 32;
        auto four = [&](uint32_t v, bool rest, const Four &z, uint64_t (&m)[4]) {
            shares(wt, mt, usual_t, v, z.t, m);
            if (!rest) return;
            if (kModel) {
                uint64_t q[4];
                shares(wd, md, usual_q, v, z.q, q);
#pragma unroll
                for (int u = 0; u < 4; u++) m[u] = m[u] > q[u] ? m[u] - q[u] : 0;
            } else {  // q is all at x, and p at most that
#pragma unroll
                for (int u = 0; u < 4; u++) m[u] = v + lane + 32 * u == x ? 0 : m[u];
            }
        };
        // p less q after a rejection; should that be nothing at all, p
        bool rest = rejected;
        unsigned long long total = 0, mine = 0, below = 0;
        for (int round = 0; round < 2; round++, rest = false) {
            mine = 0;
            Four next;
            if (v0 < v1) fetch(v0, rest, next);
            uint32_t next_run = v0 + run, at_run = 0;
            unsigned long long lanes = 0;
            for (uint32_t v = v0; v < v1; v += 128) {  // the next step's logits under way while this one's are summed
                const Four z = next;
                if (v + 128 < v1) fetch(v + 128, rest, next);
                // nothing where p is nothing
                const int32_t most = max(max(z.t[0], z.t[1]), max(z.t[2], z.t[3]));
                if (!wt.fast || !__all_sync(~0u, wt.base - (uint32_t)most >= wt.most)) {
                    uint64_t m[4];
                    four(v, rest, z, m);
                    lanes += (m[0] + m[1]) + (m[2] + m[3]);
                }
                if (v + 128 >= v1 || v + 128 == next_run) {
                    mine = sum_lanes(lanes);
                    if (lane == 0) run_sum[warp][at_run] = mine;  // of all runs so far
                    at_run++;
                    next_run += run;
                }
            }
            if (round > 0) __syncthreads();  // the last round's sums have been read
            if (lane == 0) warp_sum[warp] = mine;
            __syncthreads();
            const unsigned long long of_warp = lane < kDrawWarps ? warp_sum[lane] : 0, cta = sum_lanes(of_warp);
            below = sum_lanes(lane < warp ? of_warp : 0);
            if (S > 1) {
                if ((int)threadIdx.x < S)
                    st_async(remote(&cta_sum[round][rank], threadIdx.x), (uint64_t)cta, remote(&sums_full[round], threadIdx.x));
                total = 0;
                if (__syncthreads_or(!mbar_wait_cluster(&sums_full[round], 0, d.lose >> rank & 1 ? 0 : a.polls))) {
                    if ((int)threadIdx.x < S) arrive_remote(remote(lost + rank, threadIdx.x));
                    break;  // the CTA's threads go on, or give up, as one
                }
                const unsigned long long of_cta = lane < S ? cta_sum[round][lane] : 0;
                total = sum_lanes(of_cta);
                below += sum_lanes(lane < rank ? of_cta : 0);
            } else {
                total = cta;
            }
            if (total != 0 || !rest) break;
        }
        if (S > 1) {
            __syncwarp();
            cluster_arrive();  // nothing more is sent
        }
        const uint64_t point = mul_frac(total, a.sample_u[b]);
        if (total != 0 && point >= below && point - below < mine) {  // one warp of the cluster holds the point
            __syncwarp();
            // the run that holds it: the first whose running sum passes the point
            const int runs = (int)((v1 - v0 + run - 1) / run);
            const unsigned passed = __ballot_sync(~0u, lane < runs && below + run_sum[warp][lane < runs ? lane : 0] > point);
            const int hit_run = __ffs((int)passed) - 1;
            if (hit_run > 0) below += run_sum[warp][hit_run - 1];
            for (uint32_t v = v0 + hit_run * run; v < v1; v += 128) {
                Four z;
                uint64_t m[4];
                fetch(v, rest, z);
                four(v, rest, z, m);
                unsigned long long sum[4], hit = 0;
                int at = -1;
#pragma unroll
                for (int u = 0; u < 4; u++) sum[u] = sum_lanes(m[u]);
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (at < 0) {
                        if (below + sum[u] > point) at = u, hit = m[u];
                        else below += sum[u];
                    }
                if (at < 0) continue;
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long t = __shfl_up_sync(~0u, hit, o);
                    if (lane >= o) hit += t;
                }
                drawn = v + 32 * at + (uint32_t)__ffs((int)__ballot_sync(~0u, below + hit > point)) - 1;
                break;
            }
        }
        none = total == 0;
    } else if (S > 1) {
        __syncthreads();  // (the others' part of this lies in the sums) no thread arrives before all have passed the last wait
        cluster_arrive();
    }
    uint32_t *out = a.tokens + (size_t)b * (a.max_drafts + 1);
    if (rank == 0) {
        const uint32_t from = *(const volatile uint32_t *)&begin_s;  // (begin would take a register until here)
        for (uint32_t j = threadIdx.x; j <= a.max_drafts; j += kDrawThreads)
            if (bad || j > n) out[j] = kNoToken;
            else if (j < n) out[j] = a.draft_tokens[from + j];
    }
    // no count and no drawn token is written before every CTA has said whether it got the sums
    if (S > 1) {
        __syncwarp();
        cluster_wait();
        if (__any_sync(~0u, lane < S && mbar_test_cluster(lost + lane, 0))) {
            if (rank == 0)
                for (uint32_t j = threadIdx.x; j <= a.max_drafts; j += kDrawThreads) out[j] = kNoToken;
            bad = true;
            let_land();
        }
    }
    if (drawn != kNoToken && !bad && lane == 0) out[n] = drawn;
    if (rank == 0 && threadIdx.x == 0) {
        if (none && !bad) out[n] = kNoToken;
        a.accepted[b] = bad ? kNoToken : n;
    }
}

// CTAs per row that are considered: 9 and 6 fill a group of 18 SMs that cannot hold
// a cluster together with its neighbours.
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 9, 12, 16};
// Loaded once (a cluster's shares fit), loaded twice.
void (*const kMass[2])(Args) = {k_mass<false, 8>, k_mass<true, 4>};
// Per device: how many clusters of k_mass run at once, by their size.
struct DeviceSetup {
    bool ready = false;
    int sms = 0;
    int clusters[kMaxCluster + 1] = {};
};
constexpr int kMaxDevices = 64;
std::mutex g_setup_mu;
DeviceSetup g_setup[kMaxDevices];

cudaError_t configure(cudaLaunchConfig_t &cfg, cudaLaunchAttribute (&attr)[2], dim3 grid, int threads, size_t smem, int cluster,
                      cudaStream_t s) {
    cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaSuccess;
}

cudaError_t device_setup(DeviceSetup &out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lock(g_setup_mu);
    DeviceSetup &d = g_setup[dev];
    if (!d.ready) {
        if ((e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
        const int smem = kMaxRing * kChunkBytes;
        for (auto fn : kMass) {
            if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
            if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        }
        if ((e = cudaFuncSetAttribute(k_draw<false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        if ((e = cudaFuncSetAttribute(k_draw<true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        d.clusters[1] = d.sms;
        for (int c : kSplits) {
            if (c == 1) continue;
            cudaLaunchConfig_t cfg;
            cudaLaunchAttribute attr[2];
            configure(cfg, attr, dim3((unsigned)c), mass_threads(true), smem, c, nullptr);
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kMass[1], &cfg) != cudaSuccess) {
                (void)cudaGetLastError();
                n = 0;
            }
            d.clusters[c] = n;
        }
        d.ready = true;
    }
    out = d;
    return cudaSuccess;
}

int fail(int code, const std::string &msg) {
    llmx::set_last_error("verify_drafts: " + msg);
    return code;
}
// Reports a failed runtime call, whose code would else be found by the thread's next
// check of a launch.
int cuda_fail(const char *what, cudaError_t e) {
    (void)cudaGetLastError();
    return fail(LLMX_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace

extern "C" size_t llmx_verify_workspace_bytes(uint32_t requests, uint32_t drafts, uint32_t vocab) {
    (void)vocab;  // the rows' sums only: nothing of a row is kept in memory
    return ((2ull * drafts + requests) * sizeof(RowPart) + 255) / 256 * 256;
}

extern "C" int llmx_verify_drafts(const int32_t *target, size_t ld_target, const int32_t *draft, size_t ld_draft,
                                  uint32_t vocab, const uint32_t *draft_tokens, const uint32_t *offsets,
                                  uint32_t requests, uint32_t drafts, uint32_t max_drafts, const float *temperature,
                                  const uint32_t *accept_u, const uint32_t *sample_u, uint32_t *tokens,
                                  uint32_t *accepted, uint64_t *probs, void *workspace, size_t workspace_bytes,
                                  void *stream) {
    if (!target || !offsets || !temperature || !sample_u || !tokens || !accepted || !workspace)
        return fail(LLMX_ERR_ARG, "null pointer");
    if (drafts && (!draft_tokens || !accept_u)) return fail(LLMX_ERR_ARG, "null pointer with drafts > 0");
    if (vocab == 0 || vocab > kMaxVocab) return fail(LLMX_ERR_ARG, "vocab must be 1..2^22, got " + std::to_string(vocab));
    if (requests == 0 || requests > kMaxRequests)
        return fail(LLMX_ERR_ARG, "requests must be 1..65535, got " + std::to_string(requests));
    if (drafts > kMaxTotal) return fail(LLMX_ERR_ARG, "drafts must be at most 2^24, got " + std::to_string(drafts));
    if (max_drafts > kMaxDrafts)
        return fail(LLMX_ERR_ARG, "max_drafts must be at most 1023, got " + std::to_string(max_drafts));
    if ((uint64_t)max_drafts * requests < drafts)
        return fail(LLMX_ERR_ARG, "drafts exceeds requests * max_drafts");
    if (ld_target == 0) ld_target = vocab;
    if (ld_draft == 0) ld_draft = vocab;
    if (ld_target < vocab || ld_draft < vocab) return fail(LLMX_ERR_ARG, "a row stride is smaller than vocab");
    if (((uintptr_t)target | (uintptr_t)draft | (uintptr_t)draft_tokens | (uintptr_t)offsets | (uintptr_t)temperature |
         (uintptr_t)accept_u | (uintptr_t)sample_u | (uintptr_t)tokens | (uintptr_t)accepted) & 3u ||
        ((uintptr_t)probs & 7u))
        return fail(LLMX_ERR_ARG, "a pointer is not aligned to its element");
    if ((uintptr_t)workspace & 255u) return fail(LLMX_ERR_ARG, "workspace must be 256-byte aligned");
    if (workspace_bytes < llmx_verify_workspace_bytes(requests, drafts, vocab))
        return fail(LLMX_ERR_ARG, "workspace too small: " + std::to_string(workspace_bytes) + " bytes");
    Args a{};
    a.target = target;
    a.draft = drafts ? draft : nullptr;
    a.ld_target = ld_target;
    a.ld_draft = ld_draft;
    a.vocab = vocab;
    a.requests = requests;
    a.drafts = drafts;
    a.max_drafts = max_drafts;
    a.draft_tokens = draft_tokens;
    a.offsets = offsets;
    a.temperature = temperature;
    a.accept_u = accept_u;
    a.sample_u = sample_u;
    a.tokens = tokens;
    a.accepted = accepted;
    a.probs = probs;
    a.rows = static_cast<RowPart *>(workspace);
    a.polls = llmx::serving_wait_polls();
    a.total = drafts + requests + (a.draft ? drafts : 0);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DeviceSetup dev;
    cudaError_t e = device_setup(dev);
    if (e != cudaSuccess) return cuda_fail("device set-up", e);
    // CTAs per row: the split with the least time for the busiest cluster, in
    // microseconds as measured on one SM: a chunk's first pass alone 0.4 and its second 0.5,
    // both beside one another 0.62; a row's exchange and its ends 2, or 0.6 where they are hidden.
    const int chunks = (int)((vocab + kChunk - 1) / kChunk);
    double best = 0;
    for (int split : kSplits) {
        if (dev.clusters[split] == 0 || (split > 1 && chunks < split)) continue;
        const int share = (chunks + split - 1) / split;
        const uint32_t rounds = (a.total + dev.clusters[split] - 1) / dev.clusters[split];
        for (int resident = 0; resident < 2; resident++) {
            if (resident && share > kMaxRing) continue;
            const double per = (double)chunks / split;
            const double cost = resident ? rounds * (per * 0.9 + 2.0) : rounds * (per * 0.62 + 0.6) + per * 0.4 + 2.0;
            if (a.split == 0 || cost < best) {
                best = cost;
                a.split = split;
                a.resident = resident;
                // (even: a slot is one of two groups')
                a.ring = resident ? std::min(kMaxRing, rounds > 1 ? 2 * share : (share + 1) / 2 * 2) : kMaxRing;
            }
        }
    }
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    const uint32_t groups = std::min<uint32_t>(a.total, (uint32_t)dev.clusters[a.split]);
    configure(cfg, attr, dim3(groups * a.split), mass_threads(!a.resident), (size_t)a.ring * kChunkBytes, a.split, s);
    e = cudaLaunchKernelEx(&cfg, kMass[a.resident ? 0 : 1], a);
    if (e != cudaSuccess) return cuda_fail("k_mass", e);
    DrawArgs d{a, 1, llmx::serving_lost_draws()};
    while (d.split < kMaxCluster && requests * d.split * 2 <= (uint32_t)dev.sms * 2 && vocab >= 2048u * d.split) d.split *= 2;
    configure(cfg, attr, dim3(requests * d.split), kDrawThreads, 0, d.split, s);
    e = cudaLaunchKernelEx(&cfg, a.draft ? k_draw<true> : k_draw<false>, d);
    if (e != cudaSuccess) return cuda_fail("k_draw", e);
    return LLMX_OK;
}
