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
// twice; to read it from memory once, a cluster of CTAs holds it in shared
// memory between the two passes, exchanges the maxima there, and the pieces
// of its next row arrive while this one is being summed.  k_draw tests the
// drafts of a request and draws its last token, a cluster per request.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <mutex>
#include <string>

#include "llmx.h"
#include "device_util.cuh"
#include "gemv_common.cuh"
#include "kernels.cuh"

namespace {

using llmx::bulk_g2s;
using llmx::mbar_arrive;
using llmx::mbar_expect_tx;
using llmx::mbar_init;
using llmx::mbar_wait;
using llmx::pdl_trigger;
using llmx::pdl_wait;
using llmx::smem_u32;

constexpr int kExcluded = INT_MIN;
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr uint32_t kMaxVocab = 1u << 22, kMaxRequests = 65535, kMaxDrafts = 1023, kMaxTotal = 1u << 24;
constexpr float kMinTemperature = 1e-6f;     // at or below: greedy
constexpr float kLog2e16 = 0x1.715476p-16f;  // log2(e) / 2^16: Q16.16 differences to octaves
constexpr int kMaxCluster = 16;

// What a row of logits is reduced to, as k_mass leaves it: every CTA of the
// row's cluster writes its part, the sum of its weights or (greedy) the first
// position of the maximum in its share.
constexpr unsigned long long kNoPart = ~0ull;   // greedy: not here
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
    int resident;    // a CTA's share of a row fits the ring
    unsigned long long minus_zero;  // two -0.0f (mul2)
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
// a * b, rounded on its own: a fused operation with -0, which the compiler must not
// see through (it fuses a packed product, mul.rn or with a constant -0, with the
// addition that follows it, and the weights would differ in their last bits).
// So the -0 is a kernel argument.
static __device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b, f32x2 minus_zero) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(minus_zero));
    return r;
}
static __device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// floor(2^31 * 2^-e), e = (top - z) * scale capped at 100, of two logits.  Every
// float step is rounded on its own (no contraction), so that the weight is the
// same integer wherever it is computed.  2^x = 2^round(x) 2^f and 2^f on
// [-1/2, 1/2] is 1 + f q(f), q of degree 4 fitted to the relative error at
// Chebyshev points: below 2e-7 with the rounding of its steps.  x = -e; adding
// 1.5 * 2^23 rounds it to the nearest whole number (even at ties) and leaves that number in the
// low bits, from where one shifted addition puts it into the exponent.  The
// cap keeps the exponent in range; beyond e = 32 the weight is 0 anyway.  The
// coefficients carry the 2^31.  Packed pairs halve the float instructions, which
// are what a row's second pass spends its time on.
static __device__ __forceinline__ void soft_weight2(int32_t z0, int32_t z1, int32_t top, f32x2 minus_scale, f32x2 mz, uint32_t &w0,
                                                    uint32_t &w1) {
    const f32x2 magic = pack2(12582912.0f, 12582912.0f), minus_magic = pack2(-12582912.0f, -12582912.0f);
    float x0 = __uint2float_rn((uint32_t)top - (uint32_t)z0), x1 = __uint2float_rn((uint32_t)top - (uint32_t)z1);
    unpack2(mul2(pack2(x0, x1), minus_scale, mz), x0, x1);
    const f32x2 x = pack2(fmaxf(x0, -100.0f), fmaxf(x1, -100.0f));
    const f32x2 m = add2(x, magic), r = add2(m, minus_magic);
    float r0, r1, m0, m1, p0, p1;
    unpack2(r, r0, r1);
    const f32x2 f = add2(x, pack2(-r0, -r1));
    f32x2 p = add2(mul2(f, pack2(0x1.5bba12p21f, 0x1.5bba12p21f), mz), pack2(0x1.3cea88p24f, 0x1.3cea88p24f));
    p = add2(mul2(p, f, mz), pack2(0x1.c6b752p26f, 0x1.c6b752p26f));
    p = add2(mul2(p, f, mz), pack2(0x1.ebf9bcp28f, 0x1.ebf9bcp28f));
    p = add2(mul2(p, f, mz), pack2(0x1.62e42ap30f, 0x1.62e42ap30f));
    p = add2(mul2(p, f, mz), pack2(0x1p31f, 0x1p31f));
    unpack2(m, m0, m1);
    unpack2(p, p0, p1);
    w0 = __float2uint_rz(__int_as_float(__float_as_int(p0) + (__float_as_int(m0) << 23)));
    w1 = __float2uint_rz(__int_as_float(__float_as_int(p1) + (__float_as_int(m1) << 23)));
}
// Whether an excluded logit needs a test of its own: not when its difference to the
// maximum is 40 octaves or more, where the weight is 0 by the formula.
static __device__ __forceinline__ bool must_test_excluded(int32_t top, float scale) {
    return !(__fmul_rn(__uint2float_rn((uint32_t)top - (uint32_t)kExcluded), scale) >= 40.0f);
}

// A row's numbers as k_draw uses them.
struct RowMass {
    int32_t top;
    float scale;
    uint32_t first;    // greedy: the maximum's first position
    uint32_t inverse;  // floor(2^62 / (S >> h)), 0 when nothing is left
    int32_t shift;     // 22 + h
    bool ok;
};
static __device__ RowMass load_row(const RowPart *rows, uint32_t row, int split) {
    const RowPart *p = rows + row;
    RowMass r;
    r.top = p->top;
    r.scale = p->scale;
    r.first = kNoToken;
    r.ok = true;
    unsigned long long sum = 0;
    for (int i = 0; i < split; i++) {
        const unsigned long long v = p->part[i];
        if (v == kGaveUp) r.ok = false;
        else if (r.scale < 0.0f) r.first = min(r.first, (uint32_t)v);
        else sum += v;
    }
    if (r.scale < 0.0f) sum = r.top != kExcluded && r.first != kNoToken ? 1ull << 31 : 0;
    int h = 32 - __clzll((long long)sum);  // sum has 64 - clz bits; 32 remain
    h = h < 0 ? 0 : h;
    r.inverse = sum ? (uint32_t)((1ull << 62) / (sum >> h)) : 0u;
    r.shift = 22 + h;
    return r;
}
static __device__ __forceinline__ void row_weight2(const RowMass &r, f32x2 mz, int32_t z0, int32_t z1, uint32_t v0,
                                                   uint32_t v1, uint32_t &w0, uint32_t &w1) {
    if (r.scale < 0.0f) {
        w0 = v0 == r.first ? 0x80000000u : 0u;
        w1 = v1 == r.first ? 0x80000000u : 0u;
    } else {
        soft_weight2(z0, z1, r.top, pack2(-r.scale, -r.scale), mz, w0, w1);
    }
    if (z0 == kExcluded) w0 = 0;
    if (z1 == kExcluded) w1 = 0;
}
static __device__ __forceinline__ uint64_t row_share(uint32_t w, const RowMass &r) {
    return ((uint64_t)w * r.inverse) >> r.shift;
}
// floor(a * u / 2^32)
static __device__ __forceinline__ uint64_t mul_frac(uint64_t a, uint32_t u) { return __umul64hi(a, (uint64_t)u << 32); }

// ---- clusters -------------------------------------------------------------------
static __device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
static __device__ __forceinline__ uint32_t remote(const void *p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
static __device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
static __device__ __forceinline__ bool mbar_wait_cluster(uint64_t *bar, uint32_t parity) {
    for (uint32_t i = 0; i < llmx::kSpinLimit; i++) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}

// ---------------------------------------------------------------------------
// rows -> maxima and sums
// ---------------------------------------------------------------------------
constexpr int kMassWarps = 16, kMassThreads = (kMassWarps + 2) * 32;  // sums, loads, the rows' requests
constexpr int kChunk = 4096;                                          // logits per chunk: two 16-byte vectors per thread
constexpr int kChunkBytes = kChunk * 4;
constexpr int kMaxRing = 13;

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
        v0 = (uint32_t)((uint64_t)vectors * rank / a.split);
        v1 = (uint32_t)((uint64_t)vectors * (rank + 1) / a.split);
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

__global__ void __launch_bounds__(kMassThreads, 1) k_mass(const Args a) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t full[kMaxRing], empty[kMaxRing];
    __shared__ uint64_t info_full[2], info_empty[2];  // a row's temperature
    __shared__ uint64_t top_full[2];                  // every CTA's maximum of the row
    __shared__ float scale_s[2];
    __shared__ int32_t tops[2][kMaxCluster];
    __shared__ int32_t warp_top[kMassWarps];
    __shared__ unsigned long long warp_part[2][kMassWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = a.split, rank = S > 1 ? (int)cluster_rank() : 0;
    const uint32_t group = blockIdx.x / S, groups = gridDim.x / S;
    const int passes = a.resident ? 1 : 2;  // times that a row is loaded
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.ring; i++) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, kMassWarps);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(info_full + i, 1);
            mbar_init(info_empty + i, kMassWarps);
            mbar_init(top_full + i, S);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (S > 1) cluster_sync();
    else __syncthreads();
    pdl_wait();
    pdl_trigger();

    if (warp == kMassWarps) {  // ---- loads ------------------------------------------
        if (lane == 0) {
            int s = 0, phase = 1, issued = 0;
            bool ok = true;
            for (uint32_t row = group; ok && row < a.total; row += groups) {
                const Row r(a, row, rank);
                for (int pass = 0; ok && pass < passes; pass++)
                    for (uint32_t v = r.v0; v < r.v1; v += kChunk / 4) {
                        if (issued >= a.ring && !mbar_wait(empty + s, phase)) {
                            ok = false;
                            break;
                        }
                        const uint32_t bytes = min(r.v1 - v, (uint32_t)kChunk / 4) * 16;
                        mbar_expect_tx(full + s, bytes);
                        bulk_g2s(smem + s * kChunkBytes, r.z + r.head + (size_t)v * 4, bytes, full + s);
                        issued++;
                        if (++s == a.ring) {
                            s = 0;
                            phase ^= 1;
                        }
                    }
            }
            for (int q = 0; !ok && q < a.ring && q < issued; q++) {  // the copies in flight land before the CTA ends
                const int last = q + ((issued - 1 - q) / a.ring) * a.ring;
                (void)mbar_wait(full + q, (last / a.ring) & 1);
            }
        }
    } else if (warp == kMassWarps + 1) {  // ---- the rows' temperatures --------------------
        uint32_t i = 0;
        for (uint32_t row = group; row < a.total; row += groups, i++) {
            const uint32_t b = owner_of(a, row);
            const float scale = b == kNoToken ? -1.0f : row_scale(a.temperature[b]);
            if (i >= 2 && !__all_sync(~0u, mbar_wait(info_empty + (i & 1), ((i >> 1) - 1) & 1))) break;
            if (lane == 0) {
                scale_s[i & 1] = scale;
                mbar_arrive(info_full + (i & 1));
            }
            __syncwarp();
        }
    } else {  // ---- maxima and sums ----------------------------------------------------
        int s = 0, phase = 0;
        uint32_t i = 0;
        bool ok = true;
        for (uint32_t row = group; row < a.total; row += groups, i++) {
            if (!ok) {  // a wait ran out: this row and the rest have no sums
                if (threadIdx.x == 0) a.rows[row].part[rank] = kGaveUp;
                continue;
            }
            const Row r(a, row, rank);
            const int b = i & 1;
            // the head and the tail, one logit of a thread
            int32_t edge = kExcluded;
            uint32_t edge_at = kNoToken;
            if (threadIdx.x < 3 && rank == 0 && threadIdx.x < r.head) edge_at = threadIdx.x;
            const uint32_t tail = r.head + r.vectors * 4;
            if (threadIdx.x >= 4 && threadIdx.x < 7 && rank == S - 1 && tail + threadIdx.x - 4 < a.vocab)
                edge_at = tail + threadIdx.x - 4;
            if (edge_at != kNoToken) edge = r.z[edge_at];
            int32_t top = edge;
            const int s0 = s, phase0 = phase;
            for (uint32_t v = r.v0; ok && v < r.v1; v += kChunk / 4) {
                ok = mbar_wait(full + s, phase);
                const int4 *p = reinterpret_cast<const int4 *>(smem + s * kChunkBytes);
                const int n = min(r.v1 - v, (uint32_t)kChunk / 4);
#pragma unroll
                for (int u = 0; u < kChunk / 4; u += kMassWarps * 32) {
                    const int at = u + threadIdx.x;
                    if (at < n) {
                        const int4 q = p[at];
                        top = max(max(top, q.x), max(max(q.y, q.z), q.w));
                    }
                }
                if (!a.resident) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty + s);
                }
                if (++s == a.ring) {
                    s = 0;
                    phase ^= 1;
                }
            }
            top = __reduce_max_sync(~0u, top);
            if (lane == 0) warp_top[warp] = top;
            asm volatile("bar.sync 1, %0;" ::"n"(kMassWarps * 32) : "memory");
            top = __reduce_max_sync(~0u, warp_top[lane & (kMassWarps - 1)]);
            if (S > 1) {  // push it to every CTA of the cluster, wait for theirs
                if (warp == 0 && lane < S) {
                    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(remote(&tops[b][rank], lane)), "r"(top) : "memory");
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote(top_full + b, lane))
                                 : "memory");
                }
                ok = mbar_wait_cluster(top_full + b, (i >> 1) & 1) && ok;
                top = __reduce_max_sync(~0u, lane < S ? tops[b][lane] : kExcluded);
            }
            ok = mbar_wait(info_full + b, (i >> 1) & 1) && ok;
            const float scale = scale_s[b];
            __syncwarp();
            if (lane == 0) mbar_arrive(info_empty + b);
            unsigned long long sum = 0;
            const bool greedy = scale < 0.0f, test = must_test_excluded(top, scale);
            const f32x2 minus_scale = pack2(-scale, -scale);
            uint32_t first = kNoToken;
            if (edge_at != kNoToken) {
                uint32_t w, none;
                soft_weight2(edge, edge, top, minus_scale, a.minus_zero, w, none);
                sum = edge == kExcluded ? 0 : w;
                if (edge == top) first = edge_at;
            }
            if (a.resident) {
                s = s0;
                phase = phase0;
            }
            for (uint32_t v = r.v0; ok && v < r.v1; v += kChunk / 4) {
                if (!a.resident) ok = mbar_wait(full + s, phase);
                const int4 *p = reinterpret_cast<const int4 *>(smem + s * kChunkBytes);
                const int n = min(r.v1 - v, (uint32_t)kChunk / 4);
#pragma unroll
                for (int u = 0; u < kChunk / 4; u += kMassWarps * 32) {
                    const int at = u + threadIdx.x;
                    if (at < n) {
                        const int4 q = p[at];
                        if (!greedy) {
                            uint32_t w0, w1, w2, w3;
                            soft_weight2(q.x, q.y, top, minus_scale, a.minus_zero, w0, w1);
                            soft_weight2(q.z, q.w, top, minus_scale, a.minus_zero, w2, w3);
                            if (test) {
                                w0 = q.x == kExcluded ? 0u : w0;
                                w1 = q.y == kExcluded ? 0u : w1;
                                w2 = q.z == kExcluded ? 0u : w2;
                                w3 = q.w == kExcluded ? 0u : w3;
                            }
                            sum += (unsigned long long)w0 + w1;
                            sum += (unsigned long long)w2 + w3;
                        } else {
                            const uint32_t e = r.head + (v + at) * 4;
                            if (q.w == top) first = min(first, e + 3);
                            if (q.z == top) first = min(first, e + 2);
                            if (q.y == top) first = min(first, e + 1);
                            if (q.x == top) first = min(first, e);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + s);
                if (++s == a.ring) {
                    s = 0;
                    phase ^= 1;
                }
            }
            if (greedy) {
                first = __reduce_min_sync(~0u, first);
                sum = first == kNoToken ? kNoPart : first;
            } else {
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            }
            // read by thread 0 below before the next but one row's are written
            if (lane == 0) warp_part[b][warp] = sum;
            int fine;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.red.and.pred q, 1, %2, p;\n selp.b32 %0, 1, 0, q;\n}"
                         : "=r"(fine)
                         : "r"((int)ok), "n"(kMassWarps * 32)
                         : "memory");
            ok = fine != 0;  // all warps go on, or none
            if (threadIdx.x == 0) {
                unsigned long long part = greedy ? kNoPart : 0;
                for (int q = 0; q < kMassWarps; q++) part = greedy ? min(part, warp_part[b][q]) : part + warp_part[b][q];
                RowPart *out = a.rows + row;
                out->part[rank] = ok ? part : kGaveUp;
                if (rank == 0) {
                    out->top = top;
                    out->scale = scale;
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// accept tests and the drawn token, a cluster per request
// ---------------------------------------------------------------------------
constexpr int kDrawWarps = 16, kDrawThreads = kDrawWarps * 32;
struct DrawArgs {
    Args a;
    int split;  // CTAs per request
};

__global__ void __launch_bounds__(kDrawThreads) k_draw(const DrawArgs d) {
    const Args &a = d.a;
    __shared__ uint32_t first_s, bad_s;
    __shared__ RowMass mt_s, md_s;
    __shared__ unsigned long long warp_sum[kDrawWarps], cta_sum[2][kMaxCluster];
    const int S = d.split, rank = S > 1 ? (int)cluster_rank() : 0;
    const uint32_t b = blockIdx.x / S;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t *out = a.tokens + (size_t)b * (a.max_drafts + 1);
    pdl_wait();
    pdl_trigger();
    uint32_t begin, count;
    const bool valid = request_range(a, b, begin, count);
    if (!valid) begin = count = 0;
    if (threadIdx.x == 0) {
        first_s = count;
        bad_s = valid ? 0u : 1u;
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < count; j += kDrawThreads) {
        const uint32_t e = begin + j, x = a.draft_tokens[e];
        uint64_t pq[2] = {0, a.draft ? 0 : 1ull << 40};
        for (int side = 0; side < (a.draft ? 2 : 1); side++) {
            const RowMass m = load_row(a.rows, side ? a.drafts + a.requests + e : e + b, a.split);
            if (!m.ok) bad_s = 1;
            if (x < a.vocab) {
                const int32_t z = side ? a.draft[e * a.ld_draft + x] : a.target[(e + b) * a.ld_target + x];
                uint32_t w, none;
                row_weight2(m, a.minus_zero, z, z, x, x, w, none);
                pq[side] = row_share(w, m);
            }
        }
        if (a.probs && rank == 0) {
            a.probs[2 * (size_t)e] = pq[0];
            a.probs[2 * (size_t)e + 1] = pq[1];
        }
        if (mul_frac(pq[1], a.accept_u[e]) >= pq[0]) atomicMin(&first_s, j);
    }
    __syncthreads();
    const uint32_t n = first_s;
    const bool rejected = n < count, both = rejected && a.draft != nullptr;
    const uint32_t trow = begin + b + n, drow = begin + n;
    if (threadIdx.x == 0) {
        mt_s = load_row(a.rows, min(trow, a.drafts + a.requests - 1), a.split);
        if (!mt_s.ok) bad_s = 1;
    }
    if (threadIdx.x == 32 && both) md_s = load_row(a.rows, a.drafts + a.requests + drow, a.split);
    __syncthreads();
    // one path for the whole cluster from here: all of it depends on the request alone
    uint32_t drawn = kNoToken;
    const bool bad = bad_s != 0;
    if (!bad) {
        const RowMass mt = mt_s, md = md_s;
        const int32_t *zt = a.target + trow * a.ld_target, *zd = both ? a.draft + drow * a.ld_draft : zt;
        const uint32_t x = rejected ? a.draft_tokens[drow] : kNoToken;
        // a CTA has a run of the vocabulary, a warp a run of that, in steps of 128
        const uint32_t steps = (a.vocab + 127) / 128, parts = S * kDrawWarps, part = rank * kDrawWarps + warp;
        const uint32_t v0 = (uint32_t)((uint64_t)steps * part / parts) * 128,
                       v1 = min(a.vocab, (uint32_t)((uint64_t)steps * (part + 1) / parts) * 128);
        // what is drawn from, of logits v + lane + 32 u; rest: p less q
        auto four = [&](uint32_t v, bool rest, uint64_t (&m)[4]) {
            int32_t t[4], q[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const uint32_t at = v + lane + 32 * u;
                t[u] = at < v1 ? zt[at] : kExcluded;
                q[u] = both && rest && at < v1 ? zd[at] : kExcluded;
            }
#pragma unroll
            for (int u = 0; u < 4; u += 2) {
                const uint32_t at = v + lane + 32 * u;
                uint32_t w0, w1;
                row_weight2(mt, a.minus_zero, t[u], t[u + 1], at, at + 32, w0, w1);
                m[u] = row_share(w0, mt);
                m[u + 1] = row_share(w1, mt);
                if (!rest) continue;
                uint64_t q0 = at == x ? 1ull << 40 : 0, q1 = at + 32 == x ? 1ull << 40 : 0;
                if (both) {
                    row_weight2(md, a.minus_zero, q[u], q[u + 1], at, at + 32, w0, w1);
                    q0 = row_share(w0, md);
                    q1 = row_share(w1, md);
                }
                m[u] = m[u] > q0 ? m[u] - q0 : 0;
                m[u + 1] = m[u + 1] > q1 ? m[u + 1] - q1 : 0;
            }
        };
        // p less q after a rejection; should that be nothing at all, p
        bool rest = rejected;
        unsigned long long total = 0, mine = 0, below = 0;
        for (int round = 0; round < 2; round++, rest = false) {
            mine = 0;
            for (uint32_t v = v0; v < v1; v += 128) {
                uint64_t m[4];
                four(v, rest, m);
                mine += (m[0] + m[1]) + (m[2] + m[3]);
            }
            for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
            if (lane == 0) warp_sum[warp] = mine;
            __syncthreads();
            unsigned long long cta = 0;
            below = 0;
            for (int q = 0; q < kDrawWarps; q++) {
                if (q < warp) below += warp_sum[q];
                cta += warp_sum[q];
            }
            if (S > 1) {
                if ((int)threadIdx.x < S)
                    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(&cta_sum[round][rank], threadIdx.x)), "l"(cta)
                                 : "memory");
                cluster_sync();
                total = 0;
                for (int q = 0; q < S; q++) {
                    if (q < rank) below += cta_sum[round][q];
                    total += cta_sum[round][q];
                }
            } else {
                total = cta;
                __syncthreads();  // the warps' sums are read before the next round's
            }
            if (total != 0 || !rest) break;
        }
        const uint64_t point = mul_frac(total, a.sample_u[b]);
        if (total != 0 && point >= below && point - below < mine) {  // one warp of the cluster holds the point
            for (uint32_t v = v0; v < v1; v += 128) {
                uint64_t m[4];
                four(v, rest, m);
                for (int u = 0; u < 4; u++) {
                    unsigned long long sum = m[u];
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long t = __shfl_up_sync(~0u, sum, o);
                        if (lane >= o) sum += t;
                    }
                    const unsigned hit = __ballot_sync(~0u, below + sum > point);
                    if (hit && drawn == kNoToken) drawn = v + 32 * u + (uint32_t)__ffs((int)hit) - 1;
                    below += __shfl_sync(~0u, sum, 31);
                }
                if (drawn != kNoToken) break;
            }
            if (lane == 0) out[n] = drawn;
        } else if (total == 0 && rank == 0 && threadIdx.x == 0) {
            out[n] = kNoToken;
        }
    }
    if (rank == 0) {
        for (uint32_t j = threadIdx.x; j <= a.max_drafts; j += kDrawThreads) {
            if (bad) out[j] = kNoToken;
            else if (j != n) out[j] = j < n ? a.draft_tokens[begin + j] : kNoToken;
        }
        if (threadIdx.x == 0) a.accepted[b] = bad ? kNoToken : n;
    }
}

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
        if ((e = cudaFuncSetAttribute(k_mass, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
        if ((e = cudaFuncSetAttribute(k_mass, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        if ((e = cudaFuncSetAttribute(k_draw, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        d.clusters[1] = d.sms;
        for (int c = 2; c <= kMaxCluster; c *= 2) {
            cudaLaunchConfig_t cfg;
            cudaLaunchAttribute attr[2];
            configure(cfg, attr, dim3((unsigned)c), kMassThreads, smem, c, nullptr);
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, k_mass, &cfg) != cudaSuccess) {
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
    a.minus_zero = 0x8000000080000000ull;
    a.rows = static_cast<RowPart *>(workspace);
    a.total = drafts + requests + (a.draft ? drafts : 0);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DeviceSetup dev;
    cudaError_t e = device_setup(dev);
    if (e != cudaSuccess) return fail(LLMX_ERR_CUDA, std::string("device set-up: ") + cudaGetErrorString(e));
    // CTAs per row: the split with the least work for the busiest CTA, counting a
    // row's exchange of maxima as a chunk and a half; a row's share has to fit the ring with some
    // chunks to spare, else it is loaded twice.
    const int chunks = (int)((vocab + kChunk - 1) / kChunk);
    double best = 0;
    for (int split = 1; split <= kMaxCluster; split *= 2) {
        if (dev.clusters[split] == 0 || (split > 1 && chunks < split)) continue;
        const int share = (chunks + split - 1) / split;
        const bool fits = share <= kMaxRing;
        const uint32_t rounds = (a.total + dev.clusters[split] - 1) / dev.clusters[split];
        const double cost = rounds * ((double)chunks / split * (fits ? 1 : 2) + 1.5) + (share + 3 > kMaxRing ? 0.3 * rounds * share : 0);
        if (a.split == 0 || cost < best) {
            best = cost;
            a.split = split;
            a.resident = fits;
        }
    }
    a.ring = std::min(kMaxRing, std::max(2, 2 * ((chunks + a.split - 1) / a.split) + 1));
    if (!a.resident) a.ring = kMaxRing;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    const uint32_t groups = std::min<uint32_t>(a.total, (uint32_t)dev.clusters[a.split]);
    configure(cfg, attr, dim3(groups * a.split), kMassThreads, (size_t)a.ring * kChunkBytes, a.split, s);
    e = cudaLaunchKernelEx(&cfg, k_mass, a);
    if (e != cudaSuccess) return fail(LLMX_ERR_CUDA, std::string("k_mass: ") + cudaGetErrorString(e));
    DrawArgs d{a, 1};
    while (d.split < kMaxCluster && requests * d.split * 2 <= (uint32_t)dev.sms * 2 && vocab >= 2048u * d.split) d.split *= 2;
    configure(cfg, attr, dim3(requests * d.split), kDrawThreads, 0, d.split, s);
    e = cudaLaunchKernelEx(&cfg, k_draw, d);
    if (e != cudaSuccess) return fail(LLMX_ERR_CUDA, std::string("k_draw: ") + cudaGetErrorString(e));
    return LLMX_OK;
}
