// Log probabilities of given tokens, with their rank, the rows' entropy and the most
// likely tokens, from Q16.16 logits.
//
// No counterpart in the LLM-ACCEL tree: its host takes the maximum only (lm_head_argmax,
// host/host_qwen_8x64.cpp:937-977).  For a row z at temperature T, with m its maximum
// and d_v = (m - z_v) / (2^16 T):
//   rest = sum of exp(-d_v) over all tokens but one maximum
//   logprob(v) = -d_v - log1p(rest)
//   entropy    = log1p(rest) + sum of d_v exp(-d_v) / (1 + rest)
// so that nothing cancels where one token has nearly all the probability.
//
// Two launches.  k_rows reads the logits once.  All rows are one line of chunks of 512 logits, cut
// into runs, one per warp; for every row that its run touches a warp leaves a
// part: the maximum, both sums relative to it (binary32, of 16 terms at a time) and the tokens
// ahead of the given one; and every chunk's maximum.  k_rows_join adds up a row's parts, in
// binary64 and in order, so a result depends on no timing.
//
// The most likely tokens need no more of the first launch than the chunks' maxima: the k best tokens
// lie in the k best chunks (by maximum, then by index: every chunk has a token that is ahead of
// whatever lies in a chunk behind it), which k_rows_join reads again.  A warp holds the best 64-bit keys
// (logit, then the lower index) in order, one a lane; keys above the least of them go to a buffer in
// shared memory, of which 32 at a time are sorted over the lanes and merged.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <string>

#include "llmx.h"
#include "device_util.cuh"
#include "kernels.cuh"

namespace {

using llmx::pdl_trigger;
using llmx::pdl_wait;

constexpr int kExcluded = INT_MIN;
constexpr uint32_t kNone = 0xffffffffu;
constexpr uint32_t kMaxVocab = 1u << 22, kMaxRows = 1u << 20, kMaxTop = 32;
constexpr float kMinTemperature = 1e-6f;  // at or below: the first maximum alone
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kChunk = 512;               // logits: four 16-byte loads a lane
constexpr uint32_t kMaxCtas = 592;        // of k_rows: four on each of 148 SMs

// What a warp leaves of a row.
struct __align__(16) Part {
    int32_t top;      // maximum; kExcluded: nothing but excluded tokens
    uint32_t ahead;   // tokens ahead of the given one
    float rest, sum;  // of exp(-d) and of log2(e) d exp(-d), without one maximum
};

struct Call {
    const int32_t *logits;
    size_t ld;
    uint32_t vocab, rows, top;
    const uint32_t *tokens;
    const float *temperature;
    float *logprob;
    uint32_t *rank;
    float *entropy;
    uint32_t *top_tokens;
    float *top_logprobs;
    // Parts of a warp's rows lie one after another, and those of a row's warps too: warp w's part of row r is
    // number w + r, and on the way from one to the next either w or r grows by one.
    Part *parts;
    int32_t *maxima;       // [rows][chunks]
    uint32_t chunks;       // of a row
    uint32_t warps;        // of k_rows; warp w has chunks w * all / warps to (w + 1) * all / warps, one or more
};

static __device__ __forceinline__ bool is_greedy(float t) { return !(t > kMinTemperature); }

static __device__ __forceinline__ unsigned long long key_of(int z, uint32_t token) {
    return (unsigned long long)((uint32_t)z ^ 0x80000000u) << 32 | (kNone - token);
}
static __device__ __forceinline__ int logit_of(unsigned long long key) { return (int)((uint32_t)(key >> 32) ^ 0x80000000u); }

static __device__ __forceinline__ unsigned long long shfl64(unsigned long long v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// One step of a sorting network: lanes whose index has `bit` clear keep the larger of the two
// (down) or the smaller.
static __device__ __forceinline__ unsigned long long step64(unsigned long long v, int bit, bool down) {
    const unsigned long long o = shfl64(v, bit);
    const bool first = (threadIdx.x & bit) == 0;
    return (first == down) == (o > v) ? o : v;
}
// 32 keys over the lanes, sorted from the largest.
static __device__ __forceinline__ unsigned long long sort64(unsigned long long v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int bit = size / 2; bit; bit /= 2) v = step64(v, bit, (lane & size) == 0 || size == 32);
    return v;
}
// The 32 largest of two sorted lists, sorted.
static __device__ __forceinline__ unsigned long long merge64(unsigned long long a, unsigned long long b) {
    const unsigned long long r = __shfl_sync(0xffffffffu, b, 31 - (threadIdx.x & 31));
    unsigned long long v = a > r ? a : r;
#pragma unroll
    for (int bit = 16; bit; bit /= 2) v = step64(v, bit, true);
    return v;
}

// The best keys that a warp has met.
struct Best {
    unsigned long long list;  // sorted over the lanes; 0: none
    unsigned long long *buf;  // [64] in shared memory, the warp's own
    int count;                // in it
    uint32_t top;

    __device__ void start(unsigned long long *buffer, uint32_t n) {
        list = 0;
        buf = buffer;
        count = 0;
        top = n;
    }
    // The least key of the list: what does not exceed it stays out.
    __device__ unsigned long long least() const { return __shfl_sync(0xffffffffu, list, (int)top - 1); }
    __device__ void flush() {
        const int lane = threadIdx.x & 31;
        __syncwarp();
        const unsigned long long k = lane < count ? buf[lane] : 0;
        const unsigned long long rest = lane + 32 < count ? buf[lane + 32] : 0;
        __syncwarp();
        if (lane + 32 < count) buf[lane] = rest;
        count = max(count - 32, 0);
        list = merge64(list, sort64(k));
    }
    // By all lanes; `in`: this lane's key belongs in.
    __device__ void push(bool in, unsigned long long key) {
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        if (!who) return;
        if (in) buf[count + __popc(who & ((1u << (threadIdx.x & 31)) - 1))] = key;
        count += __popc(who);
        if (count >= 32) flush();
    }
    __device__ void finish() {
        while (count > 0) flush();
    }
};

// Rows are taken from the 16-byte boundary at or before their start on, so that a chunk is read by four
// 16-byte loads a lane wherever the row starts: token v of a row is place v + shift.
static __device__ __forceinline__ uint32_t shift_of(const int32_t *row) { return (uint32_t)((uintptr_t)row >> 2) & 3u; }
// Places i0 + 128 j + 4 lane .. + 3 of a row, excluded tokens in place of those that are not there.
static __device__ __forceinline__ void load(const int32_t *row, uint32_t vocab, uint32_t i0, int (&z)[16]) {
    const uint32_t shift = shift_of(row), first = i0 + 4 * (threadIdx.x & 31);
    if (i0 >= shift && i0 + kChunk - shift <= vocab) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            asm volatile("ld.global.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(z[4 * j]), "=r"(z[4 * j + 1]), "=r"(z[4 * j + 2]), "=r"(z[4 * j + 3])
                         : "l"(row - shift + first + 128 * j)
                         : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint32_t v = first + 128 * (i / 4) + i % 4 - shift;
            z[i] = kExcluded;
            if (v < vocab) z[i] = __ldcg(row + v);  // (one in front of the row is far beyond it)
        }
    }
}

// Pairs of binary32 numbers.
using f32x2 = unsigned long long;
static __device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
static __device__ __forceinline__ void unpack2(f32x2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
static __device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
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
static __device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// A warp's run: a chunk is on its way while the one before is added up.  A term costs a difference, its conversion, the exponent in
// two parts, 2^x and two sums, of which pairs share an instruction (packed binary32).  512 rows of 151936: 56 us for 311 MB
// (5.6 TB/s, 85 % of a copy), 61 % of the issue slots; four CTAs an SM would need 64 registers, which spill
// (59 us in all became 63).  64 rows: 14 us for 39 MB, half of it the way to the first chunk and from the last.
__global__ void __launch_bounds__(kThreads, 3) k_rows(const Call c) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned long long w = (unsigned long long)blockIdx.x * kWarps + warp;
    const unsigned long long all = (unsigned long long)c.chunks * c.rows, begin = w * all / c.warps, end = (w + 1) * all / c.warps;
    pdl_wait();
    pdl_trigger();
    if (w >= c.warps) return;
    uint32_t r = (uint32_t)(begin / c.chunks), chunk = (uint32_t)(begin - (unsigned long long)r * c.chunks);
    const int32_t *row = c.logits + (size_t)r * c.ld;
    int next[16];
    load(row, c.vocab, chunk * kChunk, next);
    for (unsigned long long at = begin; at < end;) {
        // one row's share of the run
        const uint32_t share = (uint32_t)min((unsigned long long)(c.chunks - chunk), end - at);
        const float temperature = c.temperature ? c.temperature[r] : 1.0f;
        const bool greedy = is_greedy(temperature);
        // -log2(e) / 2^16 / T in two parts: a rounded one alone would turn all terms the same way
        const double scale = greedy ? 0.0 : -1.4426950408889634 / 65536.0 / (double)temperature;
        const float s_hi = (float)scale, s_lo = (float)(scale - (double)s_hi);
        const f32x2 hi2 = pack2(s_hi, s_hi), lo2 = pack2(s_lo, s_lo);
        const uint32_t token = c.tokens ? c.tokens[r] : kNone;
        const int mine = token < c.vocab ? __ldcg(row + token) : kExcluded;
        const uint32_t place = token + shift_of(row);
        int m = kExcluded;   // of the warp
        bool far = false;    // an excluded token's term is 0 by itself, so far away is it
        float rest = 0, sum = 0;
        uint32_t ahead = 0;
        for (uint32_t n = 0; n < share; n++) {
            int z[16];
#pragma unroll
            for (int i = 0; i < 16; i++) z[i] = next[i];
            const uint32_t i0 = (chunk + n) * kChunk;
            if (n + 1 < share) load(row, c.vocab, i0 + kChunk, next);
            else if (at + share < end) load(row + c.ld, c.vocab, 0, next);
            int most = z[0];
#pragma unroll
            for (int i = 1; i < 16; i++) most = max(most, z[i]);
            const int top = __reduce_max_sync(0xffffffffu, most);
            if (lane == 0) c.maxima[(size_t)r * c.chunks + chunk + n] = top;
            if (top == kExcluded) continue;
            if (top >= mine && mine != kExcluded) {
                const uint32_t first = i0 + 4 * lane;
                if (place - i0 < (uint32_t)kChunk) {
#pragma unroll
                    for (int i = 0; i < 16; i++) ahead += z[i] > mine || (z[i] == mine && first + 128 * (i / 4) + i % 4 < place);
                } else {
                    const int over = place < i0 ? mine : mine - 1;  // in front of the token equal ones are ahead
#pragma unroll
                    for (int i = 0; i < 16; i++) ahead += z[i] > over;
                }
            }
            if (greedy) {
                m = max(m, top);
                continue;
            }
            if (top > m) {
                if (m != kExcluded) {  // the old maximum becomes an ordinary token
                    const float d = (float)((uint32_t)top - (uint32_t)m);
                    const float e = fmaf(d, s_hi, d * s_lo), f = exp2f(e);
                    if (lane == 0) rest += 1.0f;  // (it is 0 away from itself)
                    sum = f * fmaf(rest, e, sum);
                    rest *= f;
                }
                m = top;
                far = (float)((uint32_t)m ^ 0x80000000u) * s_hi < -150.0f;
                // The new one stays out: one lane takes those that it has for excluded and counts all but one.
                const uint32_t who = __ballot_sync(0xffffffffu, most == top);
                const bool here = lane == __ffs(who) - 1;
                const int gone = here ? top : kExcluded;
                int count = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    count += z[i] == gone;
                    z[i] = z[i] == gone ? kExcluded : z[i];
                }
                if (here) rest += (float)(count - 1);
            }
            if (far) {
                f32x2 r2 = 0, s2 = 0;
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const f32x2 d = pack2((float)((uint32_t)m - (uint32_t)z[i]), (float)((uint32_t)m - (uint32_t)z[i + 1]));
                    const f32x2 e = fma2(d, hi2, mul2(d, lo2));
                    float e0, e1;
                    unpack2(e, e0, e1);
                    const f32x2 x = pack2(exp2_fast(e0), exp2_fast(e1));
                    r2 = add2(r2, x);
                    s2 = fma2(x, e, s2);
                }
                float a, b;
                unpack2(r2, a, b);
                rest += a + b;
                unpack2(s2, a, b);
                sum += a + b;
            } else {
                float r16 = 0, s16 = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float d = (float)((uint32_t)m - (uint32_t)z[i]), e = fmaf(d, s_hi, d * s_lo);
                    const float x = z[i] == kExcluded ? 0.0f : exp2_fast(e);
                    r16 += x;
                    s16 = fmaf(x, e, s16);
                }
                rest += r16;
                sum += s16;
            }
        }
        ahead = __reduce_add_sync(0xffffffffu, ahead);
#pragma unroll
        for (int o = 16; o; o /= 2) {
            rest += __shfl_xor_sync(0xffffffffu, rest, o);
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (lane == 0) c.parts[w + r] = Part{m, ahead, rest, -sum};
        at += share;
        chunk += share;
        if (chunk == c.chunks) {
            chunk = 0;
            r++;
            row += c.ld;
        }
    }
}

// The warps' lists put together, in the first warp.
static __device__ __forceinline__ unsigned long long gather(unsigned long long list, unsigned long long (&lists)[kWarps][32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int half = kWarps / 2; half; half /= 2) {
        if (warp >= half && warp < 2 * half) lists[warp][lane] = list;
        __syncthreads();
        if (warp < half) list = merge64(list, lists[warp + half][lane]);
    }
    return list;
}

constexpr int kCandidates = 256;  // tokens whose places are found by comparing all with all

// A row per CTA.  Latency bounds it (10 to 13 us with cold caches): the chunks' maxima, the best ones' order over the lanes
// and warps, their logits, binary64 exponents and logarithm, one after another.  With 16 warps, each for two of the
// best chunks, 77 rows of 32003 took 12.7 us in all for 9.8.
__global__ void __launch_bounds__(kThreads) k_rows_join(const Call c) {
    __shared__ unsigned long long buffers[kWarps][64];
    __shared__ unsigned long long lists[kWarps][32];
    __shared__ unsigned long long chosen[32], candidates[kCandidates];
    __shared__ double rests[kWarps], sums[kWarps];
    __shared__ uint32_t aheads[kWarps], withs[kWarps], found;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) found = 0;
    const uint32_t r = blockIdx.x;
    const int32_t *row = c.logits + (size_t)r * c.ld;
    // This launch starts once every CTA of k_rows has waited for what is before it, so that the call's arguments can be
    // read, through the L2, before its own wait.
    const float temperature = c.temperature ? __ldcg(c.temperature + r) : 1.0f;
    const uint32_t token = c.tokens ? __ldcg(c.tokens + r) : kNone;
    const int mine = token < c.vocab ? __ldcg(row + token) : kExcluded;
    const bool greedy = is_greedy(temperature);
    const double scale = greedy ? 0.0 : 1.4426950408889634 / 65536.0 / (double)temperature, step = greedy ? 0.0 : 1.0 / (65536.0 * (double)temperature);
    // the warps of k_rows that had a share of this row
    const unsigned long long all = (unsigned long long)c.chunks * c.rows;
    auto warp_of = [&](unsigned long long chunk) { return ((chunk + 1) * c.warps - 1) / all; };
    const unsigned long long first = warp_of((unsigned long long)r * c.chunks), last = warp_of((unsigned long long)(r + 1) * c.chunks - 1);
    const int parts = (int)(last - first + 1);
    const Part *part = c.parts + first + r;
    const int32_t *maxima = c.maxima + (size_t)r * c.chunks;
    pdl_wait();
    pdl_trigger();
    // (all loads are on their way before the first is used)
    const Part mine_part = (int)threadIdx.x < parts ? part[threadIdx.x] : Part{kExcluded, 0, 0, 0};
    auto key_at = [&](uint32_t i) -> unsigned long long {
        const int z = i < c.chunks ? maxima[i] : kExcluded;
        return z == kExcluded ? 0 : key_of(z, i);
    };
    const unsigned long long key0 = key_at(threadIdx.x), key1 = key_at(kThreads + threadIdx.x);
    // The best chunks.
    unsigned long long list;
    if (c.top <= 1) {  // the best one: maxima of keys
        unsigned long long k = key0 > key1 ? key0 : key1;
        for (uint32_t i = 2 * kThreads + threadIdx.x; i < c.chunks; i += kThreads) k = max(k, key_at(i));
        const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
        const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
        if (lane == 0) lists[warp][0] = (unsigned long long)hi << 32 | lo;
        __syncthreads();
        list = 0;
        for (int w = 0; w < kWarps; w++) list = max(list, lists[w][0]);
        if (threadIdx.x == 0) chosen[0] = list;
    } else {
        Best best;
        best.start(buffers[warp], c.top);
        best.list = sort64(key0);
        unsigned long long bound = best.least();
        best.push(key1 > bound, key1);
        for (uint32_t i = 2 * kThreads + warp * 32; i < c.chunks; i += kThreads) {
            const unsigned long long key = key_at(i + lane);
            best.push(key > bound, key);
            bound = max(bound, best.least());
        }
        best.finish();
        list = gather(best.list, lists);
        if (warp == 0) chosen[lane] = list;
    }
    __syncthreads();
    // Their logits, on their way while the parts are added up; four chunks a warp at most.
    const unsigned long long most = chosen[0], least = c.top ? chosen[c.top - 1] : 0;
    int z[16];
    const bool any = (uint32_t)warp < c.top && chosen[min(warp, 31)] != 0;
    if (any) load(row, c.vocab, (kNone - (uint32_t)chosen[warp]) * kChunk, z);
    const int m = most ? logit_of(most) : kExcluded;
    // One maximum stays out of the sums: the parts that have it count one less.
    double rest = 0, sum = 0;
    uint32_t ahead = 0;
    uint32_t with = 0;
    auto add = [&](const Part &p) {
        ahead += p.ahead;
        if (p.top == kExcluded || greedy) return;
        if (p.top == m) {
            with++;
            rest += (double)p.rest;
            sum += (double)p.sum;
        } else {
            const double e = (double)((uint32_t)m - (uint32_t)p.top) * scale, f = exp2(-e), all = (double)p.rest + 1.0;
            rest += f * all;
            sum += f * ((double)p.sum + all * e);
        }
    };
    add(mine_part);
    for (int i = kThreads + threadIdx.x; i < parts; i += kThreads) add(part[i]);
#pragma unroll
    for (int o = 16; o; o /= 2) {
        rest += __shfl_xor_sync(0xffffffffu, rest, o);
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    with = __reduce_add_sync(0xffffffffu, with);
    if (lane == 0) {
        rests[warp] = rest;
        sums[warp] = sum;
        aheads[warp] = ahead;
        withs[warp] = with;  // (not in lists: gather writes there, below, while others may still add these up)
    }
    // The best tokens: the maximum of the last of the best chunks bounds them from below (any token with that
    // logit may be one).
    const unsigned long long bound = least ? (least >> 32 << 32) - 1 : 0;
    auto chunk_keys = [&](uint32_t i, auto use) {
        const uint32_t i0 = (kNone - (uint32_t)chosen[i]) * kChunk + 4 * lane - shift_of(row);
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const unsigned long long key = z[k] == kExcluded ? 0 : key_of(z[k], i0 + 128 * (k / 4) + k % 4);
            use(key > bound, key);
        }
    };
    for (uint32_t i = warp; i < c.top && chosen[i] != 0; i += kWarps) {
        if (i >= (uint32_t)kWarps) load(row, c.vocab, (kNone - (uint32_t)chosen[i]) * kChunk, z);
        chunk_keys(i, [&](bool in, unsigned long long key) {
            if (in) {
                const uint32_t at = atomicAdd(&found, 1u);
                if (at < (uint32_t)kCandidates) candidates[at] = key;
            }
        });
    }
    __syncthreads();
    double all_rest = 0, all_sum = 0;
    long long all_with = -1;
    ahead = 0;
    for (int i = 0; i < kWarps; i++) {
        all_rest += rests[i];
        all_sum += sums[i];
        ahead += aheads[i];
        all_with += withs[i];
    }
    if (greedy || m == kExcluded) all_with = 0;
    rest = all_rest + (double)all_with;
    sum = all_sum;
    const double log_sum = log1p(rest);
    // of a token that is not excluded
    auto logprob = [&](int z, bool ahead_of_all) -> float {
        if (greedy) return ahead_of_all ? 0.0f : -INFINITY;
        return (float)(-(double)((uint32_t)m - (uint32_t)z) * step - log_sum);
    };
    if (threadIdx.x == 0) {
        if (c.tokens) {
            c.logprob[r] = mine == kExcluded ? -INFINITY : logprob(mine, ahead == 0);
            c.rank[r] = mine == kExcluded ? kNone : ahead;
        }
        c.entropy[r] = greedy || m == kExcluded ? 0.0f : (float)(log_sum + 0.6931471805599453 * sum / (1.0 + rest));
    }
    if (c.top == 0) return;
    auto put = [&](uint32_t place, unsigned long long key) {
        c.top_tokens[(size_t)r * c.top + place] = key ? kNone - (uint32_t)key : kNone;
        c.top_logprobs[(size_t)r * c.top + place] = key ? logprob(logit_of(key), place == 0) : -INFINITY;
    };
    const uint32_t n = found;
    if (n <= (uint32_t)kCandidates) {
        if (threadIdx.x < n) {
            const unsigned long long key = candidates[threadIdx.x];
            uint32_t place = 0;
            for (uint32_t i = 0; i < n; i++) place += candidates[i] > key;
            if (place < c.top) put(place, key);
        }
        if (threadIdx.x >= n && threadIdx.x < c.top) put(threadIdx.x, 0);  // fewer than asked for
        return;
    }
    // many equal ones: in order, by warps
    Best best;
    best.start(buffers[warp], c.top);
    for (uint32_t i = warp; i < c.top && chosen[i] != 0; i += kWarps) {
        load(row, c.vocab, (kNone - (uint32_t)chosen[i]) * kChunk, z);
        unsigned long long most_key = 0;
        chunk_keys(i, [&](bool, unsigned long long key) { most_key = max(most_key, key); });
        // the top-th of the lanes' best bounds from below as well
        const unsigned long long t = __shfl_sync(0xffffffffu, sort64(most_key), (int)c.top - 1), floor = max(best.least(), t ? t - 1 : 0);
        chunk_keys(i, [&](bool in, unsigned long long key) { best.push(in && key > floor, key); });
    }
    best.finish();
    list = gather(best.list, lists);
    if (warp == 0 && lane < (int)c.top) put((uint32_t)lane, list);
}

// (of rows that may start anywhere)
uint64_t chunks_of(uint32_t rows, uint32_t vocab) { return (uint64_t)rows * ((vocab + 3 + kChunk - 1) / kChunk); }

// Bytes of the workspace in front of the chunks' maxima: the parts.
size_t maxima_at(uint32_t rows, uint32_t vocab) {
    const uint64_t warps = std::min<uint64_t>(chunks_of(rows, vocab), (uint64_t)kMaxCtas * kWarps);
    return ((warps + rows) * sizeof(Part) + 255) / 256 * 256;
}

int fail(int code, const std::string &msg) {
    llmx::set_last_error("token_logprobs: " + msg);
    return code;
}
int cuda_fail(const char *what, cudaError_t e) {
    (void)cudaGetLastError();
    return fail(LLMX_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

cudaError_t launch(const void *fn, unsigned grid, const Call &call, cudaStream_t s) {
    Call copy = call;
    void *args[] = {&copy};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace

extern "C" size_t llmx_logprobs_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t top) {
    (void)top;  // the best tokens pass through no memory
    return maxima_at(rows, vocab) + (chunks_of(rows, vocab) * sizeof(int32_t) + 255) / 256 * 256;
}

extern "C" int llmx_token_logprobs(const int32_t *logits, size_t ld, uint32_t vocab, uint32_t rows, const uint32_t *tokens,
                                   const float *temperature, uint32_t top, float *logprob, uint32_t *rank, float *entropy,
                                   uint32_t *top_tokens, float *top_logprobs, void *workspace, size_t workspace_bytes,
                                   void *stream) {
    if (vocab == 0 || vocab > kMaxVocab) return fail(LLMX_ERR_ARG, "vocab must be 1..2^22, got " + std::to_string(vocab));
    if (rows > kMaxRows) return fail(LLMX_ERR_ARG, "rows must be at most 2^20, got " + std::to_string(rows));
    if (top > kMaxTop) return fail(LLMX_ERR_ARG, "top must be at most 32, got " + std::to_string(top));
    if (ld == 0) ld = vocab;
    if (ld < vocab) return fail(LLMX_ERR_ARG, "the row stride is smaller than vocab");
    if (rows == 0) return LLMX_OK;
    if (!logits || !entropy || !workspace) return fail(LLMX_ERR_ARG, "null pointer");
    if (tokens && (!logprob || !rank)) return fail(LLMX_ERR_ARG, "null pointer with tokens");
    if (top && (!top_tokens || !top_logprobs)) return fail(LLMX_ERR_ARG, "null pointer with top > 0");
    if (((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)temperature | (uintptr_t)logprob | (uintptr_t)rank | (uintptr_t)entropy |
         (uintptr_t)top_tokens | (uintptr_t)top_logprobs) & 3u)
        return fail(LLMX_ERR_ARG, "a pointer is not aligned to its element");
    if ((uintptr_t)workspace & 255u) return fail(LLMX_ERR_ARG, "workspace must be 256-byte aligned");
    if (workspace_bytes < llmx_logprobs_workspace_bytes(rows, vocab, top))
        return fail(LLMX_ERR_ARG, "workspace too small: " + std::to_string(workspace_bytes) + " bytes");
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_fail("device", e);
    Call c{};
    c.logits = logits;
    c.ld = ld;
    c.vocab = vocab;
    c.rows = rows;
    c.top = top;
    c.tokens = tokens;
    c.temperature = temperature;
    c.logprob = logprob;
    c.rank = rank;
    c.entropy = entropy;
    c.top_tokens = top_tokens;
    c.top_logprobs = top_logprobs;
    c.parts = static_cast<Part *>(workspace);
    c.maxima = reinterpret_cast<int32_t *>(static_cast<unsigned char *>(workspace) + maxima_at(rows, vocab));
    const bool aligned = (((uintptr_t)logits | (ld * 4)) & 15u) == 0;
    c.chunks = (vocab + (aligned ? 0 : 3) + kChunk - 1) / kChunk;
    const uint64_t all = (uint64_t)rows * c.chunks, most = std::min<uint64_t>((uint64_t)sms * 3, kMaxCtas) * kWarps;
    // All warps that there can be at once share the chunks, unless runs of one length leave few of them idle: those make
    // fewer parts.  Measured both ways at 2 to 1000 rows of 32003 to 256000, 5 best (122 calls): the 35 where all share take up to 1.9 us
    // less that way, all but one (64 rows of 151936 14.8 for 16.0, 128 of 50257 12.2 for 13.2, 64 of 256000 18.4 for 20.2; 77 of 50257
    // 10.8 for 10.7).  Of the others, those with runs of 2 may be ahead either way by 0.6 us (64 of 32003 9.0 and 9.5 if all shared,
    // 64 of 50257 10.5 and 9.9); where less than 1/16 is idle, all sharing would be from 1.4 us less to 1.0 more, mostly 0.4 less.
    const uint64_t per = (all + most - 1) / most, even = (all + per - 1) / per;
    c.warps = (uint32_t)(per > 2 && even * 16 < most * 15 ? most : even);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    e = launch((const void *)k_rows, (c.warps + kWarps - 1) / kWarps, c, s);
    if (e == cudaSuccess) e = launch((const void *)k_rows_join, rows, c, s);
    return e == cudaSuccess ? LLMX_OK : cuda_fail("launch", e);
}
