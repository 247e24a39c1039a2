// Verification of drafted tokens against the target's probabilities, from
// random numbers that the caller gives.
//
// No counterpart in the LLM-ACCEL tree: its host decodes greedily
// (lm_head_argmax, host/host_qwen_8x64.cpp:937-977) and never forms
// probabilities.  The arithmetic follows the path's rule that a result is a
// whole number which no order of summation can change: a logit becomes a
// 32-bit weight, sums of weights are 64-bit integers, probabilities are Q0.40
// integers, and both the accept test and the draw compare integers.
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <string>

#include "llmx.h"
#include "device_util.cuh"
#include "kernels.cuh"

namespace {

constexpr int kExcluded = INT_MIN;
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr uint32_t kMaxVocab = 1u << 22, kMaxRequests = 65535, kMaxDrafts = 1023, kMaxTotal = 1u << 24;
constexpr float kMinTemperature = 1e-6f;  // at or below: greedy
constexpr float kLog2e16 = 0x1.715476p-16f;  // log2(e) / 2^16: Q16.16 differences to octaves

// What a row of logits is reduced to.
struct RowMass {
    int32_t top;       // maximum
    uint32_t first;    // its first position
    float scale;       // log2(e) / 2^16 / T; negative: greedy
    uint32_t inverse;  // floor(2^62 / (S >> h)), 0 when nothing is left
    int32_t shift;     // 22 + h
    uint32_t pad[3];
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
    RowMass *mass;        // [drafts + requests] target rows, then [drafts] draft rows
    uint64_t *p_token;    // [drafts][2]: P and Q of each drafted token
};

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

// floor(2^31 * 2^-e), e = (top - z) * scale capped at 100, every float step
// rounded on its own (no contraction), so that the weight is the same integer
// wherever it is computed.  2^x on [-1/2, 1/2] is 1 + x q(x) with q of degree 4
// fitted to the relative error at Chebyshev points: below 2e-7 with the
// rounding of its steps.  The cap keeps the round-by-constant trick in range; beyond
// e = 32 the weight is 0 anyway.
static __device__ __forceinline__ uint32_t soft_weight(int32_t z, int32_t top, float scale) {
    const float d = __uint2float_rn((uint32_t)top - (uint32_t)z);
    const float e = fminf(__fmul_rn(d, scale), 100.0f);
    const float m = __fadd_rn(e, 12582912.0f);  // 1.5 * 2^23: round to nearest even in the low bits
    const float f = __fsub_rn(__fsub_rn(m, 12582912.0f), e);
    float p = __fadd_rn(__fmul_rn(f, 0x1.5bba12p-10f), 0x1.3cea88p-7f);
    p = __fadd_rn(__fmul_rn(p, f), 0x1.c6b752p-5f);
    p = __fadd_rn(__fmul_rn(p, f), 0x1.ebf9bcp-3f);
    p = __fadd_rn(__fmul_rn(p, f), 0x1.62e42ap-1f);
    p = __fadd_rn(__fmul_rn(p, f), 1.0f);
    // times 2^(31 - i): i is what m's low bits hold above 0x4b400000
    const int i = __float_as_int(m) - 0x4b400000;
    const uint32_t w = __float2uint_rz(__int_as_float(__float_as_int(p) + ((31 - i) << 23)));
    return z == kExcluded ? 0u : w;
}
static __device__ __forceinline__ uint32_t row_weight(int32_t z, uint32_t v, const RowMass &r) {
    if (r.scale < 0.0f) return v == r.first && z != kExcluded ? 0x80000000u : 0u;
    return soft_weight(z, r.top, r.scale);
}
static __device__ __forceinline__ uint64_t row_share(uint32_t w, const RowMass &r) {
    return ((uint64_t)w * r.inverse) >> r.shift;
}
// floor(a * u / 2^32)
static __device__ __forceinline__ uint64_t mul_frac(uint64_t a, uint32_t u) {
    return __umul64hi(a, (uint64_t)u << 32);
}

// Reduction of one row by one block.
__global__ void __launch_bounds__(512) k_row_mass(const Args a) {
    const uint32_t targets = a.drafts + a.requests;
    const bool is_draft = blockIdx.x >= targets;
    const uint32_t row = is_draft ? blockIdx.x - targets : blockIdx.x;
    __shared__ uint32_t owner_s;
    __shared__ int32_t top_s[16];
    __shared__ uint32_t first_s[16];
    __shared__ unsigned long long sum_s[16];
    if (threadIdx.x == 0) owner_s = kNoToken;
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < a.requests; b += blockDim.x) {
        uint32_t begin, count;
        if (!request_range(a, b, begin, count)) continue;
        const uint32_t lo = is_draft ? begin : begin + b, n = is_draft ? count : count + 1;
        if (row >= lo && row < lo + n) owner_s = b;
    }
    __syncthreads();
    const uint32_t b = owner_s;
    if (b == kNoToken) return;
    const int32_t *z = is_draft ? a.draft + row * a.ld_draft : a.target + row * a.ld_target;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int32_t top = INT_MIN;
    uint32_t first = kNoToken;
    for (uint32_t v = threadIdx.x; v < a.vocab; v += blockDim.x) {
        const int32_t x = z[v];
        if (x > top || first == kNoToken) {
            top = x;
            first = v;
        }
    }
    for (int o = 16; o; o >>= 1) {
        const int32_t t = __shfl_xor_sync(~0u, top, o);
        const uint32_t f = __shfl_xor_sync(~0u, first, o);
        if (t > top || (t == top && f < first)) {
            top = t;
            first = f;
        }
    }
    if (lane == 0) {
        top_s[warp] = top;
        first_s[warp] = first;
    }
    __syncthreads();
    RowMass r{};
    r.top = top_s[0];
    r.first = first_s[0];
    for (int q = 1; q < nw; q++)
        if (top_s[q] > r.top || (top_s[q] == r.top && first_s[q] < r.first)) {
            r.top = top_s[q];
            r.first = first_s[q];
        }
    r.scale = row_scale(a.temperature[b]);
    unsigned long long sum = 0;
    for (uint32_t v = threadIdx.x; v < a.vocab; v += blockDim.x) sum += row_weight(z[v], v, r);
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) sum_s[warp] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    sum = 0;
    for (int q = 0; q < nw; q++) sum += sum_s[q];
    int h = 32 - __clzll((long long)sum);  // sum has 64 - clz bits; 32 remain
    h = h < 0 ? 0 : h;
    r.inverse = sum ? (uint32_t)((1ull << 62) / (sum >> h)) : 0u;
    r.shift = 22 + h;
    a.mass[(is_draft ? targets : 0u) + row] = r;
    // the drafted token's probability in this row
    const uint32_t j = is_draft ? row : row - b;
    if (is_draft || j < a.offsets[b + 1]) {
        const uint32_t x = a.draft_tokens[j];
        const uint64_t p = x < a.vocab ? row_share(row_weight(z[x], x, r), r) : 0;
        a.p_token[2 * (size_t)j + (is_draft ? 1 : 0)] = p;
        if (!a.draft) a.p_token[2 * (size_t)j + 1] = 1ull << 40;
    }
}

// Accept tests and the drawn token of one request by one block.
__global__ void __launch_bounds__(1024) k_draw(const Args a) {
    const uint32_t b = blockIdx.x;
    uint32_t *out = a.tokens + (size_t)b * (a.max_drafts + 1);
    uint32_t begin, count;
    if (!request_range(a, b, begin, count)) {
        for (uint32_t j = threadIdx.x; j <= a.max_drafts; j += blockDim.x) out[j] = kNoToken;
        if (threadIdx.x == 0) a.accepted[b] = kNoToken;
        return;
    }
    __shared__ uint32_t first_s, drawn_s;
    __shared__ unsigned long long sum_s[32], less_s[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        first_s = count;
        drawn_s = kNoToken;
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < count; j += blockDim.x) {
        const uint64_t p = a.p_token[2 * (size_t)(begin + j)], q = a.p_token[2 * (size_t)(begin + j) + 1];
        if (a.probs) {
            a.probs[2 * (size_t)(begin + j)] = p;
            a.probs[2 * (size_t)(begin + j) + 1] = q;
        }
        if (mul_frac(q, a.accept_u[begin + j]) >= p) atomicMin(&first_s, j);
    }
    __syncthreads();
    const uint32_t n = first_s;
    const uint32_t trow = begin + b + n, drow = begin + n;
    const int32_t *zt = a.target + trow * a.ld_target;
    const RowMass mt = a.mass[trow];
    const bool rejected = n < count, has_draft = a.draft != nullptr;
    const uint32_t x = rejected ? a.draft_tokens[drow] : kNoToken;
    const int32_t *zd = rejected && has_draft ? a.draft + drow * a.ld_draft : nullptr;
    RowMass md{};
    if (zd) md = a.mass[a.drafts + a.requests + drow];
    // warp w covers one contiguous run of the vocabulary
    const uint32_t per = ((a.vocab + 31) / 32 + 31) / 32 * 32;
    const uint32_t v0 = min(a.vocab, warp * per), v1 = min(a.vocab, v0 + per);
    auto rest = [&](uint32_t v, uint64_t p) -> uint64_t {
        if (!rejected) return p;
        const uint64_t q = zd ? row_share(row_weight(zd[v], v, md), md) : (v == x ? 1ull << 40 : 0);
        return p > q ? p - q : 0;
    };
    unsigned long long all = 0, less = 0;
    for (uint32_t v = v0 + lane; v < v1; v += 32) {
        const uint64_t p = row_share(row_weight(zt[v], v, mt), mt);
        all += p;
        less += rest(v, p);
    }
    for (int o = 16; o; o >>= 1) {
        all += __shfl_xor_sync(~0u, all, o);
        less += __shfl_xor_sync(~0u, less, o);
    }
    if (lane == 0) {
        sum_s[warp] = all;
        less_s[warp] = less;
    }
    __syncthreads();
    unsigned long long total = 0, total_less = 0;
    for (int q = 0; q < 32; q++) {
        total += sum_s[q];
        total_less += less_s[q];
    }
    const bool use_rest = rejected && total_less > 0;
    if (use_rest) total = total_less;
    const uint64_t point = mul_frac(total, a.sample_u[b]);
    unsigned long long below = 0;
    for (int q = 0; q < warp; q++) below += use_rest ? less_s[q] : sum_s[q];
    const unsigned long long mine = use_rest ? less_s[warp] : sum_s[warp];
    if (total && point >= below && point < below + mine) {  // one warp holds the point
        for (uint32_t v = v0; v < v1; v += 32) {
            unsigned long long s = 0;
            if (v + lane < v1) {
                s = row_share(row_weight(zt[v + lane], v + lane, mt), mt);
                if (use_rest) s = rest(v + lane, s);
            }
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long t = __shfl_up_sync(~0u, s, o);
                if (lane >= o) s += t;
            }
            const unsigned hit = __ballot_sync(~0u, below + s > point);
            if (hit) {
                if (lane == 0) drawn_s = v + (uint32_t)__ffs((int)hit) - 1;
                break;
            }
            below += __shfl_sync(~0u, s, 31);
        }
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j <= a.max_drafts; j += blockDim.x)
        out[j] = j < n ? a.draft_tokens[begin + j] : j == n ? drawn_s : kNoToken;
    if (threadIdx.x == 0) a.accepted[b] = n;
}

int fail(int code, const std::string &msg) {
    llmx::set_last_error("verify_drafts: " + msg);
    return code;
}

size_t mass_bytes(uint64_t rows) { return (rows * sizeof(RowMass) + 255) / 256 * 256; }

}  // namespace

extern "C" size_t llmx_verify_workspace_bytes(uint32_t requests, uint32_t drafts, uint32_t vocab) {
    (void)vocab;
    return mass_bytes(2ull * drafts + requests) + ((size_t)drafts * 16 + 255) / 256 * 256;
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
    a.mass = static_cast<RowMass *>(workspace);
    a.p_token = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + mass_bytes(2ull * drafts + requests));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint32_t rows = drafts + requests + (a.draft ? drafts : 0);
    k_row_mass<<<rows, 512, 0, s>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(LLMX_ERR_CUDA, std::string("k_row_mass: ") + cudaGetErrorString(e));
    k_draw<<<requests, 1024, 0, s>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return fail(LLMX_ERR_CUDA, std::string("k_draw: ") + cudaGetErrorString(e));
    return LLMX_OK;
}
