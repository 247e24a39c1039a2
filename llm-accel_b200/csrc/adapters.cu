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
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <new>
#include <string>

#include "llmx.h"
#include "device_util.cuh"
#include "fixed.cuh"
#include "kernels.cuh"

struct llmx_adapters {
    int dev = 0;
    uint32_t in_dim = 0, out_dim = 0, slots = 0, max_rank = 0, max_rows = 0;
    int16_t *weight = nullptr;  // [out_dim][in_dim]
    int16_t *down = nullptr;    // [slots][max_rank][in_dim]
    int16_t *up = nullptr;      // [slots][out_dim][max_rank]
    int32_t *rank = nullptr;    // [slots]
    int32_t *scale = nullptr;   // [slots]
    int16_t *t = nullptr;       // [max_rows][max_rank]
    int *error = nullptr;
    uint64_t bytes = 0;
};

namespace {

using namespace llmx;

constexpr uint32_t kMaxIn = 32768, kMaxOut = 1u << 22, kMaxSlots = 65536, kMaxRank = 128, kMaxCallRows = 65536;

struct Call {
    const int16_t *x;
    size_t ld_x;
    const int32_t *slot;
    void *out;
    size_t ld_out;
    uint32_t rows;
    int wide;
};

static __device__ __forceinline__ int slot_of(const llmx_adapters &h, const Call &c, uint32_t row) {
    if (!c.slot) return -1;
    const int a = c.slot[row];
    return a >= 0 && a < (int)h.slots && h.rank[a] > 0 ? a : -1;
}

// t of one row: one warp per rank.
__global__ void __launch_bounds__(256) k_down(const llmx_adapters h, const Call c) {
    const uint32_t row = blockIdx.x;
    const int a = slot_of(h, c, row);
    if (a < 0) return;
    const int16_t *x = c.x + row * c.ld_x;
    const int lane = threadIdx.x & 31;
    for (int j = threadIdx.x >> 5; j < h.rank[a]; j += blockDim.x >> 5) {
        const int16_t *w = h.down + ((size_t)a * h.max_rank + j) * h.in_dim;
        int64_t s = 0;
        for (uint32_t k = lane; k < h.in_dim; k += 32) s += (int32_t)x[k] * (int32_t)w[k];
        for (int o = 16; o; o >>= 1) s += shfl_xor64(s, o);
        if (lane == 0) h.t[(size_t)row * h.max_rank + j] = (int16_t)sat16(rnd(s * h.scale[a], 24));
    }
}

// One warp per (row, output).
__global__ void __launch_bounds__(256) k_up(const llmx_adapters h, const Call c) {
    const int lane = threadIdx.x & 31;
    const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x >> 5);
    for (uint64_t i = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < (uint64_t)c.rows * h.out_dim;
         i += warps) {
        const uint32_t n = (uint32_t)(i / c.rows), row = (uint32_t)(i - (uint64_t)n * c.rows);
        const int a = slot_of(h, c, row);
        const int16_t *x = c.x + row * c.ld_x, *w = h.weight + (size_t)n * h.in_dim;
        int64_t s = 0;
        for (uint32_t k = lane; k < h.in_dim; k += 32) s += (int32_t)x[k] * (int32_t)w[k];
        if (a >= 0)
            for (int j = lane; j < h.rank[a]; j += 32)
                s += (int32_t)h.t[(size_t)row * h.max_rank + j] *
                     (int32_t)h.up[((size_t)a * h.out_dim + n) * h.max_rank + j];
        for (int o = 16; o; o >>= 1) s += shfl_xor64(s, o);
        if (lane == 0) {
            const int32_t q = sat32(rnd(s, 4));
            if (c.wide) static_cast<int32_t *>(c.out)[row * c.ld_out + n] = q;
            else static_cast<int16_t *>(c.out)[row * c.ld_out + n] = (int16_t)sat16(rnd(q, 8));
        }
    }
}

// up [out_dim][rank] -> [out_dim][max_rank]
__global__ void k_set_up(int16_t *dst, const int16_t *src, uint32_t out_dim, uint32_t max_rank, uint32_t rank) {
    const uint64_t n = (uint64_t)out_dim * rank;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (uint64_t)gridDim.x * blockDim.x)
        dst[i / rank * max_rank + i % rank] = src[i];
}
__global__ void k_set_slot(int32_t *ranks, int32_t *scales, uint32_t slot, int32_t rank, int32_t scale) {
    ranks[slot] = rank;
    scales[slot] = scale;
}

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
    int before = -1;
    cudaError_t err;
    explicit DeviceScope(int dev) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != dev) err = cudaSetDevice(dev);
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

void release(llmx_adapters *h) {
    cudaFree(h->weight);
    cudaFree(h->down);
    cudaFree(h->up);
    cudaFree(h->rank);
    cudaFree(h->scale);
    cudaFree(h->t);
    cudaFree(h->error);
    delete h;
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
    h->max_rank = slots ? max_rank : 1;
    h->max_rows = max_rows;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto get = [&](auto **p, size_t n) {
        h->bytes += n;
        return cudaMalloc(reinterpret_cast<void **>(p), n);
    };
    const size_t ns = slots ? slots : 1;
    cudaError_t e;
    if ((e = get(&h->weight, (size_t)out_dim * in_dim * 2)) != cudaSuccess ||
        (e = get(&h->down, (size_t)slots * h->max_rank * in_dim * 2 + 16)) != cudaSuccess ||
        (e = get(&h->up, (size_t)slots * h->max_rank * out_dim * 2 + 16)) != cudaSuccess ||
        (e = get(&h->rank, ns * 4)) != cudaSuccess || (e = get(&h->scale, ns * 4)) != cudaSuccess ||
        (e = get(&h->t, (size_t)max_rows * h->max_rank * 2)) != cudaSuccess || (e = get(&h->error, 4)) != cudaSuccess ||
        (e = cudaMemsetAsync(h->rank, 0, ns * 4, s)) != cudaSuccess ||
        (e = cudaMemsetAsync(h->error, 0, 4, s)) != cudaSuccess ||
        (e = cudaMemcpyAsync(h->weight, weight, (size_t)out_dim * in_dim * 2, cudaMemcpyDeviceToDevice, s)) != cudaSuccess) {
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
    cudaError_t e = cudaSuccess;
    if (rank) {
        e = cudaMemcpyAsync(h->down + (size_t)slot * h->max_rank * h->in_dim, down, (size_t)rank * h->in_dim * 2,
                            cudaMemcpyDeviceToDevice, s);
        if (e != cudaSuccess) return cuda_fail("set", e);
        k_set_up<<<1024, 256, 0, s>>>(h->up + (size_t)slot * h->max_rank * h->out_dim, up, h->out_dim, h->max_rank, rank);
    }
    k_set_slot<<<1, 1, 0, s>>>(h->rank, h->scale, slot, (int32_t)rank, scale);
    e = cudaGetLastError();
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
    const Call c{x, ld_x, h->slots ? slot : nullptr, out, ld_out, rows, wide};
    if (c.slot) k_down<<<rows, 256, 0, s>>>(*h, c);
    k_up<<<148 * 8, 256, 0, s>>>(*h, c);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LLMX_OK : cuda_fail("project", e);
}

extern "C" int llmx_adapters_error(llmx_adapters *h, void *stream) {
    if (!h) return fail(LLMX_ERR_ARG, "null handle");
    DeviceScope scope(h->dev);
    if (scope.err != cudaSuccess) return cuda_fail("cudaSetDevice", scope.err);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int word = 0;
    cudaError_t e = cudaMemcpyAsync(&word, h->error, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(h->error, 0, 4, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return cuda_fail("error", e);
    return word ? fail(LLMX_ERR_TIMEOUT, "a kernel's bounded wait expired (code " + std::to_string(word) + ")") : LLMX_OK;
}

extern "C" uint64_t llmx_adapters_device_bytes(const llmx_adapters *h) { return h ? h->bytes : 0; }
