// grad_clip.cu -- the 2-norm over all elements of many tensors, and the tensors scaled down to a norm.
//
//   n = sqrt(sum g^2),  s = min(1, max_norm / (n + eps)),  out = g s
//
// The tensors' addresses and sizes are kernel parameters, so nothing is copied to the device and a call can be
// captured.  Each block leaves its share of the sum of squares as a 64-bit number in the workspace; the
// scaling kernel's blocks add them in a fixed order, so the result does not change from run to run.
#include <cuda_runtime.h>

#include <cstdint>

#include "dense_ops.h"
#include "nfx_internal.h"

namespace nfx {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16384;  // elements that a block takes at a time
constexpr int kPartBlocks = 592;

struct Entry {
    const void* src;
    void* dst;
    int64_t n;
    int64_t first;  // the tensor's first chunk
};
template <int CAP>
struct Table {
    Entry e[CAP];
    uint8_t src_type[CAP], dst_type[CAP];
    int count;
    int64_t chunks;
};
constexpr int kCap = 900;

// The tensor that chunk c belongs to (tensors without elements have no chunk).
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& t, int64_t c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].first <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < kThreads / 32; ++w) s += red[w];
    return s;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads) grad_squares_kernel(const __grid_constant__ Table<CAP> t, double* part) {
    __shared__ double red[kThreads / 32];
    double s = 0.0;
    for (int64_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        const int64_t i0 = (c - t.e[k].first) * kChunk, i1 = min(t.e[k].n, i0 + kChunk);
        for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads) {
            const double g = load_any(t.e[k].src, t.src_type[k], i);
            s += g * g;
        }
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double joined_norm(const double* part, int64_t parts, double* red) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < parts; i += kThreads) s += part[i];
    return sqrt(block_sum(s, red));
}

__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const double* part, int64_t parts, float* norm) {
    __shared__ double red[kThreads / 32];
    const double n = joined_norm(part, parts, red);
    if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

template <int CAP>
__global__ void __launch_bounds__(kThreads)
grad_scale_kernel(const __grid_constant__ Table<CAP> t, const double* part, int64_t parts, double max_norm, double eps, float* norm) {
    __shared__ double red[kThreads / 32];
    const double n = joined_norm(part, parts, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
    // (a NaN stays one; a norm of zero leaves the zeros as they are, also with max_norm and eps of zero)
    const double q = n == 0.0 ? 1.0 : max_norm / (n + eps);
    const float s = q >= 1.0 ? 1.0f : static_cast<float>(q);
    for (int64_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        if (s == 1.0f && t.e[k].dst == t.e[k].src) continue;
        const int64_t i0 = (c - t.e[k].first) * kChunk, i1 = min(t.e[k].n, i0 + kChunk);
        for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads)
            store_any(t.e[k].dst, t.dst_type[k], i, load_any(t.e[k].src, t.src_type[k], i) * s);
    }
}

// The next tensors of the list, as many as the table holds; their number.
template <int CAP>
int64_t fill(Table<CAP>& t, const GradTensor* g, int64_t tensors) {
    t.count = 0, t.chunks = 0;
    int64_t i = 0;
    for (; i < tensors && t.count < CAP; ++i) {
        if (g[i].n == 0) continue;
        t.e[t.count] = {g[i].src, g[i].dst, g[i].n, t.chunks};
        t.src_type[t.count] = static_cast<uint8_t>(g[i].src_type);
        t.dst_type[t.count] = static_cast<uint8_t>(g[i].dst_type);
        t.chunks += (g[i].n + kChunk - 1) / kChunk;
        ++t.count;
    }
    return i;
}
int grid_of(int64_t chunks) { return static_cast<int>(chunks < 1 ? 1 : (chunks < kPartBlocks ? chunks : kPartBlocks)); }

cudaError_t squares(const GradTensor* g, int64_t tensors, double* part, int64_t* parts, cudaStream_t s) {
    *parts = 0;
    static thread_local Table<kCap> t;
    while (tensors > 0) {
        const int64_t took = fill(t, g, tensors);
        g += took, tensors -= took;
        if (t.count == 0) continue;
        const int grid = grid_of(t.chunks);
        grad_squares_kernel<kCap><<<grid, kThreads, 0, s>>>(t, part + *parts);
        if (const cudaError_t e = cudaGetLastError()) return e;
        *parts += grid;
    }
    return cudaSuccess;
}

}  // namespace

int64_t grad_norm_partials(int64_t tensors) { return ((tensors + kCap - 1) / kCap + 1) * kPartBlocks; }

cudaError_t grad_norm_launch(const GradTensor* g, int64_t tensors, double* part, float* norm, cudaStream_t s) {
    int64_t parts = 0;
    if (const cudaError_t e = squares(g, tensors, part, &parts, s)) return e;
    grad_norm_kernel<<<1, kThreads, 0, s>>>(part, parts, norm);
    return cudaGetLastError();
}

cudaError_t grad_clip_launch(const GradTensor* g, int64_t tensors, double* part, double max_norm, double eps, float* norm,
                             cudaStream_t s) {
    int64_t parts = 0;
    if (const cudaError_t e = squares(g, tensors, part, &parts, s)) return e;
    static thread_local Table<kCap> t;
    bool told = false;
    while (tensors > 0 || !told) {
        const int64_t took = fill(t, g, tensors);
        g += took, tensors -= took;
        if (t.count == 0 && told) continue;
        grad_scale_kernel<kCap><<<grid_of(t.chunks), kThreads, 0, s>>>(t, part, parts, max_norm, eps, told ? nullptr : norm);
        if (const cudaError_t e = cudaGetLastError()) return e;
        told = true;
    }
    return cudaSuccess;
}

}  // namespace nfx
