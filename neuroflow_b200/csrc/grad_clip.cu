// grad_clip.cu -- the 2-norm over all elements of many tensors, and the tensors scaled down to a norm.
//
//   n = sqrt(sum g^2),  s = min(1, max_norm / (n + eps)),  out = g s
//
// The tensors' addresses and sizes are kernel parameters, so nothing is copied to the device and a call can be
// captured.  Squares are added in fp32 over the 32 (16 of fp32) elements that a thread has at a time and in 64
// bits from there; where such a sum leaves the range in which fp32 squares are exact enough, its elements are
// squared in 64 bits instead.  Each block leaves its share in the workspace, and whoever needs the norm adds the
// shares in a fixed order, so the result does not change from run to run.
//
// Bound by HBM: the elements are read twice, as more of them than L2 holds are seldom there the second time.  Measured (one
// B200, GPU time): 120M bf16 in 300 tensors, norm alone 42 us, 5.7 TB/s; into bf16 132 us, into unaligned fp32 166 us
// (4.4 TB/s of the bytes that one reading would take); 120M fp32 249 us; 6 tensors of 66,000 fp32 in one launch 5.0 us.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "dense_ops.h"
#include "launch.cuh"
#include "nfx_internal.h"
#include "rms_parts.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

constexpr int kThreads = 256;
constexpr int kGroupPacks = 4;                                // packs of 16 bytes that a thread has in flight
constexpr int kFewThreads = 512, kFewCluster = 8;
constexpr int kPartBlocks = 4 * 148;                          // shares that one launch leaves, at most
// Blocks of the scaling kernel at most: far more than are resident, so that one which ends early is followed by another
// (134M bf16 into fp32: 200 us with 4 * 148, 193 with 8, 187 with 16, 184 with 32, 188 with one for each chunk).  The
// kernel of the squares leaves a share for each block; there 4 are best (45 us; 53 with 16).
constexpr int kScaleBlocks = 32 * 148;

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
    int64_t chunks, chunk;
};
// Kernel parameters hold 32,764 bytes; a launch copies all of them (two launches with 900 entries take 6.5 us longer on
// the host than with 48), so short lists have tables of their own.
constexpr int kCap = 900, kCapMid = 240, kCapFew = 48;
static_assert(sizeof(Table<kCap>) + 64 <= 32764, "kernel parameters");

// The tensor that chunk c belongs to (tensors without elements have no entry).
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

template <int THREADS>
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) s += red[w];
    return s;
}

// The sum of squares of chunk elements [i0, i1) of a tensor, `i` counted from the last 16-byte boundary before its
// first element (`shift` elements in front of it); this thread's share.
template <typename T, int THREADS>
__device__ __forceinline__ double squares_of(const T* src, int64_t n, int shift, int64_t i0, int64_t i1, int tid) {
    constexpr int VE = 16 / sizeof(T);
    double sum = 0.0;
    for (int64_t b = i0 + tid * VE; b < i1; b += static_cast<int64_t>(THREADS) * VE * kGroupPacks) {
        Elems<T, VE> v[kGroupPacks];
#pragma unroll
        for (int k = 0; k < kGroupPacks; ++k) {
            const int64_t c = b + static_cast<int64_t>(k) * THREADS * VE - shift;  // the pack's first element
            if (c + shift < i1 && c >= 0 && c + VE <= n) {
                v[k].load(src + c);
            } else {
                v[k].zero();
                if (c + shift < i1) {
                    // (an edge of the tensor: the pack's elements that it has)
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        if (c + i < 0 || c + i >= n) continue;
                        if constexpr (sizeof(T) == 4) v[k].w[i] = __ldg(reinterpret_cast<const uint32_t*>(src) + c + i);
                        else v[k].w[i / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(src) + c + i)) << (16 * (i & 1));
                    }
                }
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < kGroupPacks; ++k)
#pragma unroll
            for (int i = 0; i < VE; ++i) s = fmaf(v[k].at(i), v[k].at(i), s);
        if (s > 0x1p-80f && s < 0x1p100f) {
            sum += static_cast<double>(s);
        } else {
            uint32_t any = 0;
#pragma unroll
            for (int k = 0; k < kGroupPacks; ++k)
#pragma unroll
                for (int i = 0; i < Elems<T, VE>::kWords; ++i) any |= v[k].w[i] & (sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu);
            if (any) {
#pragma unroll
                for (int k = 0; k < kGroupPacks; ++k)
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        const double g = static_cast<double>(v[k].at(i));
                        sum = fma(g, g, sum);
                    }
            }
        }
    }
    return sum;
}

// Elements of a chunk, counted from a 16-byte boundary.  Finding a chunk's tensor takes a few hundred cycles, so chunks
// are large where there are enough of them (120M bf16 into bf16: 121 us with 16,384, 126 with 8,192, 123 with 32,768;
// 605,000 fp32: 7.7, 5.7, 11.3).  A warp of the cluster's kernel takes as much as it can have in flight.
constexpr int64_t kChunk = 16384, kChunkSmall = 8192, kChunkWarp = 1024;
__host__ __device__ __forceinline__ int shift_el(const void* p, int type) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / (type == kF32 ? 4 : 2));
}

template <int CAP, int THREADS>
__device__ __forceinline__ double chunk_squares(const Table<CAP>& t, int64_t c, int tid) {
    const int k = tensor_of(t, c);
    const int64_t n = t.e[k].n;
    const int type = t.src_type[k], shift = shift_el(t.e[k].src, type);
    const int64_t i0 = (c - t.e[k].first) * t.chunk, i1 = min(n + shift, i0 + t.chunk);
    if (type == kF32) return squares_of<float, THREADS>(static_cast<const float*>(t.e[k].src), n, shift, i0, i1, tid);
    if (type == kBF16) return squares_of<__nv_bfloat16, THREADS>(static_cast<const __nv_bfloat16*>(t.e[k].src), n, shift, i0, i1, tid);
    return squares_of<__half, THREADS>(static_cast<const __half*>(t.e[k].src), n, shift, i0, i1, tid);
}

// N elements that lie `q` elements behind a boundary: the words that hold them, and how they are moved into place.
// Boundaries are of 16 bytes, or of what N elements take where that is less.  MOVED: q > 0.
template <typename T, int N, bool MOVED>
struct Moved {
    static constexpr int kUnit = N * static_cast<int>(sizeof(T)) < 16 ? N * static_cast<int>(sizeof(T)) : 16;  // bytes
    static constexpr int kUnits = N * static_cast<int>(sizeof(T)) / kUnit + (MOVED ? 1 : 0);
    static constexpr int kWords = kUnits * kUnit / 4;
    static constexpr int kSpan = kUnits * kUnit / static_cast<int>(sizeof(T));  // elements that are read
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* boundary) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            if constexpr (kUnit == 16) {
                const uint4 u = __ldcs(reinterpret_cast<const uint4*>(boundary) + i);
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            } else {
                const uint2 u = __ldcs(reinterpret_cast<const uint2*>(boundary) + i);
                w[2 * i] = u.x, w[2 * i + 1] = u.y;
            }
        }
    }
    __device__ __forceinline__ void get(int q, float (&o)[N]) {
        if constexpr (MOVED) {
            const int words = sizeof(T) == 4 ? q : q >> 1;
            if (words & 2) {
#pragma unroll
                for (int i = 0; i + 2 < kWords; ++i) w[i] = w[i + 2];
            }
            if (words & 1) {
#pragma unroll
                for (int i = 0; i + 1 < kWords; ++i) w[i] = w[i + 1];
            }
            if (sizeof(T) == 2 && (q & 1)) {
#pragma unroll
                for (int i = 0; i < N / 2; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
            }
        }
        Elems<T, N> e;
#pragma unroll
        for (int i = 0; i < Elems<T, N>::kWords; ++i) e.w[i] = w[i];
        e.get(o);
    }
};

// out = src s for packs of 16 bytes of `dst`, elements [i0, i1) counted from the last 16-byte boundary before its
// first element.
template <typename T, typename D, int THREADS, bool MOVED>
__device__ __forceinline__ void scale_packs(const T* src, D* dst, int64_t n, int shift, int q, int64_t i0, int64_t i1, float s, int tid) {
    constexpr int N = 16 / sizeof(D), kSpan = Moved<T, N, MOVED>::kSpan, kStep = THREADS * N;
    const auto put = [&](int64_t c, Moved<T, N, MOVED>& m) {
        float v[N];
        m.get(q, v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= s;
        Elems<D, N> o;
        o.set(v);
        __stcs(reinterpret_cast<uint4*>(dst + c), make_uint4(o.w[0], o.w[1], o.w[2], o.w[3]));
    };
    for (int64_t b = i0 + tid * N; b < i1; b += kStep * kGroupPacks) {
        const int64_t c = b - shift;
        Moved<T, N, MOVED> m[kGroupPacks];
        // the words of all packs lie inside the tensor
        if (c - q >= 0 && b + (kGroupPacks - 1) * kStep < i1 && c - q + (kGroupPacks - 1) * kStep + kSpan <= n) {
#pragma unroll
            for (int k = 0; k < kGroupPacks; ++k) m[k].load(src + c + k * kStep - q);
#pragma unroll
            for (int k = 0; k < kGroupPacks; ++k) put(c + k * kStep, m[k]);
            continue;
        }
        for (int k = 0; k < kGroupPacks && b + k * kStep < i1; ++k) {
            const int64_t at = c + k * kStep;
            if (at - q >= 0 && at - q + kSpan <= n) {
                m[0].load(src + at - q);
                put(at, m[0]);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (at + i >= 0 && at + i < n) dst[at + i] = from_f32<D>(to_f32(src[at + i]) * s);
            }
        }
    }
}
template <typename T, typename D, int THREADS>
__device__ __forceinline__ void scale_chunk(const T* src, D* dst, int64_t n, int shift, int64_t i0, int64_t i1, float s, int tid) {
    constexpr int kUnit = Moved<T, 16 / sizeof(D), false>::kUnit;
    const int q = static_cast<int>((reinterpret_cast<uintptr_t>(src) - shift * sizeof(T)) % kUnit / sizeof(T));
    if (q == 0) scale_packs<T, D, THREADS, false>(src, dst, n, shift, q, i0, i1, s, tid);
    else scale_packs<T, D, THREADS, true>(src, dst, n, shift, q, i0, i1, s, tid);
}

template <int CAP, int THREADS>
__device__ __forceinline__ void chunk_scale(const Table<CAP>& t, int64_t c, float s, int tid) {
    const int k = tensor_of(t, c);
    const Entry& e = t.e[k];
    if (s == 1.0f && e.dst == e.src) return;  // every element times one
    // chunks are counted by the source's boundaries, packs by the destination's: a chunk's packs are those that
    // begin in it
    const int64_t n = e.n, at = (c - e.first) * t.chunk - shift_el(e.src, t.src_type[k]), end = at + t.chunk;
    const int dt = t.dst_type[k], st = t.src_type[k];
    const int shift = shift_el(e.dst, dt), pack = dt == kF32 ? 4 : 8;
    const auto pack_from = [&](int64_t i) { return i <= -shift ? static_cast<int64_t>(0) : (i + shift + pack - 1) / pack * pack; };
    const int64_t i0 = at <= 0 ? 0 : pack_from(at), i1 = end >= n ? n + shift : pack_from(end);
    const auto go = [&](auto* src) {
        if (dt == kF32) scale_chunk<std::remove_const_t<std::remove_pointer_t<decltype(src)>>, float, THREADS>(src, static_cast<float*>(e.dst), n, shift, i0, i1, s, tid);
        else if (dt == kBF16) scale_chunk<std::remove_const_t<std::remove_pointer_t<decltype(src)>>, __nv_bfloat16, THREADS>(src, static_cast<__nv_bfloat16*>(e.dst), n, shift, i0, i1, s, tid);
        else scale_chunk<std::remove_const_t<std::remove_pointer_t<decltype(src)>>, __half, THREADS>(src, static_cast<__half*>(e.dst), n, shift, i0, i1, s, tid);
    };
    if (st == kF32) go(static_cast<const float*>(e.src));
    else if (st == kBF16) go(static_cast<const __nv_bfloat16*>(e.src));
    else go(static_cast<const __half*>(e.src));
}

// (a NaN stays one; a norm of zero leaves the zeros as they are, also with max_norm and eps of zero, and a max_norm of
// infinity leaves everything, also with an infinite norm)
__device__ __forceinline__ float scale_for(double n, double max_norm, double eps) {
    const double q = n == 0.0 || (isinf(max_norm) && !isnan(n)) ? 1.0 : max_norm / (n + eps);
    return q >= 1.0 ? 1.0f : static_cast<float>(q);
}

template <int CAP>
__global__ void __launch_bounds__(kThreads) grad_squares_kernel(const __grid_constant__ Table<CAP> t, double* part) {
    __shared__ double red[kThreads / 32];
    grid_dep_wait();
    double s = 0.0;
    for (int64_t c = blockIdx.x; c < t.chunks; c += gridDim.x) s += chunk_squares<CAP, kThreads>(t, c, threadIdx.x);
    grid_dep_launch();  // the kernel that needs the norm may be placed
    s = block_sum<kThreads>(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double joined_norm(const double* part, int64_t parts, double* red) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < parts; i += kThreads) s += part[i];
    return sqrt(block_sum<kThreads>(s, red));
}

__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const double* part, int64_t parts, float* norm) {
    __shared__ double red[kThreads / 32];
    grid_dep_wait();
    const double n = joined_norm(part, parts, red);
    if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

// The chunks in the other order than the squares were summed in: what was read last is still in L2.
template <int CAP>
__global__ void __launch_bounds__(kThreads)
grad_scale_kernel(const __grid_constant__ Table<CAP> t, const double* part, int64_t parts, double max_norm, double eps, float* norm) {
    __shared__ double red[kThreads / 32];
    grid_dep_wait();
    grid_dep_launch();
    const double n = joined_norm(part, parts, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
    const float s = scale_for(n, max_norm, eps);
    for (int64_t c = t.chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) chunk_scale<CAP, kThreads>(t, c, s, threadIdx.x);
}

// A few tensors of few elements: one cluster sums, joins through its shared memory and scales, in one launch; a chunk
// is a warp's.
template <bool SCALE>
__global__ void __launch_bounds__(kFewThreads)
grad_few_kernel(const __grid_constant__ Table<kCapFew> t, double max_norm, double eps, float* norm) {
    __shared__ double red[kFewThreads / 32];
    __shared__ double mine;
    const uint32_t rank = cluster_ctarank();
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, first = static_cast<int>(rank) + kFewCluster * static_cast<int>(threadIdx.x >> 5);
    constexpr int kStep = kFewCluster * kFewThreads / 32;
    double s = 0.0;
    for (int64_t c = first; c < t.chunks; c += kStep) s += chunk_squares<kCapFew, 32>(t, c, lane);
    s = block_sum<kFewThreads>(s, red);
    if (threadIdx.x == 0) mine = s;
    cluster_sync();
    double n = 0.0;
    for (int r = 0; r < kFewCluster; ++r) {
        double v;
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(map_rank(smem_u32(&mine), r)) : "memory");
        n += v;
    }
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    n = sqrt(n);
    if (rank == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
    if constexpr (SCALE) {
        const float f = scale_for(n, max_norm, eps);
        for (int64_t c = first; c < t.chunks; c += kStep) chunk_scale<kCapFew, 32>(t, c, f, lane);
        __syncwarp();
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // no CTA leaves while another may still read its share
}

// The next tensors of the list, as many as the table holds; their number.
template <int CAP>
int64_t fill(Table<CAP>& t, const GradTensor* g, int64_t tensors, int64_t chunk) {
    t.count = 0, t.chunks = 0, t.chunk = chunk;
    int64_t i = 0;
    for (; i < tensors && t.count < CAP; ++i) {
        if (g[i].n == 0) continue;
        t.e[t.count] = {g[i].src, g[i].dst, g[i].n, t.chunks};
        t.src_type[t.count] = static_cast<uint8_t>(g[i].src_type);
        t.dst_type[t.count] = static_cast<uint8_t>(g[i].dst_type);
        t.chunks += (g[i].n + shift_el(g[i].src, g[i].src_type) + chunk - 1) / chunk;
        ++t.count;
    }
    return i;
}
int64_t chunk_for(const GradTensor* g, int64_t tensors) {
    int64_t n = 0;
    for (int64_t i = 0; i < tensors; ++i) n += g[i].n;
    return n < 4 * kPartBlocks * kChunk ? kChunkSmall : kChunk;
}
int grid_of(int64_t chunks, int64_t most) { return static_cast<int>(chunks < 1 ? 1 : (chunks < most ? chunks : most)); }

template <int CAP>
cudaError_t squares(Table<CAP>& t, const GradTensor* g, int64_t tensors, double* part, int64_t* parts, cudaStream_t s) {
    *parts = 0;
    const int64_t chunk = chunk_for(g, tensors);
    while (tensors > 0) {
        const int64_t took = fill(t, g, tensors, chunk);
        g += took, tensors -= took;
        if (t.count == 0) continue;
        const int grid = grid_of(t.chunks, std::min<int64_t>(4 * device_sm_count(), kPartBlocks));
        if (const cudaError_t e = launch_early(grad_squares_kernel<CAP>, grid, kThreads, 0, 1, s, t, part + *parts)) return e;
        *parts += grid;
    }
    return cudaSuccess;
}

template <int CAP>
cudaError_t clip(const GradTensor* g, int64_t tensors, double* part, double max_norm, double eps, float* norm, cudaStream_t s) {
    static thread_local Table<CAP> t;
    int64_t parts = 0;
    if (const cudaError_t e = squares(t, g, tensors, part, &parts, s)) return e;
    const int64_t chunk = chunk_for(g, tensors);
    const bool whole = tensors <= CAP;  // the table holds all of them, as it was filled
    bool told = false;
    while (tensors > 0 || !told) {
        const int64_t took = whole ? tensors : fill(t, g, tensors, chunk);
        g += took, tensors -= took;
        if (t.count == 0 && told) continue;
        if (const cudaError_t e = launch_early(grad_scale_kernel<CAP>, grid_of(t.chunks, kScaleBlocks), kThreads, 0, 1, s, t, part, parts, max_norm, eps,
                                               told ? static_cast<float*>(nullptr) : norm))
            return e;
        told = true;
    }
    return cudaSuccess;
}

// One launch of a cluster: 5.4 us for 65,000 fp32 numbers, 9.4 for 245,000, where two launches over all SMs take 5.7
// for 605,000 (and a launch more on the host).
constexpr int64_t kFewBytes = 384 << 10;
bool few(const GradTensor* g, int64_t tensors) {
    if (tensors > kCapFew) return false;
    int64_t bytes = 0;
    for (int64_t i = 0; i < tensors; ++i) {
        if (g[i].n > kFewBytes) return false;
        bytes += g[i].n * type_bytes(g[i].src_type);
    }
    return bytes <= kFewBytes;
}

}  // namespace

int64_t grad_norm_partials(int64_t tensors) { return ((tensors + kCap - 1) / kCap + 1) * kPartBlocks; }

cudaError_t grad_norm_launch(const GradTensor* g, int64_t tensors, double* part, float* norm, cudaStream_t s) {
    if (few(g, tensors)) {
        static thread_local Table<kCapFew> t;
        fill(t, g, tensors, kChunkWarp);
        return launch_early(grad_few_kernel<false>, kFewCluster, kFewThreads, 0, kFewCluster, s, t, 0.0, 0.0, norm);
    }
    int64_t parts = 0;
    cudaError_t e;
    if (tensors <= kCapFew) {
        static thread_local Table<kCapFew> t;
        e = squares(t, g, tensors, part, &parts, s);
    } else if (tensors <= kCapMid) {
        static thread_local Table<kCapMid> t;
        e = squares(t, g, tensors, part, &parts, s);
    } else {
        static thread_local Table<kCap> t;
        e = squares(t, g, tensors, part, &parts, s);
    }
    if (e != cudaSuccess) return e;
    return launch_early(grad_norm_kernel, 1, kThreads, 0, 1, s, part, parts, norm);
}

cudaError_t grad_clip_launch(const GradTensor* g, int64_t tensors, double* part, double max_norm, double eps, float* norm,
                             cudaStream_t s) {
    if (few(g, tensors)) {
        static thread_local Table<kCapFew> t;
        fill(t, g, tensors, kChunkWarp);
        return launch_early(grad_few_kernel<true>, kFewCluster, kFewThreads, 0, kFewCluster, s, t, max_norm, eps, norm);
    }
    if (tensors <= kCapFew) return clip<kCapFew>(g, tensors, part, max_norm, eps, norm, s);
    if (tensors <= kCapMid) return clip<kCapMid>(g, tensors, part, max_norm, eps, norm, s);
    return clip<kCap>(g, tensors, part, max_norm, eps, norm, s);
}

}  // namespace nfx
