// layer_norm.cu -- layer norm over the last dimension of (rows, d), forward (into the
// input's type, or straight into FP8 groups of 128) and backward.
//
//   mu = sum x / d,  v = sum (x - mu)^2 / d,  r = 1 / sqrt(v + eps),  xh = (x - mu) r
//   y  = gamma xh + beta
//   a  = gamma dy,  dx = r (a - mean(a) - xh mean(a xh))
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// All statistics and sums are fp32; the variance is the mean of the centred squares (a
// second sweep), not E[x^2] - mu^2, which cancels when |mu| is large against the spread.
// The rounding error of mu is taken out of the centred values: for fp32 rows that sweep sums them too
// and their mean is the error, for 16-bit rows it is the division's remainder (sums_centred).  It
// leaves y within two or three roundings of the formula, which decides how many FP8 codes fall on the
// other side of a rounding boundary.  Outputs are rounded once.
#include <atomic>

#include "block_ops.h"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "row_pack.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

constexpr int kAnyThreads = 256;

// v, or zero where it is negative; a NaN stays one.
__device__ __forceinline__ float not_negative(float v) { return v < 0.0f ? 0.0f : v; }

// s / d with d's reciprocal at hand: the product, and one correction by the exact remainder (Markstein's
// step), which gives back a constant row's value exactly where the sum s is exact.
__device__ __forceinline__ float mean_of(float s, float fd, float inv_d) {
    const float q = s * inv_d;
    return fmaf(fmaf(-q, fd, s), inv_d, q);
}

// Sums of (a, b) over the block, the same bits in every thread.  `red` holds one pair per warp.
__device__ __forceinline__ float2 block_sums(float a, float b, float2* red) {
    a = warp_sum(a), b = warp_sum(b);
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 t = make_float2(0.0f, 0.0f);
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t.x += red[w].x, t.y += red[w].y;
    return t;
}

// Wider than the row kernels below hold: one block per row, the row read three times (from L2
// after the first).
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) norm_any_kernel(NormArgs a) {
    __shared__ float2 red[kAnyThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float fd = static_cast<float>(a.d);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        float s = 0.0f;
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) s += to_f32(x[i]);
        const float mu0 = __fdiv_rn(block_sums(s, 0.0f, red).x, fd);
        float s1 = 0.0f;
        s = 0.0f;
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            const float c = to_f32(x[i]) - mu0;
            s1 += c;
            s = fmaf(c, c, s);
        }
        const float2 t = block_sums(s1, s, red);
        const float rest = __fdiv_rn(t.x, fd);
        const float rs = __frsqrt_rn(not_negative(fmaf(-rest, rest, __fdiv_rn(t.y, fd))) + a.eps), off = -rest * rs;
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mu0 + rest;
            if (a.rstd) a.rstd[r] = rs;
        }
        auto out = [&](int i) {
            const float xh = fmaf(to_f32(x[i]) - mu0, rs, off);
            const float g = a.gamma ? load_any(a.gamma, a.ptype, i) : 1.0f;
            return fmaf(xh, g, a.beta ? load_any(a.beta, a.ptype, i) : 0.0f);
        };
        if (a.y) {
            T* y = static_cast<T*>(a.y) + r * a.ldy;
            for (int i = threadIdx.x; i < a.d; i += kAnyThreads) y[i] = from_f32<T>(out(i));
        } else {
            const int blocks = (a.d + kGroup - 1) / kGroup;
            for (int b = warp; b < blocks; b += kAnyThreads / 32) {
                float v[kGroup / 32], am = 0.0f;
#pragma unroll
                for (int j = 0; j < kGroup / 32; ++j) {
                    const int i = b * kGroup + j * 32 + lane;
                    v[j] = i < a.d ? out(i) : 0.0f;
                    am = fmaxf(am, finite_abs(v[j]));
                }
                const float sc = group_scale(warp_max(am)), inv = __frcp_rn(sc);
#pragma unroll
                for (int j = 0; j < kGroup / 32; ++j) {
                    const int i = b * kGroup + j * 32 + lane;
                    if (i < a.d) a.q.codes[r * a.q.ld + i] = static_cast<uint8_t>(e4m3_code(v[j], inv));
                }
                if (lane == 0) a.q.scales[r * a.q.srs + b * a.q.sbs] = sc;
            }
        }
    }
}

// Any width: a block takes every gridDim.x-th row and adds its rows' parameter gradients,
// in their order, to its own two rows of partial sums (each column always by one thread).
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) norm_grad_any_kernel(NormGradArgs a) {
    __shared__ float2 red[kAnyThreads / 32];
    const float fd = static_cast<float>(a.d);
    float* pg = a.part + static_cast<int64_t>(blockIdx.x) * a.d;
    float* pb = a.part + (static_cast<int64_t>(a.parts) + blockIdx.x) * a.d;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
        T* dx = static_cast<T*>(a.dx) + r * a.lddx;
        const float mu = a.mean[r], rs = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            const float xh = (to_f32(x[i]) - mu) * rs, g = to_f32(dy[i]);
            const float ga = a.gamma ? g * load_any(a.gamma, a.ptype, i) : g;
            s1 += ga;
            s2 = fmaf(ga, xh, s2);
            if (a.part) {
                const bool first = r == blockIdx.x;
                pg[i] = fmaf(g, xh, first ? 0.0f : pg[i]);
                pb[i] = g + (first ? 0.0f : pb[i]);
            }
        }
        const float2 t = block_sums(s1, s2, red);
        s1 = __fdiv_rn(t.x, fd), s2 = __fdiv_rn(t.y, fd);
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            const float xh = (to_f32(x[i]) - mu) * rs, g = to_f32(dy[i]);
            const float ga = a.gamma ? g * load_any(a.gamma, a.ptype, i) : g;
            dx[i] = from_f32<T>(rs * (ga - s1 - xh * s2));
        }
    }
}

// COLS columns per block, 1024 / COLS threads per column over the partial sums with four (8 columns) or
// eight loads in flight, joined in a fixed order.  Block row y handles the y-th set of partial sums and its
// output.  Launched with programmatic serialization: it waits for the kernel before it by itself.  Eight
// columns, a 32-byte sector of a row, spread few columns over more SMs (5003x771 backward 18.2 -> 17.2 us);
// from 2,048 columns on there are SMs enough for 32 (512x4096: 10.8 us, 16.8 with 8).
template <int COLS>
__global__ void __launch_bounds__(1024) column_reduce_kernel(const float* part, int parts, int64_t n, void* out0, void* out1,
                                                             int otype) {
    constexpr int kT = 1024 / COLS, kU = COLS == 8 ? 4 : 8;
    __shared__ float red[COLS][kT + 1];
    const int c = threadIdx.x % COLS, t = threadIdx.x / COLS;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * COLS + c;
    void* out = blockIdx.y ? out1 : out0;
    if (!out) return;
    grid_dep_wait();
    part += static_cast<int64_t>(blockIdx.y) * parts * n;
    float s = 0.0f;
    if (i < n) {
        for (int p = t; p < parts; p += kT * kU) {
            float v[kU];
#pragma unroll
            for (int k = 0; k < kU; ++k) v[k] = p + kT * k < parts ? part[static_cast<int64_t>(p + kT * k) * n + i] : 0.0f;
#pragma unroll
            for (int k = 0; k < kU; ++k) s += v[k];
        }
    }
    red[c][t] = s;
    __syncthreads();
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;  // the warp's column is w
    if (w >= COLS) return;
    s = red[w][lane];
#pragma unroll
    for (int k = 32; k < kT; k += 32) s += red[w][lane + k];
    s = warp_sum(s);
    if (lane == 0 && static_cast<int64_t>(blockIdx.x) * COLS + w < n)
        store_any(out, otype, static_cast<int64_t>(blockIdx.x) * COLS + w, s);
}

// ---------------------------------------------------------------------------
// The row in registers: read once, both statistics and the output from it.  TPR threads per row, each
// holding VPT packs of VE elements (16 bytes, or one element where rows are not 16-byte aligned).  A
// warp's packs are contiguous -- pack j of lane l of warp w is (w * VPT + j) * 32 + l of the row -- so
// the 128 elements of an FP8 group lie in one warp: half a warp's pack (16-bit types), one pack (fp32)
// or four (VE = 1), and its maximum is a few shuffles.
// ---------------------------------------------------------------------------
// VE parameters (of x's type or fp32) from element i; `vec` when they are 16-byte aligned.
template <typename T, int VE>
__device__ __forceinline__ void load_params(const void* p, int type, bool vec, int i, float none, float (&o)[VE]) {
    if (!p) {
#pragma unroll
        for (int k = 0; k < VE; ++k) o[k] = none;
    } else if (VE > 2 && vec && type == kF32) {
#pragma unroll
        for (int k = 0; k < VE; k += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + k));
            o[k] = f.x, o[k + 1] = f.y, o[k + 2] = f.z, o[k + 3] = f.w;
        }
    } else if (VE == 8 && vec) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < VE; k += 2) {
            float2 f;
            if (type == kBF16) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k / 2]));
            else f = __half22float2(*reinterpret_cast<const __half2*>(&w[k / 2]));
            o[k] = f.x, o[k + 1] = f.y;
        }
    } else if (type == kF32) {
#pragma unroll
        for (int k = 0; k < VE; ++k) o[k] = __ldg(static_cast<const float*>(p) + i + k);
    } else {
#pragma unroll
        for (int k = 0; k < VE; ++k) o[k] = load_any(p, type, i + k);
    }
}

// Sums of (a, b) over the TPR threads of a row, the same bits in each of them; of a alone without TWO.
template <int TPR, bool TWO>
__device__ __forceinline__ float2 row_sums(float a, float b, float2* red) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
        if (TWO) b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    float2 t = make_float2(a, b);
    if constexpr (TPR > 32) {
        const int w = threadIdx.x >> 5, w0 = w / (TPR / 32) * (TPR / 32);  // the row's first warp
        if ((threadIdx.x & 31) == 0) red[w] = t;
        __syncthreads();
        t = red[w0];
#pragma unroll
        for (int k = 1; k < TPR / 32; ++k) {
            const float2 u = red[w0 + k];
            t.x += u.x;
            if (TWO) t.y += u.y;
        }
    }
    return t;
}

// A pack as it was read.
template <typename T, int VE>
struct Raw {
    word_t<T, VE> u;
    __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const word_t<T, VE>*>(p)); }
    __device__ __forceinline__ void get(float (&o)[VE]) const { unpack<T, VE>(u, o); }
    __device__ __forceinline__ void zero() { u = word_t<T, VE>{}; }
};

constexpr int row_block(int tpr) { return tpr > 128 ? tpr : 128; }
// With at most 16 elements a thread, resident blocks walk over the rows: the parameters stay in registers
// (read again for every row, fp32 parameters are twice the bytes of a bf16 row from L1: without any
// parameters 8191x2048 took 10.4 us against 15.9) and the next row is fetched ahead.  8191x2048 bf16 15.9
// -> 13.2 us, 65536x512 31.9 -> 26.5, 131072x128 fp32 30.6 -> 26.9.  Wider rows keep 32 elements a thread and a
// block each (4096x8192 bf16: 34 us, 39 walking).
constexpr bool walks(int n) { return n <= 16; }
// Blocks per SM that the registers are cut for: 768 threads walking (16384x4096 bf16 56 -> 50 us against no
// bound; 1,024 threads spill, 58 us), 1,024 with wide rows (4096x16001 bf16 162 us, 236 with 512).
constexpr int row_blocks(int vpt, int ve, int tpr) {
    return walks(vpt * ve) ? (row_block(tpr) > 384 ? 1 : 768 / row_block(tpr)) : (tpr >= 512 ? 2 : 1);
}

// Whether the centred values are summed to find the rounding error of the mean (rows of at most `width`).
// fp32 numbers need it (a constant row of 20,001 times 1000.1 is 0.2 off without).  16-bit ones do not: sums
// are exact where the numbers are of one size (8 or 11 bits and log2(width) more), and where they are not
// the spread is as large as the numbers.  There the second sum would only add its own rounding, which is
// the same way for all numbers of a binade, as they have the same low bits once mu0 is taken off
// (4096 columns: the mean 1.7e-8 off, and 23 FP8 codes of 12 million on the other side of a boundary against
// 10 for the formula in plain fp32; 9 without it).
template <typename T>
constexpr bool sums_centred(int width) {
    return sizeof(T) == 4 || (std::is_same<T, __half>::value && width > 8192);
}

template <typename T, int VE, int VPT, int TPR, bool FP8>
__global__ void __launch_bounds__(row_block(TPR), row_blocks(VPT, VE, TPR)) norm_row_kernel(NormArgs a, bool pvec, bool wide) {
    __shared__ float2 red[2][row_block(TPR) / 32];
    constexpr int kRows = row_block(TPR) / TPR, N = VPT * VE;
    constexpr bool kWalk = walks(N);
    constexpr bool kCentred = sums_centred<T>(N * TPR);
    const int lane = threadIdx.x & 31, sub = threadIdx.x % TPR;
    // pack j of this thread is first + j * 32 (a row of fewer than 32 threads has one pack a thread)
    const int first = TPR < 32 ? sub : (sub >> 5) * VPT * 32 + lane;
    const float fd = static_cast<float>(a.d), inv_d = __frcp_rn(fd);
    // (the warps whose packs all lie inside the row need no test per pack)
    const bool full = TPR >= 32 && (first - lane + VPT * 32) * VE <= a.d;
    Raw<T, VE> rx[VPT];
    auto fetch = [&](int64_t r) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx + first * VE;
        if (full && r < a.rows) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) rx[j].load(x + j * 32 * VE);
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                if (r < a.rows && (first + j * 32) * VE < a.d) rx[j].load(x + j * 32 * VE);
                else rx[j].zero();
            }
        }
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    fetch(static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR);
    // walking, a thread's columns are the same in every row: their parameters stay in registers
    constexpr int kHeld = kWalk ? VPT : 1;
    float gam[kHeld][VE], bet[kHeld][VE];
    if constexpr (kWalk) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = (first + j * 32) * VE;
#pragma unroll
            for (int i = 0; i < VE; ++i) gam[j][i] = bet[j][i] = 0.0f;
            if (full || c < a.d) {
                load_params<T, VE>(a.gamma, a.ptype, pvec, c, 1.0f, gam[j]);
                load_params<T, VE>(a.beta, a.ptype, pvec, c, 0.0f, bet[j]);
            }
        }
    }
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += step) {
        const int64_t r = base + threadIdx.x / TPR;
        const bool live = r < a.rows;
        float v[VPT][VE], s;
        float* f = &v[0][0];  // the same numbers as one array (indices are constants after unrolling)
#pragma unroll
        for (int j = 0; j < VPT; ++j) rx[j].get(v[j]);
        if constexpr (kWalk) fetch(r + step);  // the next row comes while this one is worked on
        // two elements to an instruction (f32x2): with 16-bit rows, instructions and not bytes are the bound
        float2 p2 = make_float2(f[0], f[1]);
#pragma unroll
        for (int k = 2; k < N; k += 2) p2 = add2_rn(p2, make_float2(f[k], f[k + 1]));
        s = p2.x + p2.y;
        const float sum = row_sums<TPR, false>(s, 0.0f, red[0]).x, mu0 = mean_of(sum, fd, inv_d);
        float s1 = 0.0f;
        s = 0.0f;
        if (full) {
            const float2 m2 = make_float2(-mu0, -mu0);
            float2 q1 = make_float2(0.0f, 0.0f), q2 = q1;
#pragma unroll
            for (int k = 0; k < N; k += 2) {
                const float2 c = add2_rn(make_float2(f[k], f[k + 1]), m2);
                f[k] = c.x, f[k + 1] = c.y;
                if (kCentred) q1 = add2_rn(q1, c);
                q2 = fma2_rn(c, c, q2);
            }
            s1 = q1.x + q1.y;
            s = q2.x + q2.y;
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                if ((first + j * 32) * VE < a.d) {
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        v[j][i] -= mu0;
                        if (kCentred) s1 += v[j][i];
                        s = fmaf(v[j][i], v[j][i], s);
                    }
                }
            }
        }
        // what the rounding of mu0 left over: of its sum too (the centred values' own mean), or of the division
        const float2 t = row_sums<TPR, kCentred>(kCentred ? s1 : s, s, red[1]);
        const float rest = (kCentred ? t.x : fmaf(-mu0, fd, sum)) * inv_d, mu = mu0 + rest;
        // (a constant row of rounded sums can leave this difference below zero)
        const float rs = __frsqrt_rn(not_negative(fmaf(-rest, rest, (kCentred ? t.y : t.x) * inv_d)) + a.eps), off = -rest * rs;
        if (live && sub == 0) {
            if (a.mean) a.mean[r] = mu;
            if (a.rstd) a.rstd[r] = rs;
        }
        auto finish = [&](int j) {
            const int c = (first + j * 32) * VE;
            float g[VE], b[VE];
            if constexpr (kWalk) {
#pragma unroll
                for (int i = 0; i < VE; ++i) g[i] = gam[j][i], b[i] = bet[j][i];
            } else {
                load_params<T, VE>(a.gamma, a.ptype, pvec, c, 1.0f, g);
                load_params<T, VE>(a.beta, a.ptype, pvec, c, 0.0f, b);
            }
            if constexpr (VE == 1) {
                v[j][0] = fmaf(fmaf(v[j][0], rs, off), g[0], b[0]);
            } else {
#pragma unroll
                for (int i = 0; i < VE; i += 2) {
                    const float2 xh = fma2_rn(make_float2(v[j][i], v[j][i + 1]), make_float2(rs, rs), make_float2(off, off));
                    const float2 y = fma2_rn(xh, make_float2(g[i], g[i + 1]), make_float2(b[i], b[i + 1]));
                    v[j][i] = y.x, v[j][i + 1] = y.y;
                }
            }
            if constexpr (!FP8) {
                if (live) store_pack<T, VE>(static_cast<T*>(a.y) + r * a.ldy + c, v[j]);
            }
        };
        if (full) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) finish(j);
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j)
                if ((first + j * 32) * VE < a.d) finish(j);
        }
        if constexpr (FP8) store_codes<VE, VPT, TPR>(v, a.q, r, a.d, live, first, lane, wide);
        if constexpr (!kWalk) break;
    }
}

template <typename T, int VE, int VPT, int TPR, bool FP8>
cudaError_t norm_row_go(const NormArgs& a, bool pvec, bool wide, cudaStream_t s) {
    constexpr int kThreads = row_block(TPR), kRows = kThreads / TPR;
    auto kern = norm_row_kernel<T, VE, VPT, TPR, FP8>;
    const int64_t want = (a.rows + kRows - 1) / kRows;
    int64_t grid = want;
    if constexpr (walks(VPT * VE)) {
        static std::atomic<int> known[64];  // asked for once per kernel and device
        const int d = current_device() & 63;
        int most = known[d].load(std::memory_order_relaxed);
        if (most == 0) {
            if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&most, kern, kThreads, 0) != cudaSuccess || most < 1) most = 1;
            most *= device_sm_count();
            known[d].store(most, std::memory_order_relaxed);
        }
        grid = want < most ? want : most;
    }
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
    kern<<<static_cast<unsigned>(grid), kThreads, 0, s>>>(a, pvec, wide);
    return cudaGetLastError();
}

template <typename T, int VE, int VPT, int TPR>
cudaError_t norm_row(const NormArgs& a, bool pvec, cudaStream_t s) {
    if (a.y) return norm_row_go<T, VE, VPT, TPR, false>(a, pvec, false, s);
    const bool wide = reinterpret_cast<uintptr_t>(a.q.codes) % 8 == 0 && (a.rows == 1 || a.q.ld % 8 == 0);
    return norm_row_go<T, VE, VPT, TPR, true>(a, pvec, wide, s);
}

// Threads and packs per row by the width: 16 elements a thread up to 4,096 columns and 32 above; with packs
// of one or two elements 8 up to 4,096 columns (more loads to a row than a warp should queue:
// 5003x771 fp32 took 19 us with 32).
template <typename T, int VE>
cudaError_t norm_width(const NormArgs& a, bool pvec, cudaStream_t s) {
    if constexpr (VE > 2) {
        constexpr int kV = 32 / VE;  // packs of 32 elements
        if (a.d <= 16 * VE) return norm_row<T, VE, 1, 16>(a, pvec, s);
        if (a.d <= 32 * VE) return norm_row<T, VE, 1, 32>(a, pvec, s);
        if (a.d <= 64 * VE) return norm_row<T, VE, 2, 32>(a, pvec, s);
        if constexpr (VE == 4) {  // (packs of eight are there with two of them)
            if (a.d <= 512) return norm_row<T, VE, 4, 32>(a, pvec, s);
        }
        if (a.d <= 1024) return norm_row<T, VE, kV / 2, 64>(a, pvec, s);
        if (a.d <= 2048) return norm_row<T, VE, kV / 2, 128>(a, pvec, s);
        if (a.d <= 4096) return norm_row<T, VE, kV / 2, 256>(a, pvec, s);
        if (a.d <= 8192) return norm_row<T, VE, kV, 256>(a, pvec, s);
        return norm_row<T, VE, kV, 512>(a, pvec, s);
    } else {
        constexpr int k8 = 8 / VE;  // packs of eight elements
        if (a.d <= 128) return norm_row<T, VE, k8 / 2, 32>(a, pvec, s);
        if (a.d <= 256) return norm_row<T, VE, k8, 32>(a, pvec, s);
        if (a.d <= 512) return norm_row<T, VE, k8, 64>(a, pvec, s);
        if (a.d <= 1024) return norm_row<T, VE, k8, 128>(a, pvec, s);
        if (a.d <= 2048) return norm_row<T, VE, k8, 256>(a, pvec, s);
        if (a.d <= 4096) return norm_row<T, VE, k8, 512>(a, pvec, s);
        if (a.d <= 8192) return norm_row<T, VE, 2 * k8, 512>(a, pvec, s);
        return norm_row<T, VE, 4 * k8, 512>(a, pvec, s);
    }
}

template <typename T>
cudaError_t norm_t(const NormArgs& a, cudaStream_t s) {
    constexpr int VE = 16 / sizeof(T);
    if (a.d <= 16384 && a.rows <= 0x7FFFFFFF) {
        const bool pvec = aligned16(a.gamma) && aligned16(a.beta) && (a.ptype == kF32 || VE == 8);
        const auto rows_on = [&](int64_t bytes) {
            return aligned_rows(a.x, a.rows, a.ldx, sizeof(T), bytes) && (!a.y || aligned_rows(a.y, a.rows, a.ldy, sizeof(T), bytes)) &&
                   a.d * static_cast<int64_t>(sizeof(T)) % bytes == 0;
        };
        if (rows_on(16)) return norm_width<T, VE>(a, pvec, s);
        if (rows_on(2 * sizeof(T))) return norm_width<T, 2>(a, false, s);
        return norm_width<T, 1>(a, false, s);
    }
    const int64_t cap = 8ll * device_sm_count();
    norm_any_kernel<T><<<static_cast<int>(a.rows < cap ? a.rows : cap), kAnyThreads, 0, s>>>(a);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Backward with a row of x and dy in registers: TPR threads per row, VPT packs each, both row sums in
// one reduction.  Blocks walk over the rows; a thread's columns are the same in every row, so the
// parameter gradients are sums in its registers (in shared memory where a block of 1,024 threads
// leaves 64 registers a thread), written once per block.  The next row's loads are issued before this
// row's sums are joined.
// ---------------------------------------------------------------------------
// Sums of (a, b) over the TPR threads of a row; `buf` alternates between calls, so that one barrier
// separates a call's reads from the next but one's writes.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2 (*red)[32], int buf) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
        b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    if constexpr (TPR > 32) {
        const int w = threadIdx.x >> 5, w0 = w / (TPR / 32) * (TPR / 32);
        if ((threadIdx.x & 31) == 0) red[buf][w] = make_float2(a, b);
        __syncthreads();
        float2 t = red[buf][w0];
#pragma unroll
        for (int k = 1; k < TPR / 32; ++k) {
            const float2 u = red[buf][w0 + k];
            t.x += u.x, t.y += u.y;
        }
        return t;
    }
    return make_float2(a, b);
}

constexpr int grad_block(int tpr) { return tpr > 256 ? tpr : 256; }
// blocks per SM that the registers are cut for, with e elements a thread
constexpr int grad_blocks(int e, int tpr) { return tpr > 256 ? 1 : (e > 8 ? 2 : (e > 4 ? 3 : 4)); }

template <typename T, int VE, int VPT, int TPR>
__global__ void __launch_bounds__(grad_block(TPR), grad_blocks(VE * VPT, TPR))
norm_grad_row_kernel(NormGradArgs a, bool pvec) {
    constexpr int kThreads = grad_block(TPR), kRows = kThreads / TPR;
    constexpr bool kShared = TPR == 1024;
    __shared__ float2 red[2][32];
    // The block's sums: number e of a row's thread t at e * TPR + t (no bank conflicts), E of dgamma, then E
    // of dbeta; used at the end to join the row groups, with kShared all along.
    extern __shared__ float sums[];
    constexpr int E = VPT * VE;
    const int lane = threadIdx.x & 31, sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const int first = (sub >> 5) * VPT * 32 + lane;
    const float inv_d = __frcp_rn(static_cast<float>(a.d));
    float gam[VPT][VE], pg[VPT][VE], pb[VPT][VE];
    Raw<T, VE> rx[VPT], rg[VPT];
    float mu_next = 0.0f, rs_next = 0.0f;
    const bool full = (first - lane + VPT * 32) * VE <= a.d;
    auto fetch = [&](int64_t r) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx + first * VE;
        const T* dy = static_cast<const T*>(a.dy) + r * a.lddy + first * VE;
        if (r < a.rows && full) {
            mu_next = __ldg(a.mean + r), rs_next = __ldg(a.rstd + r);
#pragma unroll
            for (int j = 0; j < VPT; ++j) rx[j].load(x + j * 32 * VE), rg[j].load(dy + j * 32 * VE);
        } else {
            if (r < a.rows) mu_next = __ldg(a.mean + r), rs_next = __ldg(a.rstd + r);
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                if (r < a.rows && (first + j * 32) * VE < a.d) rx[j].load(x + j * 32 * VE), rg[j].load(dy + j * 32 * VE);
                else rx[j].zero(), rg[j].zero();
            }
        }
    };
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = (first + j * 32) * VE;
#pragma unroll
        for (int i = 0; i < VE; ++i) pg[j][i] = pb[j][i] = gam[j][i] = 0.0f;
        if (!kShared && c < a.d) load_params<T, VE>(a.gamma, a.ptype, pvec, c, 1.0f, gam[j]);
        if (kShared && a.part) {
#pragma unroll
            for (int i = 0; i < VE; ++i) sums[(j * VE + i) * TPR + sub] = sums[(E + j * VE + i) * TPR + sub] = 0.0f;
        }
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int buf = 0;
    if (!kShared) fetch(static_cast<int64_t>(blockIdx.x) * kRows + group);
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += step, buf ^= 1) {
        const int64_t r = base + group;
        const bool live = r < a.rows;
        if (kShared) fetch(r);
        const float mu = mu_next, rs = rs_next;
        float xh[VPT][VE], g[VPT][VE];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            rx[j].get(xh[j]);
            rg[j].get(g[j]);
            const int c = (first + j * 32) * VE;
            float w[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) w[i] = gam[j][i];
            if (kShared && c < a.d) load_params<T, VE>(a.gamma, a.ptype, pvec, c, 1.0f, w);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                xh[j][i] = (xh[j][i] - mu) * rs;
                const float ga = g[j][i] * w[i];
                s1 += ga;
                s2 = fmaf(ga, xh[j][i], s2);
                if constexpr (!kShared) {
                    pg[j][i] = fmaf(g[j][i], xh[j][i], pg[j][i]);
                    pb[j][i] += g[j][i];
                }
            }
            if (kShared && a.part) {
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    float& sg = sums[(j * VE + i) * TPR + sub];
                    float& sb = sums[(E + j * VE + i) * TPR + sub];
                    sg = fmaf(g[j][i], xh[j][i], sg);
                    sb += g[j][i];
                }
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) g[j][i] *= w[i];
        }
        if (!kShared) fetch(r + step);
        const float2 t = row_sum2<TPR>(s1, s2, red, buf);
        const float m1 = t.x * inv_d, m2 = t.y * inv_d;
        T* dx = static_cast<T*>(a.dx) + r * a.lddx + first * VE;
        auto put = [&](int j) {
            float o[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) o[i] = rs * (g[j][i] - m1 - xh[j][i] * m2);
            store_pack<T, VE>(dx + j * 32 * VE, o);
        };
        if (live && full) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) put(j);
        } else if (live) {
#pragma unroll
            for (int j = 0; j < VPT; ++j)
                if ((first + j * 32) * VE < a.d) put(j);
        }
    }
    if (!a.part) return;
    grid_dep_launch();  // the kernel that joins the blocks' sums may be placed
    // the block's row groups join their sums, one after the other
    if constexpr (!kShared) {
        for (int k = 1; k < kRows; ++k) {
            if (group == k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    sums[e * TPR + sub] = pg[e / VE][e % VE];
                    sums[(E + e) * TPR + sub] = pb[e / VE][e % VE];
                }
            }
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    pg[e / VE][e % VE] += sums[e * TPR + sub];
                    pb[e / VE][e % VE] += sums[(E + e) * TPR + sub];
                }
            }
            __syncthreads();
        }
        if (group != 0) return;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            pg[e / VE][e % VE] = sums[e * TPR + sub];
            pb[e / VE][e % VE] = sums[(E + e) * TPR + sub];
        }
    }
    float* out_g = a.part + static_cast<int64_t>(blockIdx.x) * a.d;
    float* out_b = a.part + (static_cast<int64_t>(a.parts) + blockIdx.x) * a.d;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = (first + j * 32) * VE;
        if (c >= a.d) continue;
        if constexpr (VE <= 2) {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                out_g[c + i] = pg[j][i];
                out_b[c + i] = pb[j][i];
            }
        } else {  // (d is a multiple of VE, the workspace 16-byte aligned)
#pragma unroll
            for (int i = 0; i < VE; i += 4) {
                *reinterpret_cast<float4*>(out_g + c + i) = make_float4(pg[j][i], pg[j][i + 1], pg[j][i + 2], pg[j][i + 3]);
                *reinterpret_cast<float4*>(out_b + c + i) = make_float4(pb[j][i], pb[j][i + 1], pb[j][i + 2], pb[j][i + 3]);
            }
        }
    }
}

// Launches as many blocks as are resident, at most a.parts, and leaves their number there.
template <typename T, int VE, int VPT, int TPR>
cudaError_t norm_grad_row(NormGradArgs& a, bool pvec, cudaStream_t s) {
    auto kern = norm_grad_row_kernel<T, VE, VPT, TPR>;
    const int smem = a.part && (TPR == 1024 || grad_block(TPR) > TPR) ? 2 * VPT * VE * TPR * 4 : 0;
    cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
    if (e != cudaSuccess) return e;
    const int resident = grad_blocks(VE * VPT, TPR) * device_sm_count();
    if (a.parts > resident) a.parts = resident;
    kern<<<a.parts, grad_block(TPR), smem, s>>>(a, pvec);
    return cudaGetLastError();
}

// Eight elements a thread up to 1,024 columns, three blocks an SM (four blocks' registers spilled: 5003x771
// fp32 17.3 us, 12.9 with three); sixteen and two blocks above, and for 16-bit packs from 257 columns on
// (65536x512 bf16: 39.6 us, 42.5 with eight).
template <typename T, int VE>
cudaError_t norm_grad_width(NormGradArgs& a, bool pvec, cudaStream_t s) {
    if constexpr (VE == 4) {
        if (a.d <= 128) return norm_grad_row<T, VE, 1, 32>(a, pvec, s);
    }
    if (a.d <= 256) return norm_grad_row<T, VE, 8 / VE, 32>(a, pvec, s);
    if constexpr (VE == 8) {
        if (a.d <= 512) return norm_grad_row<T, VE, 2, 32>(a, pvec, s);
        if (a.d <= 1024) return norm_grad_row<T, VE, 2, 64>(a, pvec, s);
    } else {
        if (a.d <= 512) return norm_grad_row<T, VE, 8 / VE, 64>(a, pvec, s);
        if (a.d <= 1024) return norm_grad_row<T, VE, 8 / VE, 128>(a, pvec, s);
    }
    if (a.d <= 2048) return norm_grad_row<T, VE, 16 / VE, 128>(a, pvec, s);
    if (a.d <= 4096) return norm_grad_row<T, VE, 16 / VE, 256>(a, pvec, s);
    if (a.d <= 8192) return norm_grad_row<T, VE, 16 / VE, 512>(a, pvec, s);
    return norm_grad_row<T, VE, 16 / VE, 1024>(a, pvec, s);
}

template <typename T>
cudaError_t norm_grad_t(NormGradArgs& a, cudaStream_t s) {
    if (a.rows == 0) return cudaSuccess;
    if (a.d <= 16384) {
        constexpr int VE = 16 / sizeof(T);
        const bool pvec = aligned16(a.gamma) && (a.ptype == kF32 || VE == 8);
        const auto rows_on = [&](int64_t bytes) {
            return aligned_rows(a.x, a.rows, a.ldx, sizeof(T), bytes) && aligned_rows(a.dy, a.rows, a.lddy, sizeof(T), bytes) &&
                   aligned_rows(a.dx, a.rows, a.lddx, sizeof(T), bytes) && a.d * static_cast<int64_t>(sizeof(T)) % bytes == 0;
        };
        if (rows_on(16)) return norm_grad_width<T, VE>(a, pvec, s);
        if (rows_on(2 * sizeof(T))) return norm_grad_width<T, 2>(a, false, s);
        return norm_grad_width<T, 1>(a, false, s);
    }
    norm_grad_any_kernel<T><<<a.parts, kAnyThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t layer_norm_launch(const NormArgs& a, int xtype, cudaStream_t s) {
    if (xtype == kF32) return norm_t<float>(a, s);
    if (xtype == kBF16) return norm_t<__nv_bfloat16>(a, s);
    return norm_t<__half>(a, s);
}

// The most blocks that the backward kernels launch, each with its own partial sums: enough to fill the
// SMs at the kernels' occupancy, few enough that the partial sums stay small against the rows.
int layer_norm_parts(int64_t rows, int64_t d) {
    const int64_t per_block = d <= 256 ? 8 : (d <= 512 ? 4 : (d <= 2048 ? 2 : 1));  // rows at a time
    const int64_t cap = (d <= 1024 ? 4ll : (d <= 4096 ? 2ll : 1ll)) * device_sm_count();
    const int64_t want = (rows + per_block - 1) / per_block;
    return static_cast<int>(want < cap ? want : cap);
}

cudaError_t column_reduce_launch(const float* part, int parts, int64_t n, void* out0, void* out1, int otype,
                                 cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    const int cols = n < 2048 ? 8 : 32;
    cfg.gridDim = dim3(static_cast<unsigned>((n + cols - 1) / cols), out1 ? 2 : 1);
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, cols == 8 ? column_reduce_kernel<8> : column_reduce_kernel<32>, part, parts, n, out0, out1, otype);
}

cudaError_t layer_norm_backward_launch(const NormGradArgs& args, int xtype, cudaStream_t s) {
    NormGradArgs a = args;
    cudaError_t e = xtype == kF32    ? norm_grad_t<float>(a, s)
                    : xtype == kBF16 ? norm_grad_t<__nv_bfloat16>(a, s)
                                     : norm_grad_t<__half>(a, s);
    if (e == cudaSuccess && (a.dgamma || a.dbeta))
        e = column_reduce_launch(a.part, a.parts, a.d, a.dgamma, a.dbeta, a.ptype, s);
    return e;
}

}  // namespace nfx
