// gemm_parts.cuh -- what the FP8 and the 16-bit matrix products share: the register split between warps, the
// order of tiles, reads of TMEM and of a cluster's shared memory, GELU, and packing of results.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "block_ops.h"
#include "launch.cuh"
#include "numerics.cuh"
#include "sm100.cuh"

namespace nfx {

// GELU as z * sigmoid(2u) (the tanh form's identity), the exponential by ex2.approx.  Two values
// share a reciprocal, 1 / a = b / (a b) (the special-function unit bounds this epilogue); the
// exponents are held under 2^60 so that the product stays finite.  Where that bites, z < -7 or so, the
// result is under 2^-57 in size and is returned as zero; a NaN stays one and leaves its neighbour alone.
__device__ __forceinline__ float2 gelu_sig2(float2 z) {
    const float c2 = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
    float2 e;
    const float ux = c2 * fmaf(z.x, (0.044715f * z.x) * z.x, z.x), uy = c2 * fmaf(z.y, (0.044715f * z.y) * z.y, z.y);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(fminf(ux, 60.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(fminf(uy, 60.0f)));
    const float a = 1.0f + e.x, b = 1.0f + e.y, r = __fdividef(1.0f, a * b);
    return make_float2((ux > 60.0f ? -0.0f : z.x) * (r * b), (uy > 60.0f ? -0.0f : z.y) * (r * a));
}
// Terms that a tensor core sums by itself before the sum is joined with others in fp32.  It cuts its running sum off instead
// of rounding it, so a sum of numbers of one sign comes out low, the more the longer it is: by 3e-6 of itself after 512
// terms, where fp32 results stop, by 2.4e-5 after 4,096, a twentieth of an fp16 result's own rounding, where 16-bit
// results do, and by 3.9e-4 after 65,536.
constexpr int piece_terms(int ct) { return ct == kF32 ? 512 : 4096; }

template <int R>
__device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

template <int CT>
__device__ __forceinline__ uint32_t pack_half(float2 a) {
    if constexpr (CT == kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a.x, a.y);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a.x, a.y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <int CT>
__device__ __forceinline__ float2 unpack_half(uint32_t w) {
    if constexpr (CT == kBF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Columns c0 .. of a row as the bytes of one staging chunk (16 bytes).
template <int CT, int NP>
__device__ __forceinline__ uint4 pack_chunk(const float2 (&acc)[NP], int j) {
    uint4 v;
    if constexpr (CT == kF32) {
        v = make_uint4(__float_as_uint(acc[2 * j].x), __float_as_uint(acc[2 * j].y),
                       __float_as_uint(acc[2 * j + 1].x), __float_as_uint(acc[2 * j + 1].y));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_half<CT>(acc[4 * j + i]);
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
}

// Tile t of a grid of tm x tn tiles: bands of 16 row tiles, row tiles fastest inside a band, so
// that the tiles in flight share operand rows in L2.
__device__ __forceinline__ void tile_at(int t, int tm, int tn, int& m, int& n) {
    const int band = 16 * tn, b = t / band, rem = t % band;
    const int h = min(16, tm - b * 16);
    m = b * 16 + rem % h;
    n = rem / h;
}

// W columns of this warp's TMEM lanes, complete on return.  Load and wait are one statement: a wait
// that names the registers of earlier loads as its operands makes the compiler copy them, which cost
// more than the overlap of the loads gained.
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

// Element i of a matrix that may be written by this very call (an ordinary load).
template <int CT>
__device__ __forceinline__ float plain_load(const void* p, int64_t i) {
    if constexpr (CT == kF32) return static_cast<const float*>(p)[i];
    else if constexpr (CT == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    else return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ float ld_cluster(uint32_t cluster_addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(cluster_addr)
                 : "memory");
    return v;
}


// Elements [i, i + N) of a row; those from `end` on are zeros.
template <int N>
__device__ __forceinline__ void load_single(const uint16_t* p, int i, int end, uint32_t (&w)[N / 2]) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        const uint32_t lo = i + 2 * j < end ? __ldg(p + i + 2 * j) : 0, hi = i + 2 * j + 1 < end ? __ldg(p + i + 2 * j + 1) : 0;
        w[j] = lo | hi << 16;
    }
}
// Eight elements from p on, which lies on a 16-byte boundary (VEC) or anywhere: then the two words that hold them are
// read, up to 14 bytes in front of p and behind its eight elements, and moved into place.
template <bool VEC>
__device__ __forceinline__ void load8(const uint16_t* p, uint32_t (&w)[4]) {
    if constexpr (VEC) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
        const int q = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 7;
        const uint4* b = reinterpret_cast<const uint4*>(p - q);
        const uint4 u = __ldg(b), v = __ldg(b + (q ? 1 : 0));
        uint32_t m[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 6; ++i) m[i] = q & 4 ? m[i + 2] : m[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) m[i] = q & 2 ? m[i + 1] : m[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = q & 1 ? __funnelshift_r(m[i], m[i + 1], 16) : m[i];
    }
}

}  // namespace nfx
