// rms_parts.cuh -- what the RMS norm's forward and backward kernels share: packs of a row whose first element
// may lie anywhere, and sums over a row's threads.
//
// Rows that do not start on 16-byte boundaries (an odd width) are read by 16-byte words all the same: up to VE - 1
// elements in front of the first boundary and behind the last one are the row's edges, an element each for the
// first lanes of its first warp, and what lies between them is whole packs.  That asks for tensors whose rows start
// at the same distance from a boundary, counted in elements (tensors of one shape, contiguous, do); elsewhere
// packs are single elements.
#pragma once

#include "block_ops.h"
#include "row_pack.cuh"

namespace nfx {

// VE elements as they were read.
template <typename T, int VE>
struct Elems {
    static constexpr int kWords = (static_cast<int>(sizeof(T)) * VE + 3) / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kWords >= 4) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
                w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
            }
        } else if constexpr (sizeof(T) == 4) {
            w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        } else {
            w[0] = __ldg(reinterpret_cast<const uint16_t*>(p));
        }
    }
    // by an ordinary load, of what this kernel has written
    __device__ __forceinline__ void load_plain(const T* p) {
        if constexpr (kWords >= 4) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 u = reinterpret_cast<const uint4*>(p)[i / 4];
                w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
            }
        } else if constexpr (sizeof(T) == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float((i & 1) ? (w[i / 2] & 0xFFFF0000u) : (w[i / 2] << 16));
        else return __half2float(__ushort_as_half(static_cast<unsigned short>((i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu)));
    }
    __device__ __forceinline__ void get(float (&o)[VE]) const {
#pragma unroll
        for (int i = 0; i < VE; ++i) o[i] = at(i);
    }
    // rounds and packs
    __device__ __forceinline__ void set(const float (&o)[VE]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < VE; ++i) w[i] = __float_as_uint(o[i]);
        } else if constexpr (VE == 1) {
            const T t = from_f32<T>(o[0]);
            w[0] = *reinterpret_cast<const uint16_t*>(&t);
        } else {
#pragma unroll
            for (int i = 0; i < VE; i += 2) w[i / 2] = pack2<T>(o[i], o[i + 1]);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kWords >= 4) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<uint32_t*>(p) = w[0];
        } else {
            *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
        }
    }
};

// The sum of `a` over a row's threads, the same bits in each of them: a warp (ONE), or all `warps` of the block.
// `red` alternates between two buffers, so that one barrier separates a call's reads from the next but one's
// writes.
template <bool ONE>
__device__ __forceinline__ float row_sum(float a, float* red, int warps) {
    a = warp_sum(a);
    if constexpr (!ONE) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
        __syncthreads();
        a = red[0];
        for (int k = 1; k < warps; ++k) a += red[k];
    }
    return a;
}

// How a row of d elements that starts s elements behind a boundary falls into edges and packs, and the edge element
// that a thread takes (its column, or -1).
template <int VE>
struct Split {
    int head, packs, edge;
    __device__ __forceinline__ Split(int d, int s, int sub) {
        head = min((VE - s) % VE, d);
        packs = (d - head) / VE;
        const int tail = head + packs * VE;
        edge = sub < head ? sub : (sub >= VE && tail + sub - VE < d && sub < 2 * VE ? tail + sub - VE : -1);
    }
};

// Four columns' codes, and by the group's first lane its scale: group b of row r, columns c .. c + 3.
__device__ __forceinline__ void store_codes4(const Fp8Out& q, int64_t r, int b, int c, int d, int lane, bool wide, const float (&o)[4], float sc,
                                             float inv) {
    uint32_t odd = 0, w = scaled_codes<false>(o[0], o[1], o[2], o[3], inv, odd);
    if (odd) w = scaled_codes<true>(o[0], o[1], o[2], o[3], inv, odd);
    if (lane == 0) q.scales[r * q.srs + b * q.sbs] = sc;
    uint8_t* dst = q.codes + r * q.ld + c;
    if (wide && c + 4 <= d) {
        *reinterpret_cast<uint32_t*>(dst) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < d) dst[i] = static_cast<uint8_t>(w >> (8 * i));
    }
}

// The distance in elements from the last VE-element boundary to a matrix' first element, and how a row moves it.
struct Shift {
    int base, step;
};
inline Shift shift_of(const void* p, int64_t ld, int64_t el, int ve) {
    return {static_cast<int>(reinterpret_cast<uintptr_t>(p) / static_cast<uintptr_t>(el) % static_cast<uintptr_t>(ve)), static_cast<int>(ld % ve)};
}
inline bool same_shift(const Shift& a, const Shift& b, int64_t rows) { return a.base == b.base && (rows <= 1 || a.step == b.step); }

}  // namespace nfx
