// row_pack.cuh -- rows of a matrix in the registers of a warp, by packs of 16 bytes (or single
// elements), and their FP8 form: shared by the layer norm and the quantiser.
#pragma once

#include "block_ops.h"
#include "numerics.cuh"

namespace nfx {

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T, int VE>
struct Pack {
    T v[VE];
};
template <typename T, int VE>
__device__ __forceinline__ void load_pack(const T* p, float (&o)[VE]) {
    if constexpr (VE == 1) {
        o[0] = to_f32(__ldg(p));
    } else {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        const Pack<T, VE> k = *reinterpret_cast<const Pack<T, VE>*>(&u);
#pragma unroll
        for (int i = 0; i < VE; ++i) o[i] = to_f32(k.v[i]);
    }
}
template <typename T, int VE>
__device__ __forceinline__ void store_pack(T* p, const float (&o)[VE]) {
    if constexpr (VE == 1) {
        *p = from_f32<T>(o[0]);
    } else {
        Pack<T, VE> k;
#pragma unroll
        for (int i = 0; i < VE; ++i) k.v[i] = from_f32<T>(o[i]);
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&k);
    }
}
// FP8 codes of a lane's VPT packs (values v, zero beyond column d): pack j holds columns (first_pack +
// 32 j) VE .., so a group of 128 lies in one warp.  A group's maximum is taken over all its elements
// first and again over the finite ones where it is infinite (a NaN is no maximum anyway).  `wide`:
// code rows start on 8-byte boundaries.
template <int VE, int VPT, int TPR>
__device__ __forceinline__ void store_codes(const float (&v)[VPT][VE], const Fp8Out& q, int64_t r, int64_t d, bool live,
                                            int64_t first_pack, int lane, bool wide) {
    constexpr int kPerGroup = VE == 1 ? 4 : 1;                                      // packs of a lane in one group
    constexpr int kLanes = VE == 1 ? 32 : (kGroup / VE < TPR ? kGroup / VE : TPR);  // lanes of one group
#pragma unroll
    for (int j = 0; j < VPT; j += kPerGroup) {
        float am = 0.0f;
#pragma unroll
        for (int h = 0; h < kPerGroup; ++h)
#pragma unroll
            for (int i = 0; i < VE; ++i) am = fmaxf(am, fabsf(v[j + h][i]));
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xFFFFFFFFu, am, o));
        if (__any_sync(0xFFFFFFFFu, !(am <= 3.402823466e38f))) {
            am = 0.0f;
#pragma unroll
            for (int h = 0; h < kPerGroup; ++h)
#pragma unroll
                for (int i = 0; i < VE; ++i) am = fmaxf(am, finite_abs(v[j + h][i]));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xFFFFFFFFu, am, o));
        }
        const float sc = group_scale(am), inv = __frcp_rn(sc);
        const int64_t c0 = (first_pack + j * 32) * VE;  // this lane's first column
        if (live && c0 < d && (VE == 1 ? lane == 0 : lane % kLanes == 0)) q.scales[r * q.srs + (c0 / kGroup) * q.sbs] = sc;
        uint8_t* dst = q.codes + r * q.ld + c0;
        if constexpr (VE == 1) {
            const uint32_t w = e4m3_encode4(v[j][0] * inv, v[j + 1][0] * inv, v[j + 2][0] * inv, v[j + 3][0] * inv);
#pragma unroll
            for (int h = 0; h < 4; ++h)
                if (live && c0 + h * 32 < d) dst[h * 32] = static_cast<uint8_t>(w >> (8 * h));
        } else {
            uint32_t w[VE / 4];
#pragma unroll
            for (int i = 0; i < VE / 4; ++i)
                w[i] = e4m3_encode4(v[j][4 * i] * inv, v[j][4 * i + 1] * inv, v[j][4 * i + 2] * inv, v[j][4 * i + 3] * inv);
            if (!live || c0 >= d) continue;
            if (wide) {
                if constexpr (VE == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t*>(dst) = w[0];
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i) dst[i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i % 4)));
            }
        }
    }
}

}  // namespace nfx
