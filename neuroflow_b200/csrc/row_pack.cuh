// row_pack.cuh -- rows of a matrix in the registers of a warp, by packs of 16 bytes (pairs of elements or
// single ones where rows are not aligned to more), and their FP8 form: shared by the layer norm and the
// quantiser.
#pragma once

#include <type_traits>

#include "block_ops.h"
#include "numerics.cuh"

namespace nfx {

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline bool aligned_rows(const void* p, int64_t rows, int64_t ld, int64_t el, int64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (rows == 1 || ld * el % bytes == 0);
}

template <typename T, int VE>
struct Pack {
    T v[VE];
};
template <int BYTES>
struct Word;
template <>
struct Word<2> { using type = uint16_t; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<16> { using type = uint4; };
template <typename T, int VE>
using word_t = typename Word<static_cast<int>(sizeof(T)) * VE>::type;

// the VE numbers of a pack
template <typename T, int VE>
__device__ __forceinline__ void unpack(word_t<T, VE> u, float (&o)[VE]) {
    const Pack<T, VE> k = *reinterpret_cast<const Pack<T, VE>*>(&u);
#pragma unroll
    for (int i = 0; i < VE; ++i) o[i] = to_f32(k.v[i]);
}
template <typename T, int VE>
__device__ __forceinline__ void load_pack(const T* p, float (&o)[VE]) {
    unpack<T, VE>(__ldg(reinterpret_cast<const word_t<T, VE>*>(p)), o);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <typename T, int VE>
__device__ __forceinline__ void store_pack(T* p, const float (&o)[VE]) {
    if constexpr (VE == 1) {
        *p = from_f32<T>(o[0]);
    } else if constexpr (sizeof(T) == 4) {
        if constexpr (VE == 2) *reinterpret_cast<float2*>(p) = make_float2(o[0], o[1]);
        else *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
    } else if constexpr (VE == 2) {
        *reinterpret_cast<uint32_t*>(p) = pack2<T>(o[0], o[1]);
    } else {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]), pack2<T>(o[4], o[5]), pack2<T>(o[6], o[7]));
    }
}
// The codes of four values times `inv` (two products to an instruction, each rounded by itself): plain
// conversions that note in `odd` where they may differ from the encoder, or, with MEND, its codes.
template <bool MEND>
__device__ __forceinline__ uint32_t scaled_codes(float a, float b, float c, float d, float inv, uint32_t& odd) {
    const float2 p = mul2_rn(make_float2(a, b), make_float2(inv, inv)), q = mul2_rn(make_float2(c, d), make_float2(inv, inv));
    const uint32_t w = e4m3_convert4(p.x, p.y, q.x, q.y, odd);
    return MEND ? e4m3_mend4(w, p.x, p.y, q.x, q.y) : w;
}

// FP8 codes of a lane's VPT packs (values v, zero beyond column d): pack j holds columns (first_pack +
// 32 j) VE .., so a group of 128 lies in one warp.  A group's maximum is taken over all its elements
// first and again over the finite ones where it is infinite (a NaN is no maximum anyway).  The
// division and the reciprocal of a scale are done by one lane per group, all groups at once.  `wide`:
// code rows start on 8-byte boundaries.
template <int VE, int VPT, int TPR>
__device__ __forceinline__ void store_codes(const float (&v)[VPT][VE], const Fp8Out& q, int64_t r, int64_t d, bool live,
                                            int64_t first_pack, int lane, bool wide) {
    constexpr int kPer = VE <= 2 ? 4 / VE : 1;                                      // packs of a lane in one group
    constexpr int kLanes = VE <= 2 ? 32 : (kGroup / VE < TPR ? kGroup / VE : TPR);  // lanes of one group
    constexpr int kGroups = VPT / kPer;
    static_assert(kGroups <= kLanes, "a lane for each group");
    float am[kGroups];
    auto maxima = [&](bool finite) {
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            am[j] = 0.0f;
#pragma unroll
            for (int h = 0; h < kPer; ++h)
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    am[j] = fmaxf(am[j], finite ? finite_abs(v[j * kPer + h][i]) : fabsf(v[j * kPer + h][i]));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) am[j] = fmaxf(am[j], __shfl_xor_sync(0xFFFFFFFFu, am[j], o));
        }
    };
    maxima(false);
    float mine = am[0], top = am[0];
    const int at = lane % kLanes;
#pragma unroll
    for (int j = 1; j < kGroups; ++j) top = fmaxf(top, am[j]);
    if (__any_sync(0xFFFFFFFFu, !(top <= 3.402823466e38f))) {
        maxima(true);
        mine = am[0];
    }
#pragma unroll
    for (int j = 1; j < kGroups; ++j) mine = at == j ? am[j] : mine;
    const float sc = group_scale(mine), inv_mine = __frcp_rn(sc);
    // the first column of group `at` of this lane's row
    const int64_t c_at = (first_pack - at + static_cast<int64_t>(at) * kPer * 32) * VE;
    if (live && at < kGroups && c_at < d) q.scales[r * q.srs + (c_at / kGroup) * q.sbs] = sc;
    uint32_t odd = 0;
    auto write = [&](auto mend) {
        constexpr bool kMend = decltype(mend)::value;
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            const float inv = __shfl_sync(0xFFFFFFFFu, inv_mine, j, kLanes);
            const int64_t c0 = (first_pack + j * kPer * 32) * VE;  // this lane's first column
            uint8_t* dst = q.codes + r * q.ld + c0;
            if constexpr (VE == 1) {
                const uint32_t w = scaled_codes<kMend>(v[4 * j][0], v[4 * j + 1][0], v[4 * j + 2][0], v[4 * j + 3][0], inv, odd);
                if (live && c0 - lane + kGroup <= d) {
#pragma unroll
                    for (int h = 0; h < 4; ++h) dst[h * 32] = static_cast<uint8_t>(w >> (8 * h));
                } else {
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        if (live && c0 + h * 32 < d) dst[h * 32] = static_cast<uint8_t>(w >> (8 * h));
                }
            } else if constexpr (VE == 2) {
                const uint32_t w = scaled_codes<kMend>(v[2 * j][0], v[2 * j][1], v[2 * j + 1][0], v[2 * j + 1][1], inv, odd);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!live || c0 + h * 64 >= d) continue;
                    if (wide) {
                        *reinterpret_cast<uint16_t*>(dst + h * 64) = static_cast<uint16_t>(w >> (16 * h));
                    } else {
                        dst[h * 64] = static_cast<uint8_t>(w >> (16 * h));
                        dst[h * 64 + 1] = static_cast<uint8_t>(w >> (16 * h + 8));
                    }
                }
            } else {
                uint32_t w[VE / 4];
#pragma unroll
                for (int i = 0; i < VE / 4; ++i)
                    w[i] = scaled_codes<kMend>(v[j][4 * i], v[j][4 * i + 1], v[j][4 * i + 2], v[j][4 * i + 3], inv, odd);
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
    };
    write(std::false_type{});
    if (__any_sync(0xFFFFFFFFu, odd != 0)) write(std::true_type{});  // (rare; the same bytes again, put right)
}

}  // namespace nfx
