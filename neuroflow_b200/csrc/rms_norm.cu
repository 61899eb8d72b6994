// rms_norm.cu -- root-mean-square norm over the last dimension of (rows, d) with the residual's addition,
// into the input's type or straight into FP8 groups of 128.
//
//   h = x + res, rounded to the residual's type;  r = 1 / sqrt(sum h^2 / d + eps)
//   y = h r gamma
//
// The norm is that of the sum as it is stored, so the backward pass, which reads the stored sum, is the
// gradient of exactly what was computed.  All sums are fp32.
//
// Bound by HBM.  Measured (one B200, copies at 6,543 GB/s; GPU time in graphs of launches over rows that do not fit L2):
//   16384x4096 bf16 + fp32 stream   134 us, 6.0 TB/s (bf16 + bf16 89 us, into FP8 76 us, 6.2 TB/s)
//   8191x2048 bf16 into FP8         20.6 us, 5.7 TB/s
//   8192x2047 bf16                  24.1 us, 5.6 TB/s: rows that start anywhere (into FP8 29 us, instructions)
//   5003x1031 fp16                  9.6 us, 4.3 TB/s;   131072x128 fp32   43 us, 6.2 TB/s
//   4096x16384, 2048x20000 bf16     106 us, 5.1 TB/s;   127 us, 2.6 TB/s (two sweeps)
//   1x4096 bf16                     1.8 us
#include <atomic>

#include "dense_ops.h"
#include "launch.cuh"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "rms_parts.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

// Wider rows than the registers hold: a block of 512 threads takes a row in two sweeps, the second from L2.  An
// element of a row is the same thread's in both.
constexpr int kWideThreads = 512;

template <typename T, typename H, int VE, bool FP8>
__global__ void __launch_bounds__(kWideThreads, 2) rms_wide_kernel(RmsArgs a, Shift sh, bool wide) {
    __shared__ float red[2][kWideThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x;
    grid_dep_launch();
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on
    int buf = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, buf ^= 1) {
        const Split<VE> sp(a.d, static_cast<int>((sh.base + r * sh.step) % VE), tid);
        const uint32_t packs = sp.packs;  // (up to 2^31: the number of the next one has no sign)
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        const H* res = a.res ? static_cast<const H*>(a.res) + r * a.ldres : nullptr;
        H* sum = a.sum ? static_cast<H*>(a.sum) + r * a.ldsum : nullptr;
        // x + res as it is stored; plain loads where the first sweep has written
        const auto pack = [&](int c, bool again, float (&v)[VE]) {
            if (again && sum) {
                Elems<H, VE> e;
                e.load_plain(sum + c);
                e.get(v);
                return;
            }
            Elems<T, VE> e;
            e.load(x + c);
            e.get(v);
            if (!res) return;
            Elems<H, VE> f;
            f.load(res + c);
#pragma unroll
            for (int i = 0; i < VE; ++i) v[i] += f.at(i);
            f.set(v);
            f.get(v);
            if (!again && sum) f.store(sum + c);
        };
        const auto single = [&](int c, bool again) {
            if (again && sum) return to_f32(sum[c]);
            const float v = to_f32(x[c]);
            if (!res) return v;
            const H h = from_f32<H>(v + to_f32(res[c]));
            if (!again && sum) sum[c] = h;
            return to_f32(h);
        };
        float q = 0.0f;
        for (uint32_t k = tid; k < packs; k += kWideThreads) {
            float v[VE];
            pack(sp.head + static_cast<int>(k) * VE, false, v);
#pragma unroll
            for (int i = 0; i < VE; ++i) q = fmaf(v[i], v[i], q);
        }
        if (VE > 1 && sp.edge >= 0) {
            const float v = single(sp.edge, false);
            q = fmaf(v, v, q);
        }
        const float rs = __frsqrt_rn(__fdiv_rn(row_sum<false>(q, red[buf], kWideThreads / 32), static_cast<float>(a.d)) + a.eps);
        if (tid == 0 && a.rstd) a.rstd[r] = rs;
        const auto gamma = [&](int c) { return a.gamma ? load_any(a.gamma, a.ptype, c) : 1.0f; };
        if constexpr (!FP8) {
            T* y = static_cast<T*>(a.y) + r * a.ldy;
            for (uint32_t k = tid; k < packs; k += kWideThreads) {
                const int c = sp.head + static_cast<int>(k) * VE;
                float v[VE];
                pack(c, true, v);
#pragma unroll
                for (int i = 0; i < VE; ++i) v[i] = (v[i] * rs) * gamma(c + i);
                Elems<T, VE> o;
                o.set(v);
                o.store(y + c);
            }
            if (VE > 1 && sp.edge >= 0) y[sp.edge] = from_f32<T>((single(sp.edge, true) * rs) * gamma(sp.edge));
        } else {
            if (sum) __syncthreads();  // the groups below are read by other threads than wrote the sum
            const int blocks = (a.d + kGroup - 1) / kGroup;
            for (int b = warp; b < blocks; b += kWideThreads / 32) {
                const int c = b * kGroup + lane * 4;
                float o[4], top = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[i] = c + i < a.d ? (single(c + i, true) * rs) * gamma(c + i) : 0.0f;
                    top = fmaxf(top, finite_abs(o[i]));
                }
                const float sc = group_scale(warp_max(top));
                if (c < a.d) store_codes4(a.q, r, b, c, a.d, lane, wide, o, sc, __frcp_rn(sc));
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// The row in registers: read once, written from there.  A row is a warp's (ONE, four rows to a block) or a whole
// block's, of as many warps as it takes; a thread holds VPT packs of VE elements (16 bytes of x), pack j of
// lane l of warp w being (w VPT + j) 32 + l of the row, so the 128 elements of an FP8 group lie in one warp.
// Resident blocks walk over the rows: the next row is fetched while this one is worked on, and gamma stays where
// it is, in registers, or in shared memory for rows over 4,096 columns.  EDGE: rows start and end anywhere
// (rms_parts.cuh).
// ---------------------------------------------------------------------------------------------------------
// Blocks per SM that the registers are cut for: 768 threads where a row on its way takes up to 16 registers, 512 where it
// takes more or its edges ask for more (into FP8, 8192x2047 bf16: 33 us with 768 threads, 29 with 512); of 512 threads two
// only where FP8 codes take the time (8192x8192 bf16 to FP8: 98 us with one, 86 with two; into bf16 97 and 103).
constexpr int row_blocks(int most, int coming, bool fp8, bool edge) {
    if (most >= 512) return fp8 && !edge && coming <= 16 ? 2 : 1;
    return (coming <= 8 || (coming <= 16 && !(edge && (fp8 || most == 128))) ? 768 : 512) / most;
}
// Where gamma is: in a thread's registers, up to 16 of them, or in shared memory.
constexpr bool gamma_shared(bool one, int most, int elements) { return !one && (most >= 512 || elements > 16); }

// f(the number as a constant) for 1 <= cut <= VE: what depends on it then costs nothing, in a loop whose instructions count.
template <int VE, typename F>
__device__ __forceinline__ void with_cut(int cut, const F& f) {
    switch (cut) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 5: return f(std::integral_constant<int, VE == 8 ? 5 : 4>{});
        case 6: return f(std::integral_constant<int, VE == 8 ? 6 : 4>{});
        case 7: return f(std::integral_constant<int, VE == 8 ? 7 : 4>{});
        default: return f(std::integral_constant<int, VE>{});
    }
}

// FP8 codes of a row whose packs begin `head` columns behind the groups' (0 <= head < VE): pack k of the row lies in group
// k VE / 128, but the last `head` elements of each group's last pack belong to the next one.  A warp knows all that its
// groups have, but for the first and the one behind the last, which it shares with its neighbours (`shared`: for each warp
// what the one before leaves to its first group, and what it has of that group itself).  A lane's codes and the last ones
// of the lane before it make an aligned word; the two ends of what a warp holds are stored by bytes.
template <int VE, int VPT, bool ONE>
__device__ __forceinline__ void store_codes_shifted(const float (&v)[VPT][VE], float ev, const Split<VE>& sp, const Fp8Out& q, int64_t r, int d, bool live,
                                                    int first, int lane, int warp, bool last_warp, uint2* shared) {
    constexpr int kLanes = kGroup / VE, kPer = 32 / kLanes;  // lanes of a group, groups of a warp's pack
    constexpr int kWords = VE / 4;                           // of a pack's codes
    const int groups = (d + kGroup - 1) / kGroup, base = first - lane, g0 = base / kLanes, at = lane / kLanes, cut = VE - sp.head;
    const bool over = sp.head > 0 && lane % kLanes == kLanes - 1;  // this lane's packs lie in two groups
    float lo[VPT], hi[VPT];
    with_cut<VE>(cut, [&](auto c) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            lo[j] = hi[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                if (i < c) lo[j] = fmaxf(lo[j], fabsf(v[j][i]));
                else hi[j] = fmaxf(hi[j], fabsf(v[j][i]));
            }
        }
    });
    float most = fmaxf(lo[0], hi[0]);
#pragma unroll
    for (int j = 1; j < VPT; ++j) most = fmaxf(most, fmaxf(lo[j], hi[j]));
    if (__any_sync(0xFFFFFFFFu, !(most <= 3.402823466e38f))) {  // (over the finite ones again)
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            lo[j] = hi[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float m = finite_abs(v[j][i]);
                if (i < cut) lo[j] = fmaxf(lo[j], m);
                else hi[j] = fmaxf(hi[j], m);
            }
        }
    }
    // Maxima of numbers by their bits, whose order is the same; lane k takes the warp's group k.
    const float em = sp.edge >= 0 ? finite_abs(ev) : 0.0f;
    uint32_t mine = 0, left = 0;  // `left`: what the pack before leaves to the group at hand
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        float f = over ? lo[j] : fmaxf(lo[j], hi[j]);
        if (j == 0 && sp.edge < sp.head) f = fmaxf(f, em);  // (the row's first elements are its first warp's)
        const uint32_t m = __float_as_uint(f);
#pragma unroll
        for (int h = 0; h < kPer; ++h) {
            const uint32_t all = max(left, __reduce_max_sync(0xFFFFFFFFu, kPer == 1 || at == h ? m : 0u));
            left = __float_as_uint(__shfl_sync(0xFFFFFFFFu, hi[j], h * kLanes + kLanes - 1));
            if (lane == j * kPer + h) mine = all;
        }
    }
    if (lane == VPT * kPer) mine = left;
    if (last_warp) {  // the row's last elements: in one group or two
        const int c = sp.head + sp.packs * VE, k = c / kGroup;
        const uint32_t m = sp.edge >= c ? __float_as_uint(em) : 0u;
        const bool next = sp.edge >= (k + 1) * kGroup;
        const uint32_t a = __reduce_max_sync(0xFFFFFFFFu, next ? 0u : m), b = __reduce_max_sync(0xFFFFFFFFu, next ? m : 0u);
        mine = max(mine, lane == k - g0 ? a : (lane == k + 1 - g0 ? b : 0u));
    }
    if constexpr (!ONE) {
        if (lane == 0) shared[warp + 1].x = left, shared[warp].y = mine;
        __syncthreads();
        if (lane == 0 && warp > 0) mine = max(mine, shared[warp].x);
        if (lane == VPT * kPer && !last_warp) mine = max(mine, shared[warp + 1].y);
    }
    const int g = g0 + lane;
    const bool has = lane <= VPT * kPer && g < groups;
    // (448 for a lane without a group: a division of zero takes the long way)
    const float sc = group_scale(has ? __uint_as_float(mine) : kE4m3Max), inv = __frcp_rn(sc);
    if (live && has && (lane < VPT * kPer || last_warp)) q.scales[r * q.srs + g * q.sbs] = sc;
    float mult[VPT], rest[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        mult[j] = __shfl_sync(0xFFFFFFFFu, inv, j * kPer + at);
        rest[j] = __shfl_sync(0xFFFFFFFFu, inv, j * kPer + at + (over ? 1 : 0));
    }
    uint32_t w[VPT][kWords], odd = 0;
    const auto codes = [&](auto mend, auto c) {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int i = 0; i < VE; i += 4) {
                const auto by = [&](int e) { return e < c ? mult[j] : rest[j]; };
                w[j][i / 4] = scaled_codes<decltype(mend)::value>(v[j][i], v[j][i + 1], v[j][i + 2], v[j][i + 3], make_float2(by(i), by(i + 1)),
                                                                  make_float2(by(i + 2), by(i + 3)), odd);
            }
    };
    with_cut<VE>(cut, [&](auto c) { codes(std::false_type{}, c); });
    if (__any_sync(0xFFFFFFFFu, odd != 0)) codes(std::true_type{}, cut);  // (rare)
    uint8_t* const row = q.codes + r * q.ld;
    const int behind = static_cast<int>((reinterpret_cast<uintptr_t>(row) + sp.head) % VE);  // bytes from a boundary to a pack's codes
    uint8_t* const dst = row + sp.head + first * VE;
    const int bits = 8 * (behind & 3);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        uint32_t prev[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) prev[i] = __shfl_sync(0xFFFFFFFFu, j > 0 && lane == 31 ? w[j > 0 ? j - 1 : 0][i] : w[j][i], (lane + 31) & 31);
        if (!live || first + j * 32 >= sp.packs || (j == 0 && lane == 0 && behind > 0)) continue;
        if constexpr (VE == 8) {
            const bool far = behind >= 4;
            const uint32_t a = far ? prev[0] : prev[1], b = far ? prev[1] : w[j][0], c = far ? w[j][0] : w[j][1];
            *reinterpret_cast<uint2*>(dst + j * 32 * VE - behind) = make_uint2(__funnelshift_l(a, b, bits), __funnelshift_l(b, c, bits));
        } else {
            *reinterpret_cast<uint32_t*>(dst + j * 32 * VE - behind) = __funnelshift_l(prev[0], w[j][0], bits);
        }
    }
    const int packs = min(sp.packs - base, 32 * VPT);  // of this warp
    if (behind > 0 && live && packs > 0) {
        // lanes 0 .. VE - 1: the bytes of the warp's first pack up to a boundary; VE .. 2 VE - 1: those of its last pack from one
        const int end = (packs - 1) >> 5, b = lane % VE;
        const bool tail = lane >= VE;
        uint32_t u[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            uint32_t e = w[0][i];
#pragma unroll
            for (int j = 1; j < VPT; ++j) e = end == j ? w[j][i] : e;
            const uint32_t x = __shfl_sync(0xFFFFFFFFu, w[0][i], 0), y = __shfl_sync(0xFFFFFFFFu, e, (packs - 1) & 31);
            u[i] = tail ? y : x;
        }
        const uint32_t byte = (VE == 8 && b >= 4 ? u[kWords - 1] : u[0]) >> (8 * (b & 3));
        if (lane < 2 * VE && tail == (b >= VE - behind)) row[sp.head + (base + (tail ? packs - 1 : 0)) * VE + b] = static_cast<uint8_t>(byte);
    }
    const float einv = __shfl_sync(0xFFFFFFFFu, inv, sp.edge >= 0 ? sp.edge / kGroup - g0 : 0);
    if (live && sp.edge >= 0) row[sp.edge] = e4m3_encode_fast(__fmul_rn(ev, einv));
}

template <typename T, typename H, int VE, int VPT, int MOST, bool ONE, bool FP8, bool EDGE>
__global__ void __launch_bounds__(MOST, row_blocks(MOST, VE * VPT * static_cast<int>(sizeof(T) + sizeof(H)) / 4, FP8, EDGE))
rms_row_kernel(RmsArgs a, Shift sh, bool gvec, bool wide) {
    __shared__ float red[2][MOST / 32];
    __shared__ uint2 shared[FP8 && EDGE && !ONE ? MOST / 32 + 1 : 1];
    extern __shared__ __align__(16) float room[];  // gamma (rows over 4,096 columns)
    constexpr int kRows = ONE ? MOST / 32 : 1;
    constexpr bool kGammaShared = gamma_shared(ONE, MOST, VPT * VE), kEdges = EDGE && VE > 1;
    const int lane = threadIdx.x & 31, warps = ONE ? 1 : blockDim.x >> 5;
    const int sub = ONE ? lane : threadIdx.x, mine = ONE ? threadIdx.x >> 5 : 0;
    const int first = (sub >> 5) * VPT * 32 + lane, elems = warps * 32 * VPT * VE;
    const float inv_d = __frcp_rn(static_cast<float>(a.d));
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    // (the launcher makes `step` rows a whole number of boundaries: s is the same in all rows of a thread)
    const int s = EDGE ? static_cast<int>((sh.base + (static_cast<int64_t>(blockIdx.x) * kRows + mine) * sh.step) % VE) : 0;
    // (a row's last elements are the first ones' warp's or, on their way to FP8, the last warp's: its lanes know their groups)
    const int edge = !FP8 || sub < VE ? sub : ((sub >> 5) == warps - 1 && lane >= VE ? lane : 2 * VE);
    const Split<VE> sp(a.d, s, edge);
    const auto column = [&](int j) { return (EDGE ? sp.head : 0) + (first + j * 32) * VE; };
    const auto inside = [&](int j) { return EDGE ? first + j * 32 < sp.packs : (first + j * 32) * VE < a.d; };

    Elems<T, VE> rx[VPT];
    Elems<H, VE> rr[VPT];
    Elems<T, 1> ex;  // the edge element
    Elems<H, 1> er;
    ex.zero(), er.zero();
    const auto fetch = [&](int64_t r) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        const H* res = static_cast<const H*>(a.res) + r * a.ldres;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = column(j);
            if (r < a.rows && inside(j)) {
                rx[j].load(x + c);
                if (a.res) rr[j].load(res + c);
            } else {
                rx[j].zero();
                rr[j].zero();
            }
        }
        if (kEdges && sp.edge >= 0 && r < a.rows) {
            ex.load(x + sp.edge);
            if (a.res) er.load(res + sp.edge);
        }
    };
    grid_dep_launch();
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on
    fetch(static_cast<int64_t>(blockIdx.x) * kRows + mine);
    float gam[kGammaShared ? 1 : VPT][VE];
    if constexpr (kGammaShared) {
        for (int i = threadIdx.x; i < elems; i += blockDim.x)
            room[i] = a.gamma && column(0) - first * VE + i < a.d ? load_any(a.gamma, a.ptype, column(0) - first * VE + i) : 1.0f;
        __syncthreads();
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = column(j);
            if (!EDGE && c < a.d) {
                load_params<T, VE>(a.gamma, a.ptype, gvec, c, 1.0f, gam[j]);
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i) gam[j][i] = EDGE && a.gamma && c + i < a.d ? load_any(a.gamma, a.ptype, c + i) : 1.0f;
            }
        }
    }
    const float egam = kEdges && a.gamma && sp.edge >= 0 ? load_any(a.gamma, a.ptype, sp.edge) : 1.0f;
    int buf = 0;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += step, buf ^= 1) {
        const int64_t r = base + mine;
        const bool live = r < a.rows;
        float v[VPT][VE];
        float2 q2 = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            rx[j].get(v[j]);
            if (a.res) {
                float h[VE];
                rr[j].get(h);
#pragma unroll
                for (int i = 0; i < VE; ++i) v[j][i] += h[i];
                Elems<H, VE> o;
                o.set(v[j]);  // the norm is that of the sum as it is stored
                o.get(v[j]);
                if (a.sum && live) {
                    H* sum = static_cast<H*>(a.sum) + r * a.ldsum;
                    if (inside(j)) o.store(sum + column(j));
                }
            }
            if constexpr (VE == 1) {
                q2.x = fmaf(v[j][0], v[j][0], q2.x);
            } else {
#pragma unroll
                for (int i = 0; i < VE; i += 2) {
                    const float2 f = make_float2(v[j][i], v[j][i + 1]);
                    q2 = fma2_rn(f, f, q2);
                }
            }
        }
        float ev = 0.0f;
        if (kEdges && sp.edge >= 0) {
            ev = ex.at(0);
            if (a.res) {
                const float f[1] = {ev + er.at(0)};
                Elems<H, 1> o;
                o.set(f);
                ev = o.at(0);
                if (a.sum && live) o.store(static_cast<H*>(a.sum) + r * a.ldsum + sp.edge);
            }
            q2.x = fmaf(ev, ev, q2.x);
        }
        fetch(r + step);  // the next row comes while this one is worked on
        const float rs = __frsqrt_rn(row_sum<ONE>(q2.x + q2.y, red[buf], warps) * inv_d + a.eps);
        if (live && sub == 0 && a.rstd) a.rstd[r] = rs;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            float g[VE];
            if constexpr (kGammaShared && VE > 1) {
#pragma unroll
                for (int i = 0; i < VE; i += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(room + (first + j * 32) * VE + i);
                    g[i] = f.x, g[i + 1] = f.y, g[i + 2] = f.z, g[i + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i) g[i] = kGammaShared ? room[(first + j * 32) * VE + i] : gam[j][i];
            }
            if constexpr (VE == 1) {
                v[j][0] = (v[j][0] * rs) * g[0];
            } else {
#pragma unroll
                for (int i = 0; i < VE; i += 2) {
                    const float2 y = mul2_rn(mul2_rn(make_float2(v[j][i], v[j][i + 1]), make_float2(rs, rs)), make_float2(g[i], g[i + 1]));
                    v[j][i] = y.x, v[j][i + 1] = y.y;
                }
            }
            if constexpr (!FP8) {
                Elems<T, VE> o;
                o.set(v[j]);
                if (live && inside(j)) o.store(static_cast<T*>(a.y) + r * a.ldy + column(j));
            }
        }
        if (kEdges && sp.edge >= 0) {
            ev = (ev * rs) * egam;
            if (!FP8 && live) static_cast<T*>(a.y)[r * a.ldy + sp.edge] = from_f32<T>(ev);
        }
        if constexpr (FP8 && (!EDGE || VE == 1)) {
            store_codes<VE, VPT, 32>(v, a.q, r, a.d, live, first, lane, wide);
        } else if constexpr (FP8) {
            store_codes_shifted<VE, VPT, ONE>(v, ev, sp, a.q, r, a.d, live, first, lane, ONE ? 0 : sub >> 5, (sub >> 5) == warps - 1, shared);
        }
    }
}

template <typename T, typename H, int VE, int VPT, int MOST, bool ONE, bool FP8, bool EDGE>
cudaError_t rms_row_go(const RmsArgs& a, cudaStream_t s) {
    auto kern = rms_row_kernel<T, H, VE, VPT, MOST, ONE, FP8, EDGE>;
    // (a row's packs are d / VE at most, its edges go beside them)
    const int packs = a.d / VE, threads = ONE ? MOST : (packs < 1 ? 1 : (packs + 32 * VPT - 1) / (32 * VPT)) * 32, rows = ONE ? MOST / 32 : 1;
    constexpr int kGammaBytes = gamma_shared(ONE, MOST, VPT * VE) ? VPT * VE * 4 : 0;  // a thread
    const cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), MOST * kGammaBytes);
    if (e != cudaSuccess) return e;
    static std::atomic<int> known[64][MOST / 32];  // asked for once per kernel, device and size of block
    std::atomic<int>& at = known[current_device() & 63][threads / 32 - 1];
    int most = at.load(std::memory_order_relaxed);
    if (most == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&most, kern, threads, threads * kGammaBytes) != cudaSuccess || most < 1) most = 1;
        most *= device_sm_count();
        at.store(most, std::memory_order_relaxed);
    }
    const int64_t want = (a.rows + rows - 1) / rows;
    int64_t grid = want < most ? want : most;
    if (EDGE && VE > 1 && grid < want) grid = grid >= VE ? grid / VE * VE : VE;  // steps of whole boundaries
    const Shift sh = shift_of(a.x, a.ldx, sizeof(T), VE);
    const bool gvec = aligned16(a.gamma) && (a.ptype == kF32 || VE == 8);
    const bool wide = FP8 && reinterpret_cast<uintptr_t>(a.q.codes) % 8 == 0 && (a.rows == 1 || a.q.ld % 8 == 0);
    return launch_early(kern, grid, threads, threads * kGammaBytes, 1, s, a, sh, gvec, wide);
}

// 16 elements a thread up to 8,192 columns and 32 above.
template <typename T, typename H, int VE, bool FP8, bool EDGE>
cudaError_t rms_width(const RmsArgs& a, cudaStream_t s) {
    constexpr int k16 = 16 / VE;
    const int d = a.d / VE * VE;  // (edges need no packs)
    if constexpr (VE == 1) {  // (more loads to a row than a warp should queue)
        if (d <= 2048) return rms_row_go<T, H, 1, 8, 256, false, FP8, true>(a, s);
        if (d <= 8192) return rms_row_go<T, H, 1, 16, 512, false, FP8, true>(a, s);
        return rms_row_go<T, H, 1, 32, 512, false, FP8, true>(a, s);
    } else {
        if (d <= 32 * VE) return rms_row_go<T, H, VE, 1, 128, true, FP8, EDGE>(a, s);
        if (d <= 512) return rms_row_go<T, H, VE, k16, 128, true, FP8, EDGE>(a, s);
        if (d <= 4096) return rms_row_go<T, H, VE, k16, 256, false, FP8, EDGE>(a, s);
        if constexpr (EDGE && sizeof(T) == 2 && (FP8 || sizeof(H) == 2)) {
            // (7508x4469 bf16: 55 us and into FP8 67, with 512 threads of 16 elements, one block of 288 an SM, 66 and 83)
            if (d <= 8192) return rms_row_go<T, H, VE, 2 * k16, 256, false, FP8, EDGE>(a, s);
        }
        if (d <= 8192) return rms_row_go<T, H, VE, k16, 512, false, FP8, EDGE>(a, s);
        return rms_row_go<T, H, VE, 2 * k16, 512, false, FP8, EDGE>(a, s);
    }
}

template <typename T, typename H, int VE, bool FP8>
cudaError_t rms_wide_go(const RmsArgs& a, cudaStream_t s) {
    const int64_t most = 2ll * device_sm_count();
    const bool wide = FP8 && reinterpret_cast<uintptr_t>(a.q.codes) % 8 == 0 && (a.rows == 1 || a.q.ld % 8 == 0);
    return launch_early(rms_wide_kernel<T, H, VE, FP8>, a.rows < most ? a.rows : most, kWideThreads, 0, 1, s, a, shift_of(a.x, a.ldx, sizeof(T), VE),
                        wide);
}

template <typename T, typename H, bool FP8>
cudaError_t rms_form(const RmsArgs& a, cudaStream_t s) {
    constexpr int VE = 16 / sizeof(T);
    const Shift sx = shift_of(a.x, a.ldx, sizeof(T), VE);
    const auto like = [&](const void* p, int64_t ld, int64_t el) { return !p || same_shift(sx, shift_of(p, ld, el, VE), a.rows); };
    const bool alike = like(a.res, a.ldres, sizeof(H)) && like(a.sum, a.ldsum, sizeof(H)) && (FP8 || like(a.y, a.ldy, sizeof(T)));
    if (alike && a.d > 16384) return rms_wide_go<T, H, VE, FP8>(a, s);
    if (a.d <= 16384) {
        if (alike) {
            if (sx.base == 0 && (a.rows == 1 || sx.step == 0) && a.d % VE == 0) return rms_width<T, H, VE, FP8, false>(a, s);
            return rms_width<T, H, VE, FP8, true>(a, s);
        }
    }
    if (a.d <= 16384) return rms_width<T, H, 1, FP8, true>(a, s);
    return rms_wide_go<T, H, 1, FP8>(a, s);
}
template <typename T, typename H>
cudaError_t rms_t(const RmsArgs& a, cudaStream_t s) {
    return a.y ? rms_form<T, H, false>(a, s) : rms_form<T, H, true>(a, s);
}

}  // namespace

cudaError_t rms_norm_launch(const RmsArgs& a, int xtype, int htype, cudaStream_t s) {
    if (xtype == kF32) return rms_t<float, float>(a, s);
    if (xtype == kBF16) return htype == kF32 ? rms_t<__nv_bfloat16, float>(a, s) : rms_t<__nv_bfloat16, __nv_bfloat16>(a, s);
    return htype == kF32 ? rms_t<__half, float>(a, s) : rms_t<__half, __half>(a, s);
}

}  // namespace nfx
