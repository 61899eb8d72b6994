// fp8_quant.cu -- the FP8 E4M3 block quantiser: codes with one fp32 scale per group of 128
// elements along a row, or per 128 x 128 tile; optionally also the transposed codes (whose
// groups run along the rows of the input) and the column sums, from one read of the input.
//
//   s = max(fl(max |x| / 448), 2^-126),  code = E4M3(fl(x * fl(1 / s)))
//
// with the library's E4M3 encoder.  The maximum is over the group's finite elements.
#include "block_ops.h"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "row_pack.cuh"

namespace nfx {
namespace {

// Groups along rows only: rows in registers, TPR threads by VPT packs of VE elements; rows longer than
// that in chunks.  One read, one write, a few shuffles a group.
template <typename T, int VE, int VPT, int TPR>
__global__ void __launch_bounds__(128) quant_rows_kernel(QuantArgs a, int64_t chunks, bool wide) {
    constexpr int kRows = 128 / TPR;
    const int lane = threadIdx.x & 31;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
    const int64_t r = chunks == 1 ? unit : unit / chunks;
    const int64_t first = (chunks == 1 ? 0 : unit % chunks) * (VPT * 32) + (TPR < 32 ? threadIdx.x % TPR : lane);
    const bool live = r < a.rows;
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    float v[VPT][VE];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int64_t c = (first + j * 32) * VE;
#pragma unroll
        for (int i = 0; i < VE; ++i) v[j][i] = 0.0f;
        if (live && c < a.cols) load_pack<T, VE>(x + c, v[j]);
    }
    store_codes<VE, VPT, TPR>(v, a.q, r, a.cols, live, first, lane, wide);
}

// One block per 128 x 128 tile.  A thread holds 8 rows x 8 columns in registers: lane % 16 counts the
// columns' eights, 2 * warp + lane / 16 the rows'.  A row's maximum is 8 values and four shuffles, a
// column's 8 values, a shuffle and eight partial results in shared memory.  The transposed codes go
// through shared memory (16 KB, 8-byte slots XOR-ed with the column's eight, so that neither side has
// more conflicts than its width) and leave as 128-byte rows.  The tile is read once from HBM and its
// bytes are the bound; `VEC`: rows of x start on 16-byte boundaries.
constexpr int kTileThreads = 256;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kTileThreads, 2) quant_tile_kernel(QuantArgs a, bool wide, bool wide_t) {
    __shared__ __align__(16) uint8_t tileT[kGroup * kGroup];
    __shared__ float cmax[8][kGroup], csum[8][kGroup], rscale[kGroup], cinv[kGroup];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cc = lane & 15, rr = warp * 2 + (lane >> 4);  // this thread's eights
    const int64_t cblocks = (a.cols + kGroup - 1) / kGroup;
    const int64_t br = blockIdx.x / cblocks, bc = blockIdx.x % cblocks;
    const int64_t r0 = br * kGroup + rr * 8, c0 = bc * kGroup + cc * 8;
    constexpr int VE = 16 / sizeof(T);
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const T* x = static_cast<const T*>(a.x) + (r0 + i) * a.ldx + c0;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = 0.0f;
        if (r0 + i >= a.rows) continue;
        if (VEC && c0 + 8 <= a.cols) {
#pragma unroll
            for (int k = 0; k < 8; k += VE) {
                float o[VE];
                load_pack<T, VE>(x + k, o);
#pragma unroll
                for (int e = 0; e < VE; ++e) v[i][k + e] = o[e];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c0 + k < a.cols) v[i][k] = to_f32(x[k]);
        }
    }
    // largest magnitudes and sums; `finite` is the second look, when a maximum is infinite
    float rm[8], cm[8];
    auto maxima = [&](bool finite) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rm[i] = cm[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float m = finite ? finite_abs(v[i][k]) : fabsf(v[i][k]);
                rm[i] = fmaxf(rm[i], m);
                cm[k] = fmaxf(cm[k], m);
            }
    };
    maxima(false);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, rm[i]);
    if (!(top <= 3.402823466e38f)) maxima(true);
    if (a.tile) {
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, rm[i]);
        top = warp_max(top);
        if (lane == 0) cmax[warp][0] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) top = fmaxf(top, cmax[w][0]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) rm[i] = fmaxf(rm[i], __shfl_xor_sync(0xFFFFFFFFu, rm[i], o));
        if (a.qt.codes || a.part) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += v[i][k];
                s += __shfl_xor_sync(0xFFFFFFFFu, s, 16);
                cm[k] = fmaxf(cm[k], __shfl_xor_sync(0xFFFFFFFFu, cm[k], 16));
                if (lane < 16) {
                    cmax[warp][cc * 8 + k] = cm[k];
                    csum[warp][cc * 8 + k] = s;
                }
            }
        }
    }
    // codes along the rows
    const float tscale = group_scale(top), tinv = __frcp_rn(tscale);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float sc = a.tile ? tscale : group_scale(rm[i]), inv = a.tile ? tinv : __frcp_rn(sc);
        if (!a.tile && cc == 0) rscale[rr * 8 + i] = sc;
        const uint32_t w0 = e4m3_encode4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        const uint32_t w1 = e4m3_encode4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
        if (r0 + i >= a.rows || c0 >= a.cols) continue;
        uint8_t* dst = a.q.codes + (r0 + i) * a.q.ld + c0;
        if (wide && c0 + 8 <= a.cols) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c0 + k < a.cols) dst[k] = static_cast<uint8_t>((k < 4 ? w0 : w1) >> (8 * (k & 3)));
        }
    }
    if (a.tile && threadIdx.x == 0) {
        a.q.scales[br * a.q.srs + bc * a.q.sbs] = tscale;
        if (a.qt.codes) a.qt.scales[bc * a.qt.srs + br * a.qt.sbs] = tscale;
    }
    __syncthreads();
    if (!a.tile && threadIdx.x < kGroup) {
        const int t = threadIdx.x;
        if (br * kGroup + t < a.rows) a.q.scales[(br * kGroup + t) * a.q.srs + bc * a.q.sbs] = rscale[t];
        if (a.qt.codes || a.part) {
            float m = 0.0f, s = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                m = fmaxf(m, cmax[w][t]);
                s += csum[w][t];
            }
            const float sc = group_scale(m);
            cinv[t] = __frcp_rn(sc);
            if (bc * kGroup + t < a.cols) {
                if (a.part) a.part[br * a.cols + bc * kGroup + t] = s;
                if (a.qt.codes) a.qt.scales[(bc * kGroup + t) * a.qt.srs + br * a.qt.sbs] = sc;
            }
        }
    }
    if (!a.qt.codes) return;
    if (!a.tile) __syncthreads();
    // codes along the columns
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float inv = a.tile ? tinv : cinv[cc * 8 + k];
        const uint32_t w0 = e4m3_encode4(v[0][k] * inv, v[1][k] * inv, v[2][k] * inv, v[3][k] * inv);
        const uint32_t w1 = e4m3_encode4(v[4][k] * inv, v[5][k] * inv, v[6][k] * inv, v[7][k] * inv);
        *reinterpret_cast<uint2*>(tileT + (cc * 8 + k) * kGroup + (rr ^ cc) * 8) = make_uint2(w0, w1);
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kGroup * 8 / kTileThreads; ++n) {
        const int t = n * kTileThreads + threadIdx.x, col = t >> 3, half = t & 7;  // 16 rows of one column
        const int e = col >> 3;
        uint4 w = *reinterpret_cast<const uint4*>(tileT + col * kGroup + ((2 * half) ^ (e & 14)) * 8);
        if (e & 1) w = make_uint4(w.z, w.w, w.x, w.y);
        const int64_t c = bc * kGroup + col, r = br * kGroup + half * 16;
        if (c >= a.cols || r >= a.rows) continue;
        uint8_t* dst = a.qt.codes + c * a.qt.ld + r;
        if (wide_t && r + 16 <= a.rows) {
            *reinterpret_cast<uint4*>(dst) = w;
        } else {
            const uint32_t b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (r + k < a.rows) dst[k] = static_cast<uint8_t>(b[k >> 2] >> (8 * (k & 3)));
        }
    }
}

bool code_rows(const Fp8Out& q, int64_t rows, int64_t bytes) {
    return reinterpret_cast<uintptr_t>(q.codes) % bytes == 0 && (rows == 1 || q.ld % bytes == 0);
}

template <typename T, int VE, int VPT, int TPR>
cudaError_t quant_rows(const QuantArgs& a, cudaStream_t s) {
    constexpr int kRows = 128 / TPR;
    const int64_t chunks = TPR < 32 ? 1 : (a.cols + 32 * VE * VPT - 1) / (32 * VE * VPT);
    const int64_t grid = (a.rows * chunks + kRows - 1) / kRows;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
    quant_rows_kernel<T, VE, VPT, TPR><<<static_cast<unsigned>(grid), 128, 0, s>>>(a, chunks, code_rows(a.q, a.rows, 8));
    return cudaGetLastError();
}

template <typename T>
cudaError_t quant_t(const QuantArgs& a, cudaStream_t s) {
    constexpr int VE = 16 / sizeof(T);
    const bool rows16 = aligned16(a.x) && (a.rows == 1 || a.ldx % VE == 0);
    if (!a.tile && !a.qt.codes && !a.part) {
        if (!rows16 || a.cols % VE) return quant_rows<T, 1, 8, 32>(a, s);
        if (a.cols <= 16 * VE) return quant_rows<T, VE, 1, 16>(a, s);
        if (a.cols <= 32 * VE) return quant_rows<T, VE, 1, 32>(a, s);
        return quant_rows<T, VE, 2, 32>(a, s);
    }
    const int64_t tiles = (a.rows + kGroup - 1) / kGroup * ((a.cols + kGroup - 1) / kGroup);
    const bool wide = code_rows(a.q, a.rows, 8), wide_t = code_rows(a.qt, a.cols, 16);
    if (rows16) quant_tile_kernel<T, true><<<static_cast<unsigned>(tiles), kTileThreads, 0, s>>>(a, wide, wide_t);
    else quant_tile_kernel<T, false><<<static_cast<unsigned>(tiles), kTileThreads, 0, s>>>(a, wide, wide_t);
    return cudaGetLastError();
}

}  // namespace

cudaError_t fp8_quantise_launch(const QuantArgs& a, int xtype, cudaStream_t s) {
    if (xtype == kF32) return quant_t<float>(a, s);
    if (xtype == kBF16) return quant_t<__nv_bfloat16>(a, s);
    return quant_t<__half>(a, s);
}

}  // namespace nfx
