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

namespace nfx {
namespace {

// One warp per group of 128, any alignment and stride.
template <typename T>
__global__ void __launch_bounds__(256) quant_rows_kernel(QuantArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t blocks = (a.cols + kGroup - 1) / kGroup;
    for (int64_t w = blockIdx.x * 8ll + (threadIdx.x >> 5); w < a.rows * blocks; w += gridDim.x * 8ll) {
        const int64_t r = w / blocks, b = w % blocks;
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        float v[4], am = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = b * kGroup + j * 32 + lane;
            v[j] = i < a.cols ? to_f32(x[i]) : 0.0f;
            am = fmaxf(am, finite_abs(v[j]));
        }
        const float sc = group_scale(warp_max(am)), inv = __frcp_rn(sc);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = b * kGroup + j * 32 + lane;
            if (i < a.cols) a.q.codes[r * a.q.ld + i] = static_cast<uint8_t>(e4m3_code(v[j], inv));
        }
        if (lane == 0) a.q.scales[r * a.q.srs + b * a.q.sbs] = sc;
    }
}

// One block per 128 x 128 tile, staged in shared memory as fp32.
constexpr int kPitch = kGroup + 1;
constexpr int kTileSmem = (kGroup * kPitch + 2 * kGroup) * 4;

template <typename T>
__global__ void __launch_bounds__(256) quant_tile_kernel(QuantArgs a) {
    extern __shared__ float sm[];
    float* tile = sm;
    float* rmax = sm + kGroup * kPitch;
    float* cmax = rmax + kGroup;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t cblocks = (a.cols + kGroup - 1) / kGroup;
    const int64_t br = blockIdx.x / cblocks, bc = blockIdx.x % cblocks;
    const int64_t r0 = br * kGroup, c0 = bc * kGroup;
    for (int i = warp; i < kGroup; i += 8) {
        const int64_t r = r0 + i;
        float am = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t c = c0 + j * 32 + lane;
            const float v = r < a.rows && c < a.cols ? to_f32(static_cast<const T*>(a.x)[r * a.ldx + c]) : 0.0f;
            tile[i * kPitch + j * 32 + lane] = v;
            am = fmaxf(am, finite_abs(v));
        }
        am = warp_max(am);
        if (lane == 0) rmax[i] = am;
    }
    __syncthreads();
    if (threadIdx.x < kGroup && !a.tile) {
        const int c = threadIdx.x;
        float am = 0.0f, s = 0.0f;
        for (int i = 0; i < kGroup; ++i) {
            const float v = tile[i * kPitch + c];
            am = fmaxf(am, finite_abs(v));
            s += v;
        }
        cmax[c] = am;
        if (a.part && c0 + c < a.cols) a.part[br * a.cols + c0 + c] = s;
    }
    if (a.tile && warp == 0) {
        float am = 0.0f;
        for (int j = 0; j < 4; ++j) am = fmaxf(am, rmax[j * 32 + lane]);
        am = warp_max(am);
        __syncwarp();
        for (int j = 0; j < 4; ++j) rmax[j * 32 + lane] = cmax[j * 32 + lane] = am;
    }
    __syncthreads();
    for (int i = warp; i < kGroup; i += 8) {
        const int64_t r = r0 + i;
        if (r < a.rows) {
            const float sc = group_scale(rmax[i]), inv = __frcp_rn(sc);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t c = c0 + j * 32 + lane;
                if (c < a.cols)
                    a.q.codes[r * a.q.ld + c] = static_cast<uint8_t>(e4m3_code(tile[i * kPitch + j * 32 + lane], inv));
            }
            if (lane == 0 && (!a.tile || i == 0)) a.q.scales[(a.tile ? br : r) * a.q.srs + bc * a.q.sbs] = sc;
        }
        const int64_t c = c0 + i;  // row i of the transposed tile
        if (a.qt.codes && c < a.cols) {
            const float sc = group_scale(cmax[i]), inv = __frcp_rn(sc);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t rr = r0 + j * 32 + lane;
                if (rr < a.rows)
                    a.qt.codes[c * a.qt.ld + rr] =
                        static_cast<uint8_t>(e4m3_code(tile[(j * 32 + lane) * kPitch + i], inv));
            }
            if (lane == 0 && (!a.tile || i == 0)) a.qt.scales[(a.tile ? bc : c) * a.qt.srs + br * a.qt.sbs] = sc;
        }
    }
}

template <typename T>
cudaError_t quant_t(const QuantArgs& a, cudaStream_t s) {
    const int64_t cblocks = (a.cols + kGroup - 1) / kGroup;
    if (!a.tile && !a.qt.codes && !a.part) {
        const int64_t want = (a.rows * cblocks + 7) / 8, cap = 16ll * device_sm_count();
        quant_rows_kernel<T><<<static_cast<int>(want < cap ? want : cap), 256, 0, s>>>(a);
        return cudaGetLastError();
    }
    auto kern = quant_tile_kernel<T>;
    cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kTileSmem);
    if (e != cudaSuccess) return e;
    const int64_t tiles = (a.rows + kGroup - 1) / kGroup * cblocks;
    kern<<<static_cast<unsigned>(tiles), 256, kTileSmem, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t fp8_quantise_launch(const QuantArgs& a, int xtype, cudaStream_t s) {
    if (xtype == kF32) return quant_t<float>(a, s);
    if (xtype == kBF16) return quant_t<__nv_bfloat16>(a, s);
    return quant_t<__half>(a, s);
}

}  // namespace nfx
