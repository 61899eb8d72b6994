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
#include "sm100.cuh"

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

// 128 x 128 tiles, one at a time per block.  A thread holds 8 rows x 8 columns in registers: lane % 16
// counts the columns' eights, 2 * warp + lane / 16 the rows'.  A row's maximum is 8 values and four
// shuffles, a column's 8 values, a shuffle and eight partial results in shared memory; scales and
// reciprocals are made by one thread per row and per column.  The transposed codes go through shared memory
// (16 KB, 8-byte slots XOR-ed with the column's eight, so that neither side has more conflicts than its
// width) and leave as 128-byte rows.  The bytes' latency is the bound, at the quarter of an SM's warps that
// the registers leave; what keeps them coming for 16-bit types (kAhead) is that the blocks walk over the
// tiles and a thread copies its part of the next one into shared memory (cp.async, its own slots, so no
// barrier) while it works on this one: 16384x4096 bf16 both ways with sums 74 us (85, against 147 with a
// block per tile, while each code was still corrected in the main path).  An fp32 tile is twice the bytes
// for the same work, and there a block per tile is faster (131072x128 to tiles: 17 us, 28 walking).  `VEC`:
// rows of x start on 16-byte boundaries.
constexpr int kTileThreads = 256;

template <typename T, bool VEC>
constexpr bool kAhead = VEC && sizeof(T) == 2;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kTileThreads, 2) quant_tile_kernel(QuantArgs a, int tiles, int cblocks, bool wide,
                                                                     bool wide_t) {
    extern __shared__ __align__(16) uint8_t next[];  // the next tile: slot n of thread t at (n * 256 + t) * 16
    __shared__ __align__(16) uint8_t tileT[kGroup * kGroup];
    __shared__ __align__(16) float cmax[8][kGroup], csum[8][kGroup], rmax[kGroup], rinv[kGroup], cinv[kGroup];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cc = lane & 15, rr = warp * 2 + (lane >> 4);  // this thread's eights
    constexpr int VE = 16 / sizeof(T), kPacks = 8 / VE;
    const bool cols_too = a.qt.codes || a.part;
    constexpr bool kWalk = kAhead<T, VEC>;

    auto ahead = [&](int t) {
        const int64_t r0 = static_cast<int64_t>(t / cblocks) * kGroup + rr * 8, c0 = static_cast<int64_t>(t % cblocks) * kGroup + cc * 8;
        const T* x = static_cast<const T*>(a.x) + r0 * a.ldx + c0;
        uint8_t* slot = next + threadIdx.x * 16;
        if (r0 + 8 <= a.rows && c0 + 8 <= a.cols) {
#pragma unroll
            for (int i = 0; i < 8; ++i, x += a.ldx)
#pragma unroll
                for (int k = 0; k < kPacks; ++k) cp_async16(slot + (i * kPacks + k) * kTileThreads * 16, x + k * VE, 16);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < kPacks; ++k) {
                const int64_t left = r0 + i < a.rows ? a.cols - c0 - k * VE : 0;
                const int n = left >= VE ? 16 : (left > 0 ? static_cast<int>(left * sizeof(T)) : 0);
                cp_async16(slot + (i * kPacks + k) * kTileThreads * 16, n ? x + i * a.ldx + k * VE : a.x, n);
            }
    };
    if (kWalk) ahead(blockIdx.x);

    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t br = tile / cblocks, bc = tile % cblocks;
        const int64_t r0 = br * kGroup + rr * 8, c0 = bc * kGroup + cc * 8;
        float v[8][8];
        if constexpr (kWalk) {
            cp_async_wait_all();
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int k = 0; k < kPacks; ++k) {
                    const Pack<T, VE> p =
                        *reinterpret_cast<const Pack<T, VE>*>(next + ((i * kPacks + k) * kTileThreads + threadIdx.x) * 16);
#pragma unroll
                    for (int e = 0; e < VE; ++e) v[i][k * VE + e] = to_f32(p.v[e]);
                }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const T* x = static_cast<const T*>(a.x) + (r0 + i) * a.ldx + c0;
                if (VEC && r0 + i < a.rows && c0 + 8 <= a.cols) {
#pragma unroll
                    for (int k = 0; k < kPacks; ++k) {
                        float o[VE];
                        load_pack<T, VE>(x + k * VE, o);
#pragma unroll
                        for (int e = 0; e < VE; ++e) v[i][k * VE + e] = o[e];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[i][k] = r0 + i < a.rows && c0 + k < a.cols ? to_f32(x[k]) : 0.0f;
                }
            }
        }
        // largest magnitudes; `finite` is the second look, when a maximum is infinite
        float rm[8], cm[8], top = 0.0f;
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
            top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, rm[i]);
        };
        maxima(false);
        if (!(top <= 3.402823466e38f)) maxima(true);
        if (a.tile) {
            top = warp_max(top);
            if (lane == 0) rmax[warp] = top;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) rm[i] = fmaxf(rm[i], __shfl_xor_sync(0xFFFFFFFFu, rm[i], o));
                if (cc == i) rmax[rr * 8 + i] = rm[i];
            }
            if (cols_too) {
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
        __syncthreads();
        // this tile's values are in registers: the slots are free for the next one
        if (kWalk && tile + gridDim.x < tiles) ahead(tile + gridDim.x);
        float tinv = 0.0f;
        if (a.tile) {
#pragma unroll
            for (int w = 0; w < 8; ++w) top = fmaxf(top, rmax[w]);
            const float sc = group_scale(top);
            tinv = __frcp_rn(sc);
            if (threadIdx.x == 0) {
                a.q.scales[br * a.q.srs + bc * a.q.sbs] = sc;
                if (a.qt.codes) a.qt.scales[bc * a.qt.srs + br * a.qt.sbs] = sc;
            }
        } else if (threadIdx.x < kGroup) {
            const int t = threadIdx.x;
            const float sc = group_scale(rmax[t]);
            rinv[t] = __frcp_rn(sc);
            if (br * kGroup + t < a.rows) a.q.scales[(br * kGroup + t) * a.q.srs + bc * a.q.sbs] = sc;
        } else if (cols_too) {
            const int t = threadIdx.x - kGroup;
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
        __syncthreads();
        // codes along the rows
        const bool inside = wide && c0 + 8 <= a.cols && r0 + 8 <= a.rows;
        uint8_t* row = a.q.codes + r0 * a.q.ld + c0;
        uint32_t odd = 0;
        auto along_rows = [&](auto mend) {
            constexpr bool kMend = decltype(mend)::value;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float inv = a.tile ? tinv : rinv[rr * 8 + i];
                const uint32_t w0 = scaled_codes<kMend>(v[i][0], v[i][1], v[i][2], v[i][3], inv, odd);
                const uint32_t w1 = scaled_codes<kMend>(v[i][4], v[i][5], v[i][6], v[i][7], inv, odd);
                if (inside) {
                    *reinterpret_cast<uint2*>(row + i * a.q.ld) = make_uint2(w0, w1);
                } else if (r0 + i < a.rows) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (c0 + k < a.cols) row[i * a.q.ld + k] = static_cast<uint8_t>((k < 4 ? w0 : w1) >> (8 * (k & 3)));
                }
            }
        };
        along_rows(std::false_type{});
        if (odd) along_rows(std::true_type{});  // (rare; the same bytes again, put right)
        if (!a.qt.codes) continue;
        // codes along the columns
        odd = 0;
        auto along_columns = [&](auto mend) {
            constexpr bool kMend = decltype(mend)::value;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float inv = a.tile ? tinv : cinv[cc * 8 + k];
                const uint32_t w0 = scaled_codes<kMend>(v[0][k], v[1][k], v[2][k], v[3][k], inv, odd);
                const uint32_t w1 = scaled_codes<kMend>(v[4][k], v[5][k], v[6][k], v[7][k], inv, odd);
                *reinterpret_cast<uint2*>(tileT + (cc * 8 + k) * kGroup + (rr ^ cc) * 8) = make_uint2(w0, w1);
            }
        };
        along_columns(std::false_type{});
        if (odd) along_columns(std::true_type{});
        __syncthreads();
#pragma unroll
        for (int n = 0; n < kGroup * 8 / kTileThreads; ++n) {
            const int t = n * kTileThreads + threadIdx.x, col = t >> 3, part = t & 7;  // 16 rows of one column
            const int e = col >> 3;
            uint4 w = *reinterpret_cast<const uint4*>(tileT + col * kGroup + ((2 * part) ^ (e & 14)) * 8);
            if (e & 1) w = make_uint4(w.z, w.w, w.x, w.y);
            const int64_t c = bc * kGroup + col, r = br * kGroup + part * 16;
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
        // (the next tile's maxima are written before its first barrier, its transposed codes after it)
    }
}

template <typename T, bool VEC>
cudaError_t quant_tile(const QuantArgs& a, bool wide, bool wide_t, cudaStream_t s) {
    const int64_t cblocks = (a.cols + kGroup - 1) / kGroup, tiles = (a.rows + kGroup - 1) / kGroup * cblocks;
    auto kern = quant_tile_kernel<T, VEC>;
    const int smem = kAhead<T, VEC> ? kGroup * kGroup * static_cast<int>(sizeof(T)) : 0;
    cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
    if (e != cudaSuccess) return e;
    const int64_t cap = kAhead<T, VEC> ? 2ll * device_sm_count() : tiles;
    kern<<<static_cast<unsigned>(tiles < cap ? tiles : cap), kTileThreads, smem, s>>>(
        a, static_cast<int>(tiles), static_cast<int>(cblocks), wide, wide_t);
    return cudaGetLastError();
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
        if (!rows16 || a.cols % VE)
            return aligned_rows(a.x, a.rows, a.ldx, sizeof(T), 2 * sizeof(T)) && a.cols % 2 == 0 ? quant_rows<T, 2, 4, 32>(a, s)
                                                                                             : quant_rows<T, 1, 8, 32>(a, s);
        if (a.cols <= 16 * VE) return quant_rows<T, VE, 1, 16>(a, s);
        if (a.cols <= 32 * VE) return quant_rows<T, VE, 1, 32>(a, s);
        return quant_rows<T, VE, 2, 32>(a, s);
    }
    const bool wide = code_rows(a.q, a.rows, 8), wide_t = code_rows(a.qt, a.cols, 16);
    return rows16 ? quant_tile<T, true>(a, wide, wide_t, s) : quant_tile<T, false>(a, wide, wide_t, s);
}

}  // namespace

cudaError_t fp8_quantise_launch(const QuantArgs& a, int xtype, cudaStream_t s) {
    if (xtype == kF32) return quant_t<float>(a, s);
    if (xtype == kBF16) return quant_t<__nv_bfloat16>(a, s);
    return quant_t<__half>(a, s);
}

}  // namespace nfx
