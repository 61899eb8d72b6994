// fp8_gemm.cu -- product of two FP8 E4M3 matrices with an fp32 scale for each block of 128
// along K, on tcgen05 (kind::f8f6f4).
//
//   C[m, n] = act( sum_b sa[m, b] sb[n, b] ( sum_{k in block b} A[m, k] B[n, k] ) + bias[n] )
//
// sa and sb are per row, or per 128 rows (tiles).  The tensor core sums one block of 128 (four
// K = 32 instructions) into a TMEM stage; the epilogue warps read that stage, multiply it by
// the block's scales and add it to fp32 accumulators in registers, so the sum over the blocks is
// fp32 and no product of scales is rounded to fewer bits.
//
// Two kernels: pairs of CTAs on 256 x 256 tiles for large results, and a narrow one, with K split
// over a cluster, for few rows of A or few tiles; fp8_gemm_plan() below chooses.  Both are
// warp-specialised: a TMA producer, an MMA issuer, a scale producer, and the promoting warps.
//
// Measured (one B200; HBM 6,457 GB/s, FP8 taken as twice the measured bf16 rate, 3,276 TFLOP/s; graphs of
// launches over operands that do not fit L2 together, a few milliseconds long):
//   8192x16384x4096 to bf16   481 us, 2,290 TFLOP/s; 535 us with bias and GELU.  In a loop of seconds the
//                             1,000 W power cap sets the clock: 572 us at 1.43 GHz, 636 us with bias and
//                             GELU at 1.53 GHz.  A block of K takes 745 cycles where its MMAs take 512
//                             (without the sums 670, without TMEM reads too 650: barrier hand-over); the
//                             rest is the tiles' epilogues, of which MMAs of two blocks overlap
//                             (2304x2048x512, one tile a pair: 8.0 us, 11.1 with bias and GELU)
//   4096x4096x8192 to fp32    196 us with column scales.  A block of K takes 0.68 us (2304x2048), 0.45 with
//                             tile scales: four TMEM reads, each waited for, and a second multiply
//   1x4096x4096               8.5 us, 5.9 with the weights in L2, of which 4.5 are the start and the join
//                             (1x1024x1024 takes that)
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "block_ops.h"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

constexpr int kBK = kGroup;
constexpr int kOutBytes = 32 * 128;  // one staging buffer

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
template <int R>
__device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

// Adds the bias (2 NP floats in shared memory) to one row's accumulators and applies the activation.
template <int NP>
__device__ __forceinline__ void finish_row(float2 (&acc)[NP], const float* bias, int act) {
    if (bias) {
#pragma unroll
        for (int j = 0; j < NP / 2; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(bias + 4 * j);
            acc[2 * j].x += v.x, acc[2 * j].y += v.y;
            acc[2 * j + 1].x += v.z, acc[2 * j + 1].y += v.w;
        }
    }
    if (act == 1) {
#pragma unroll
        for (int j = 0; j < NP; ++j) acc[j] = gelu_sig2(acc[j]);
    } else if (act == 2) {
#pragma unroll
        for (int j = 0; j < NP; ++j) acc[j] = make_float2(relu_ref(acc[j].x), relu_ref(acc[j].y));
    }
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

// A warp's 32 rows x 2 NP columns at (m0, n0) to C through its staging buffer `buf`, in boxes of 32
// rows x 128 bytes (the lane holds row m0 + lane).
template <int CT, int NP>
__device__ __forceinline__ void store_rows(const float2 (&acc)[NP], const Fp8GemmArgs& p, const CUtensorMap* tmC,
                                           uint8_t* buf, int m0, int n0, int lane) {
    constexpr int kEl = CT == kF32 ? 4 : 2;
    constexpr int kCols = 128 / kEl;  // columns of a box
#pragma unroll
    for (int b = 0; b < 2 * NP / kCols; ++b) {
        const int n = n0 + b * kCols;
        if (n >= p.N) break;
        if (p.tma_c) {  // the previous box has been read
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(buf + swz_offset(lane * 128 + j * 16, 128)) = pack_chunk<CT, NP>(acc, b * 8 + j);
        // a TMA store clips its box at 16 bytes, not at the element: a last box whose row ends inside 16
        // bytes goes out by elements
        if (p.tma_c && (n + kCols <= p.N || p.N * kEl % 16 == 0)) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                tma_store_2d(tmC, buf, n, m0);
                tma_store_commit();
            }
        } else {
            __syncwarp();
            const int rows = min(32, p.M - m0), cols = min(kCols, p.N - n);
            for (int r = 0; r < rows; ++r) {
                uint8_t* dst = static_cast<uint8_t*>(p.C) + (static_cast<int64_t>(m0 + r) * p.ldc + n) * kEl;
                for (int c = lane; c < cols; c += 32) {
                    const uint8_t* src = buf + swz_offset(r * 128 + c * kEl, 128);
                    if constexpr (kEl == 4) *reinterpret_cast<uint32_t*>(dst + c * 4) = *reinterpret_cast<const uint32_t*>(src);
                    else *reinterpret_cast<uint16_t*>(dst + c * 2) = *reinterpret_cast<const uint16_t*>(src);
                }
            }
            __syncwarp();
        }
    }
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

// A warp's finished accumulators (rows m0 + lane, columns n0 ..) to C, through its staging buffer.
template <int CT, int NP>
__device__ __forceinline__ void epilogue(float2 (&acc)[NP], const Fp8GemmArgs& p, const CUtensorMap* tmC,
                                         uint8_t* buf, int m0, int n0, int lane) {
    float* sb = reinterpret_cast<float*>(buf);
    if (p.bias) {
        float b[NP / 16];
#pragma unroll
        for (int j = 0; j < NP / 16; ++j) {
            const int n = n0 + j * 32 + lane;
            b[j] = n < p.N ? load_any(p.bias, p.btype, n) : 0.0f;
        }
        if (p.tma_c && lane == 0) tma_store_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NP / 16; ++j) sb[j * 32 + lane] = b[j];
        __syncwarp();
    }
    finish_row<NP>(acc, p.bias ? sb : nullptr, p.act);
    __syncwarp();  // every lane has read the bias
    if (m0 < p.M) store_rows<CT, NP>(acc, p, tmC, buf, m0, n0, lane);
}

// COL: 0 the columns of a 128-column group share a scale (B in tiles), 1 one scale per column
//
// One tile is 256 x 256, computed by a pair of CTAs with cta_group::2 MMAs: CTA r holds rows
// 128 r .. of the tile's A and half the rows of its B (so each operand byte is fetched once per pair,
// 64 KB for 128 x 256 x 256 products instead of 96 KB by two CTAs alone), and rows 128 r .. of the
// result in its TMEM.  The tile's two column halves are separate MMAs (N = 128) with two TMEM stages
// each, so a half's accumulators are handed over after 256 cycles and not after 512: the time from
// an MMA's end to the reuse of its stage (barriers, TMEM reads) is what has to be covered.
// Warps of each CTA:
//   0-15   promotion and epilogue, 32 rows x 64 columns each    16  TMA producer
//   17     TMEM owner; CTA 0's issues the MMAs
//   18     scale producer (cp.async into a ring, several blocks ahead: a scale that is fetched in
//          the promotion loop itself costs an L2 latency per block)
// Sixteen promoting warps and not eight: a warp's loop is a chain of barrier, TMEM read and sums, and
// four of them on a scheduler cover each other's latencies.  Their registers (64 accumulators, 32 on the
// way from TMEM) are given up by the other four warps: 16 x 32 x 112 + 4 x 32 x 32 = 20 x 32 x 96.
// Barriers: full (CTA 0's, both CTAs' bytes), empty and accFull (both CTAs', by commit), accEmpty (CTA
// 0's, arrivals from the epilogue warps of both), sFull and sEmpty (each CTA's own scales).
constexpr int kPairThreads = 640;
constexpr int kPairEpi = 16;

template <int COL>
struct PairCfg {
    static constexpr int kStages = 4;
    // columns of one TMEM read: 8192 x 16384 x 4096 took 525 us with 32 and 583 with 16 where the
    // columns share a scale, 798 and 713 where the column scales take registers too
    static constexpr int kRead = COL ? 16 : 32;
    static constexpr int kStageBytes = 2 * 128 * kBK;
    static constexpr int kScaleStages = 8;
    static constexpr int kScaleBytes = (128 + (COL ? 256 : 4)) * 4;
    static constexpr int kOffOut = kStages * kStageBytes;
    static constexpr int kOffScale = kOffOut + kPairEpi * kOutBytes;
    static constexpr int kOffBars = kOffScale + kScaleStages * kScaleBytes;
    static constexpr int kSmemBytes = kOffBars + 8 * (2 * kStages + 2 * 4 + 2 * kScaleStages) + 16 + 64 + 1024;
    static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

template <int COL, int CT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmC, const Fp8GemmArgs p) {
    using C = PairCfg<COL>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
    uint64_t* empty = full + C::kStages;
    uint64_t* accFull = empty + C::kStages;
    uint64_t* accEmpty = accFull + 4;
    uint64_t* sFull = accEmpty + 4;
    uint64_t* sEmpty = sFull + C::kScaleStages;
    uint32_t* sTmem = reinterpret_cast<uint32_t*>(sEmpty + C::kScaleStages);
    volatile int* sAbort = reinterpret_cast<volatile int*>(sTmem + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);  // (known to be the same in all lanes)
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int tm = (p.M + 255) / 256, tn = (p.N + 255) / 256;
    const int tiles = tm * tn;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int KB = (p.K + kBK - 1) / kBK;
    const uint64_t budget = p.wait_ns ? p.wait_ns : kWaitNs;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 4; ++s) {  // stage * 2 + column half
            mbar_init(&accFull[s], 1);
            mbar_init(&accEmpty[s], kPairEpi);
        }
        for (int s = 0; s < C::kScaleStages; ++s) {
            mbar_init(&sFull[s], 32);
            mbar_init(&sEmpty[s], kPairEpi);
        }
        *sAbort = 0;
        fence_mbar_init();
    }
    if (warp == kPairEpi + 1) tmem_alloc_pair(sTmem, 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are ready
    tc_fence_after();
    const uint32_t tmem_base = *sTmem;

    // the register split stands inside the roles' branches: where they met again, the compiler would
    // have to assume the smaller count
    if (warp >= kPairEpi) {
        reg_dec<32>();
        if (warp == kPairEpi) {
            // ---------------- TMA producer
            if (elect_one()) {
                int it = 0;
                bool ok = true;
                for (int t = first; ok && t < tiles; t += step) {
                    int mt, nt;
                    tile_at(t, tm, tn, mt, nt);
                    for (int kb = 0; kb < KB; ++kb, ++it) {
                        const int s = it % C::kStages;
                        if (!mbar_wait(&empty[s], ((it / C::kStages) & 1) ^ 1, sAbort, budget)) {
                            *sAbort = 1;
                            atomicOr(p.err, kErrWaitSlotFree);
                            ok = false;
                            break;
                        }
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::kStageBytes);
                        const uint32_t bar = map_rank(smem_u32(&full[s]), 0);
                        uint8_t* st = smem + s * C::kStageBytes;
                        tma_load_2d_pair(st, &tmA, bar, kb * kBK, mt * 256 + rank * 128);
                        // 64 rows of each column half: the half's other 64 are the other CTA's
                        tma_load_2d_pair(st + 128 * kBK, &tmB, bar, kb * kBK, nt * 256 + rank * 64);
                        tma_load_2d_pair(st + 192 * kBK, &tmB, bar, kb * kBK, nt * 256 + 128 + rank * 64);
                    }
                }
                // every load that was issued has landed and been read before the CTA exits
                for (int j = it > C::kStages ? it - C::kStages : 0; j < it; ++j)
                    if (!mbar_wait_drain(&empty[j % C::kStages], (j / C::kStages) & 1)) {
                        atomicOr(p.err, kErrWaitDrain);
                        break;
                    }
            }
            __syncwarp();
        } else if (warp == kPairEpi + 1) {
            // ---------------- MMA issuer
            if (rank == 0 && elect_one()) {
                int it = 0, issued = -1;
                uint32_t parity = 0;
                bool ok = true;
                for (int t = first; ok && t < tiles; t += step) {
                    for (int kb = 0; kb < KB; ++kb, ++it) {
                        const int s = it % C::kStages, a = (it & 1) * 2;
                        if (!mbar_wait(&full[s], (it / C::kStages) & 1, sAbort, budget)) {
                            *sAbort = 1;
                            atomicOr(p.err, kErrWaitTmaFull);
                            ok = false;
                            break;
                        }
                        const uint32_t ab = smem_u32(smem + s * C::kStageBytes), bb = ab + 128 * kBK;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (ok && !mbar_wait(&accEmpty[a + h], ((it >> 1) & 1) ^ 1, sAbort, budget)) {
                                *sAbort = 1;
                                atomicOr(p.err, kErrWaitAccFree);
                                ok = false;
                            }
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int k = 0; k < kBK / 32; ++k)
                                mma_f8_pair(tmem_base + (a + h) * 128, umma_desc(ab + 32 * k, 128),
                                            umma_desc(bb + h * 64 * kBK + 32 * k, 128), idesc_e4m3_pair(128),
                                            k > 0 ? 1u : 0u);
                            if (h == 1) mma_commit_pair(&empty[s]);
                            mma_commit_pair(&accFull[a + h]);
                            issued = a + h;
                            parity = (it >> 1) & 1;
                        }
                        if (!ok) break;
                    }
                }
                // the last commit completes before TMEM is released
                if (issued >= 0 && !mbar_wait_drain(&accFull[issued], parity))
                    atomicOr(p.err, kErrWaitDrain);
            }
            __syncwarp();
        } else if (warp == kPairEpi + 2) {
            // ---------------- scale producer
            int it = 0;
            bool ok = true;
            for (int t = first; ok && t < tiles; t += step) {
                int mt, nt;
                tile_at(t, tm, tn, mt, nt);
                const int m0 = mt * 256 + rank * 128, n0 = nt * 256;
                const float* src[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int m = min(m0 + j * 32 + lane, p.M - 1);
                    src[j] = p.sa + static_cast<int64_t>(p.a_tile ? m / 128 : m) * p.sars;
                }
                for (int kb = 0; kb < KB; ++kb, ++it) {
                    const int s = it % C::kScaleStages;
                    if (!mbar_wait_backoff(&sEmpty[s], ((it / C::kScaleStages) & 1) ^ 1, sAbort, 128, 32, budget)) {
                        *sAbort = 1;
                        atomicOr(p.err, kErrWaitSlotFree);
                        ok = false;
                        break;
                    }
                    float* dst = reinterpret_cast<float*>(smem + C::kOffScale + s * C::kScaleBytes);
#pragma unroll
                    for (int j = 0; j < 4; ++j) cp_async4(dst + j * 32 + lane, src[j] + kb * p.sabs, true);
                    if constexpr (COL == 1) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int n = n0 + j * 32 + lane;
                            cp_async4(dst + 128 + j * 32 + lane,
                                      p.sb + static_cast<int64_t>(min(n, p.N - 1)) * p.sbrs + kb * p.sbbs, n < p.N);
                        }
                    } else if (lane < 2) {
                        const int g = min(n0 + lane * 128, p.N - 1) / 128;
                        cp_async4(dst + 128 + lane, p.sb + static_cast<int64_t>(g) * p.sbrs + kb * p.sbbs, true);
                    }
                    cp_async_arrive(&sFull[s]);
                }
            }
            cp_async_wait_all();
        }
    } else {
        // ---------------- promotion and epilogue
        reg_inc<112>();
        constexpr int W = C::kRead;
        // registers are short in the loop over the blocks (64 accumulators and the columns on their way from
        // TMEM leave about sixteen): the tile's number waits in shared memory, its place is found when
        // it is needed, and the addresses are one number each
        volatile int* my_tile = reinterpret_cast<volatile int*>(sTmem + 4 + warp);
        const uint32_t accEmpty0 = map_rank(smem_u32(accEmpty), 0) + (warp >> 3) * 8;
        const uint32_t tmem0 =
            tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + (warp >> 3) * 128 + ((warp >> 2) & 1) * 64;
        const int row = (warp & 3) * 32 + lane;
        int it = 0;
        bool ok = true;
        if (lane == 0) *my_tile = first;
        __syncwarp();
        while (ok && *my_tile < tiles) {
            float2 acc[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[j] = make_float2(0.0f, 0.0f);
            for (int left = KB; left > 0; --left, ++it) {
                const int par = it & 1, ss = it % C::kScaleStages;
                const float* sc = reinterpret_cast<const float*>(smem + C::kOffScale + ss * C::kScaleBytes);
                if (!mbar_wait(&sFull[ss], (it / C::kScaleStages) & 1, sAbort, budget) ||
                    !mbar_wait(&accFull[par * 2 + (warp >> 3)], (it >> 1) & 1, sAbort, budget)) {
                    *sAbort = 1;
                    atomicOr(p.err, kErrWaitAccFull);
                    ok = false;
                    break;
                }
                tc_fence_after();
                float s = sc[row];
                if constexpr (COL == 0) {
                    s *= sc[128 + (warp >> 3)];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sEmpty[ss]);
                }
#pragma unroll
                for (int c = 0; c < 64 / W; ++c) {
                    uint32_t r[W];
                    tmem_read(tmem0 + par * 256 + c * W, r);
                    if (c == 64 / W - 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(accEmpty0 + par * 16);
                    }
#pragma unroll
                    for (int j = 0; j < W / 4; ++j) {
                        float2 f0 = make_float2(s, s), f1 = f0;
                        if constexpr (COL == 1) {
                            const float4 cs = *reinterpret_cast<const float4*>(sc + 128 + (warp >> 2) * 64 + c * W + 4 * j);
                            f0 = mul2_rn(f0, make_float2(cs.x, cs.y));
                            f1 = mul2_rn(f1, make_float2(cs.z, cs.w));
                        }
                        float2& a0 = acc[c * (W / 2) + 2 * j];
                        float2& a1 = acc[c * (W / 2) + 2 * j + 1];
                        a0 = fma2_rn(make_float2(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1])), f0, a0);
                        a1 = fma2_rn(make_float2(__uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])), f1, a1);
                    }
                }
                if constexpr (COL == 1) {
                    __syncwarp();  // every lane has read the block's scales
                    if (lane == 0) mbar_arrive(&sEmpty[ss]);
                }
            }
            if (!ok) break;
            int mt, nt;
            const int t = *my_tile;
            tile_at(t, tm, tn, mt, nt);
            epilogue<CT, 32>(acc, p, &tmC, smem + C::kOffOut + warp * kOutBytes, mt * 256 + rank * 128 + (warp & 3) * 32,
                             nt * 256 + (warp >> 2) * 64, lane);
            if (lane == 0) *my_tile = t + step;
            __syncwarp();
        }
        if (lane == 0) tma_store_wait_all<0>();
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA leaves while the other may still reach its shared memory
    if (warp == kPairEpi + 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

template <int CT>
bool c_map(CUtensorMap* tmC, const Fp8GemmArgs& p) {
    constexpr int kEl = CT == kF32 ? 4 : 2;
    return !p.tma_c || encode_2d(tmC, CT == kF32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                      : CT == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                 p.C, p.N, p.M, p.ldc * kEl, 128 / kEl, 32, 128);
}

template <int CT>
cudaError_t launch_pair(const Fp8GemmArgs& p, cudaStream_t stream) {
    CUtensorMap tmA{}, tmB{}, tmC{};
    if (p.K > 0 &&
        (!encode_2d(&tmA, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.A, p.K, p.M, p.lda, kBK, 128, 128) ||
         !encode_2d(&tmB, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.B, p.K, p.N, p.ldb, kBK, 64, 128)))
        return cudaErrorInvalidValue;
    if (!c_map<CT>(&tmC, p)) return cudaErrorInvalidValue;
    auto kern = p.b_tile ? fp8_gemm_pair_kernel<0, CT> : fp8_gemm_pair_kernel<1, CT>;
    const int smem = p.b_tile ? PairCfg<0>::kSmemBytes : PairCfg<1>::kSmemBytes;
    cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
    if (e != cudaSuccess) return e;
    const int64_t tiles = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + 255) / 256);
    const int pairs = device_sm_count() / 2;
    kern<<<2 * static_cast<int>(tiles < pairs ? tiles : pairs), kPairThreads, smem, stream>>>(tmA, tmB, tmC, p);
    return cudaGetLastError();
}

// The narrow kernel, for few rows of A (a token to a few hundred): rows of B (weights) on the 128 lanes
// of the MMA and NT rows of A as its columns, so that a product with few rows does not pad them to
// 128, and K split over the CTAs of a cluster so that all SMs read weights.  Each CTA sums its share of
// the blocks, puts the partial tile into its shared memory, and after a cluster barrier every CTA adds
// the partials of its columns in the order of the ranks (deterministic; no atomics, no workspace),
// applies bias and activation and stores.  Up to NT = 64 two CTAs fit an SM; a grid that has no more CTAs
// than SMs takes the memory of both for its own ring instead (DEEP: 64x4096x16384 18.5 -> 15.5 us, the
// latency of a copy over the stages in flight is what a block of K waits for).  Warps: four of promotion for
// each 32 columns (a warp reads 32 x 32 accumulators a block), then one TMA producer, one TMEM owner and
// MMA issuer, one scale producer.
template <int NT, bool DEEP>
struct NarrowCfg {
    static constexpr int kPart = NT < 32 ? NT : 32;  // columns of a promoting warp
    static constexpr int kEpi = 4 * (NT / kPart);
    static constexpr int kThreads = 32 * (kEpi + 4);
    static constexpr int kPerSm = DEEP || NT > 64 ? 1 : 2;
    static constexpr int kABytes = 128 * kBK;
    static constexpr int kStageBytes = kABytes + NT * kBK;
    static constexpr int kStages = (NT > 64 ? 163840 : (DEEP ? 184320 : 98304)) / kStageBytes;
    static constexpr int kAcc = 4;
    static constexpr int kTmem = NT * kAcc;
    static constexpr int kScaleStages = 8;
    static constexpr int kScaleBytes = (128 + NT) * 4;
    static constexpr int kOffScale = kStages * kStageBytes;
    static constexpr int kOffBars = kOffScale + kScaleStages * kScaleBytes;
    static constexpr int kSmemBytes = kOffBars + 8 * (2 * kStages + 2 * kAcc + 2 * kScaleStages) + 16 + 1024;
    static_assert(kPerSm * (kSmemBytes + 1024) <= 228 * 1024, "CTAs per SM");
    static_assert(128 * NT * 4 <= kStages * kStageBytes, "the partial tile takes the place of the stages");
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(cluster_addr)
                 : "memory");
    return v;
}

template <int NT, int CT, bool DEEP>
__global__ void __launch_bounds__(NarrowCfg<NT, DEEP>::kThreads, NarrowCfg<NT, DEEP>::kPerSm)
fp8_gemm_narrow_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                       const Fp8GemmArgs p, const int split) {
    using C = NarrowCfg<NT, DEEP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
    uint64_t* empty = full + C::kStages;
    uint64_t* accFull = empty + C::kStages;
    uint64_t* accEmpty = accFull + C::kAcc;
    uint64_t* sFull = accEmpty + C::kAcc;
    uint64_t* sEmpty = sFull + C::kScaleStages;
    uint32_t* sTmem = reinterpret_cast<uint32_t*>(sEmpty + C::kScaleStages);
    volatile int* sAbort = reinterpret_cast<volatile int*>(sTmem + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);  // (known to be the same in all lanes)
    const int lane = threadIdx.x & 31;
    const int rank = blockIdx.x % split, tile = blockIdx.x / split;  // a cluster is `split` blocks in a row
    const int tx = (p.M + NT - 1) / NT;
    const int n0 = tile / tx * 128, m0 = tile % tx * NT;
    const int KB = (p.K + kBK - 1) / kBK;
    const int kb0 = static_cast<int>(static_cast<int64_t>(KB) * rank / split);
    const int count = static_cast<int>(static_cast<int64_t>(KB) * (rank + 1) / split) - kb0;
    const uint64_t budget = p.wait_ns ? p.wait_ns : kWaitNs;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < C::kAcc; ++s) {
            mbar_init(&accFull[s], 1);
            mbar_init(&accEmpty[s], C::kEpi);
        }
        for (int s = 0; s < C::kScaleStages; ++s) {
            mbar_init(&sFull[s], 32);
            mbar_init(&sEmpty[s], C::kEpi);
        }
        *sAbort = 0;
        fence_mbar_init();
    }
    if (warp == C::kEpi + 1) tmem_alloc(sTmem, C::kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *sTmem;
    float* part = reinterpret_cast<float*>(smem);  // (NT, 128) partial sums, after the last block

    if (warp == C::kEpi) {
        // ---------------- TMA producer
        if (elect_one()) {
            int it = 0;
            for (; it < count; ++it) {
                const int s = it % C::kStages;
                if (!mbar_wait(&empty[s], ((it / C::kStages) & 1) ^ 1, sAbort, budget)) {
                    *sAbort = 1;
                    atomicOr(p.err, kErrWaitSlotFree);
                    break;
                }
                mbar_arrive_expect_tx(&full[s], C::kStageBytes);
                uint8_t* st = smem + s * C::kStageBytes;
                tma_load_2d(st, &tmW, &full[s], (kb0 + it) * kBK, n0);
                tma_load_2d(st + C::kABytes, &tmX, &full[s], (kb0 + it) * kBK, m0);
            }
            // every load that was issued lands before the CTA exits
            for (int j = it > C::kStages ? it - C::kStages : 0; j < it; ++j)
                if (!mbar_wait_drain(&full[j % C::kStages], (j / C::kStages) & 1)) {
                    atomicOr(p.err, kErrWaitDrain);
                    break;
                }
        }
        __syncwarp();
    } else if (warp == C::kEpi + 1) {
        // ---------------- MMA issuer
        if (elect_one()) {
            int it = 0;
            for (; it < count; ++it) {
                const int s = it % C::kStages, a = it % C::kAcc;
                const bool free = mbar_wait(&accEmpty[a], ((it / C::kAcc) & 1) ^ 1, sAbort, budget);
                if (!free || !mbar_wait(&full[s], (it / C::kStages) & 1, sAbort, budget)) {
                    *sAbort = 1;
                    atomicOr(p.err, free ? kErrWaitTmaFull : kErrWaitAccFree);
                    break;
                }
                tc_fence_after();
                const uint32_t ab = smem_u32(smem + s * C::kStageBytes), bb = ab + C::kABytes;
#pragma unroll
                for (int k = 0; k < kBK / 32; ++k)
                    mma_f8(tmem_base + a * NT, umma_desc(ab + 32 * k, 128), umma_desc(bb + 32 * k, 128), idesc_e4m3(NT),
                           k > 0 ? 1u : 0u);
                mma_commit(&empty[s]);
                mma_commit(&accFull[a]);
            }
            // the last commit completes before TMEM is released
            if (it > 0 && !mbar_wait_drain(&accFull[(it - 1) % C::kAcc], ((it - 1) / C::kAcc) & 1))
                atomicOr(p.err, kErrWaitDrain);
        }
        __syncwarp();
    } else if (warp == C::kEpi + 2) {
        // ---------------- scale producer
        const float* src[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = min(n0 + j * 32 + lane, p.N - 1);
            src[j] = p.sb + static_cast<int64_t>(p.b_tile ? n / 128 : n) * p.sbrs;
        }
        for (int it = 0; it < count; ++it) {
            const int s = it % C::kScaleStages, kb = kb0 + it;
            if (!mbar_wait_backoff(&sEmpty[s], ((it / C::kScaleStages) & 1) ^ 1, sAbort, 128, 32, budget)) {
                *sAbort = 1;
                atomicOr(p.err, kErrWaitSlotFree);
                break;
            }
            float* dst = reinterpret_cast<float*>(smem + C::kOffScale + s * C::kScaleBytes);
#pragma unroll
            for (int j = 0; j < 4; ++j) cp_async4(dst + j * 32 + lane, src[j] + kb * p.sbbs, true);
#pragma unroll
            for (int j = 0; j < NT; j += 32) {
                const int m = m0 + j + lane;
                if (j + lane < NT)
                    cp_async4(dst + 128 + j + lane,
                              p.sa + static_cast<int64_t>(min(m, p.M - 1) / (p.a_tile ? 128 : 1)) * p.sars + kb * p.sabs,
                              m < p.M);
            }
            cp_async_arrive(&sFull[s]);
        }
        cp_async_wait_all();
    } else if (warp < C::kEpi) {
        // ---------------- promotion
        constexpr int W = C::kPart;
        const int quad = warp & 3, col0 = (warp >> 2) * W;
        float2 acc[W / 2];
#pragma unroll
        for (int j = 0; j < W / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
        bool ok = true;
        for (int it = 0; it < count; ++it) {
            const int a = it % C::kAcc, ss = it % C::kScaleStages;
            const float* sc = reinterpret_cast<const float*>(smem + C::kOffScale + ss * C::kScaleBytes);
            if (!mbar_wait(&sFull[ss], (it / C::kScaleStages) & 1, sAbort, budget) ||
                !mbar_wait(&accFull[a], (it / C::kAcc) & 1, sAbort, budget)) {
                *sAbort = 1;
                atomicOr(p.err, kErrWaitAccFull);
                ok = false;
                break;
            }
            tc_fence_after();
            const float s = sc[quad * 32 + lane];
            uint32_t r[W];
            tmem_read(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + a * NT + col0, r);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&accEmpty[a]);
#pragma unroll
            for (int j = 0; j < W / 4; ++j) {
                const float4 cs = *reinterpret_cast<const float4*>(sc + 128 + col0 + 4 * j);
                const float2 f0 = mul2_rn(make_float2(s, s), make_float2(cs.x, cs.y));
                const float2 f1 = mul2_rn(make_float2(s, s), make_float2(cs.z, cs.w));
                acc[2 * j] = fma2_rn(make_float2(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1])), f0, acc[2 * j]);
                acc[2 * j + 1] =
                    fma2_rn(make_float2(__uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])), f1, acc[2 * j + 1]);
            }
            __syncwarp();  // every lane has read the block's scales
            if (lane == 0) mbar_arrive(&sEmpty[ss]);
        }
        // the last block's MMAs have read every stage: the partial tile goes in their place
        if (ok) {
#pragma unroll
            for (int j = 0; j < W / 2; ++j) {
                part[(col0 + 2 * j) * 128 + quad * 32 + lane] = acc[j].x;
                part[(col0 + 2 * j + 1) * 128 + quad * 32 + lane] = acc[j].y;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (split > 1) cluster_sync();  // the partial tiles of all ranks are there

    // ---------------- join: this CTA's columns (rows of C), a warp per column, four rows of B a lane
    const bool failed = *sAbort != 0;
    const int cols = (NT + split - 1) / split;
    constexpr int kEl = CT == kF32 ? 4 : 2;
    const bool vec = reinterpret_cast<uintptr_t>(p.C) % (4 * kEl) == 0 && p.ldc % 4 == 0;
    for (int c = rank * cols + warp; c < min(NT, (rank + 1) * cols) && !failed; c += C::kThreads / 32) {
        const int m = m0 + c, n = n0 + lane * 4;
        if (m >= p.M || n >= p.N) continue;
        float4 v;
        if (split == 1) {
            v = *reinterpret_cast<const float4*>(part + c * 128 + lane * 4);
        } else {
            const uint32_t at = smem_u32(part + c * 128 + lane * 4);
            v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float4 w[8];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < split) w[r] = ld_cluster4(map_rank(at, r));
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < split) v.x += w[r].x, v.y += w[r].y, v.z += w[r].z, v.w += w[r].w;
        }
        float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p.bias && n + i < p.N) o[i] += load_any(p.bias, p.btype, n + i);
        if (p.act == 1) {
            const float2 g0 = gelu_sig2(make_float2(o[0], o[1])), g1 = gelu_sig2(make_float2(o[2], o[3]));
            o[0] = g0.x, o[1] = g0.y, o[2] = g1.x, o[3] = g1.y;
        } else if (p.act == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = relu_ref(o[i]);
        }
        const int64_t at = static_cast<int64_t>(m) * p.ldc + n;
        if (vec && n + 4 <= p.N) {
            if constexpr (CT == kF32) {
                *reinterpret_cast<float4*>(static_cast<float*>(p.C) + at) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
                const float2 pr[2] = {make_float2(o[0], o[1]), make_float2(o[2], o[3])};
                uint2 w;
                w.x = pack_half<CT>(pr[0]);
                w.y = pack_half<CT>(pr[1]);
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.C) + at) = w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < p.N) store_any(p.C, CT, at + i, o[i]);
        }
    }

    if (warp == C::kEpi + 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmem);
    }
    if (split > 1) cluster_sync();  // no CTA leaves while another may still read its partial tile
}

template <int NT, int CT, bool DEEP>
cudaError_t launch_narrow(const Fp8GemmArgs& p, int split, cudaStream_t stream) {
    using C = NarrowCfg<NT, DEEP>;
    CUtensorMap tmW{}, tmX{};
    if (p.K > 0 &&
        (!encode_2d(&tmW, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.B, p.K, p.N, p.ldb, kBK, 128, 128) ||
         !encode_2d(&tmX, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.A, p.K, p.M, p.lda, kBK, NT, 128)))
        return cudaErrorInvalidValue;
    auto kern = fp8_gemm_narrow_kernel<NT, CT, DEEP>;
    cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), C::kSmemBytes);
    if (e != cudaSuccess) return e;
    const int64_t tiles = static_cast<int64_t>((p.N + 127) / 128) * ((p.M + NT - 1) / NT);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * split));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(split);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, tmW, tmX, p, split);
}

template <int CT>
cudaError_t dispatch(const Fp8GemmArgs& p, cudaStream_t stream) {
    const Fp8Plan c = fp8_gemm_plan(p.M, p.N, p.K, p.b_tile, device_sm_count());
    if (c.columns == 0) return launch_pair<CT>(p, stream);
    if (c.columns == 16)
        return c.deep ? launch_narrow<16, CT, true>(p, c.split, stream) : launch_narrow<16, CT, false>(p, c.split, stream);
    if (c.columns == 32)
        return c.deep ? launch_narrow<32, CT, true>(p, c.split, stream) : launch_narrow<32, CT, false>(p, c.split, stream);
    if (c.columns == 64)
        return c.deep ? launch_narrow<64, CT, true>(p, c.split, stream) : launch_narrow<64, CT, false>(p, c.split, stream);
    return launch_narrow<128, CT, true>(p, c.split, stream);
}

}  // namespace

// Which kernel, and how it is cut: the cheapest by a model fitted to measurements (us, graphs of launches
// whose operands stay in L2; with weights from HBM 1x4096x4096 takes 8.5 and not 5.9).  KB blocks of K.  Of the figures
// below the model is within 8 %, save 1x4096x4096 without (10 %) and with a split of 2 and 8 (11 and 20 %) and
// 1000x4096x1024 with 128/1 (15 %); of the choices given for a shape, its cheapest is the fastest.
//   narrow, NT columns, K over `split` CTAs   4.3 + rounds ceil(KB / split) c(NT) + 2.5 a further round, + join(NT)
//       c: 0.20, 0.24, 0.32, 0.42 for NT = 16, 32, 64, 128;  join (partials through the cluster): 0.7, 1.0, 1.5, 2.5
//   pair                                      6.5 + rounds KB 0.41 (0.65 with column scales) + 2.2 a further round
// E.g. 256x2048x2048: 7.9 with 32/1, 8.4 with 64/2, 8.8 with 128/4; 300x700x6000: 9.9 with 64/4, 11.9 with
// 128/4; 512x4096x4096: 18.2 with 128/1, 19.6 pair; 1000x4096x1024: 15.9 with 128/1, 9.8 pair; 1x4096x4096: 9.7,
// 7.4, 6.2, 7.6 with a split of 1, 2, 4, 8.  Clusters of four and eight do not fill the SMs of every
// processor cluster, hence 128 CTAs at a time there (300x700x6000 with 128/8, 144 CTAs: 16.6).
Fp8Plan fp8_gemm_plan(int64_t M, int64_t N, int64_t K, int b_tile, int64_t sms) {
    const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const int64_t KB = up(K, kBK);
    constexpr int kCost[4] = {20, 24, 32, 42}, kJoin[4] = {70, 100, 150, 250};  // hundredths of a microsecond
    int nt = 16, split = 1;
    int64_t best = -1;
    for (int i = 0; i < 4; ++i) {
        const int w = 16 << i;
        if (i > 0 && w / 2 >= M) break;
        for (int s = 1; s <= 8 && (s == 1 || 2 * s <= KB); s *= 2) {
            const int64_t ctas = up(N, 128) * up(M, w) * s;
            const int64_t rounds = up(ctas, s >= 4 && sms > 1 ? sms * 7 / 8 : sms);
            const int64_t cost = 430 + rounds * up(KB, s) * kCost[i] + (rounds - 1) * 250 + (s > 1 ? kJoin[i] : 0);
            if (best < 0 || cost < best) best = cost, nt = w, split = s;
        }
    }
    const int64_t rounds = sms > 1 ? up(up(M, 256) * up(N, 256), sms / 2) : 0;
    if (sms > 1 && 650 + rounds * KB * (b_tile ? 41 : 65) + (rounds - 1) * 220 < best) return {0, 1, false};
    return {nt, split, nt == 128 || up(N, 128) * up(M, nt) * split <= sms};
}

cudaError_t fp8_gemm_launch(const Fp8GemmArgs& p_in, cudaStream_t stream) {
    Fp8GemmArgs p = p_in;
    p.wait_ns = debug_wait_budget_ns();
    // a TMA store needs 16-byte aligned rows; a result of one row has no row stride
    if (p.M == 1) p.ldc = (static_cast<int64_t>(p.N) + 15) / 16 * 16;
    p.tma_c = reinterpret_cast<uintptr_t>(p.C) % 16 == 0 && p.ldc * type_bytes(p.ctype) % 16 == 0;
    if (p.ctype == kF32) return dispatch<kF32>(p, stream);
    return p.ctype == kBF16 ? dispatch<kBF16>(p, stream) : dispatch<kF16>(p, stream);
}

}  // namespace nfx
