// gemm_dense.cu -- product of two 16-bit matrices with bias, activation and residual in its epilogue, on
// tcgen05 (kind::f16).
//
//   Z = A B^T + bias,  C = act(Z) + R
//
// A (M, K) and B (N, K) are bf16 or fp16, each with contiguous rows (K-major) or contiguous columns (MN-major:
// the gradient products dX = dZ W and dW = dZ^T X read the forward pass's matrices as they are).  Sums are
// fp32.  The tensor core cuts its running sum off instead of rounding it, which drifts over a long K, so pieces
// of 512 terms (4,096 where C has 16 bits) are summed in TMEM and joined in registers (piece_terms()).
//
// Three kernels: pairs of CTAs on 256 x 256 tiles for large results; the same with K split over the pairs of a cluster
// where such tiles are few; and a narrow one, with K split over a cluster, for few rows of A or few tiles.
// gemm_dense_plan() below chooses; gemm_few.cu takes what has fewer rows still.
//
// Measured (one B200, 1,644 TFLOP/s for a library product of 8192^3 in a burst, 1,355 over seconds; graphs of launches over
// operands that do not fit L2, a few milliseconds long):
//   8192x16384x4096 bf16, bias and GELU   705 to 730 us, 1,510 to 1,560 TFLOP/s; call after call for seconds, as the 1,000 W
//                                         power cap sets the clock, 830 us, 1,325 TFLOP/s.  A block of K takes some 670 cycles
//                                         where its MMAs take 512: 32 KB a block are 49 bytes a cycle and SM from L2
//   4096x2048x8192 to fp32                101 us, 1,362 TFLOP/s; call after call 117 us, 1,174 TFLOP/s: 128 tiles on 74 pairs;
//                                         both operands MN-major
//   4096x4096x4096                        98 us, 1,405 TFLOP/s;   2048x2048x2048   17.1 us, 1,005 TFLOP/s
//   512x4096x4096                         19.9 us (K split over two pairs; 22.7 narrow, 25.7 pairs alone)
//   17, 64, 128, 256 x4096x4096           11.0, 11.8, 12.7, 16.1 us, 3.1 to 2.3 TB/s: 5 us before the first block of K
//   1024x1024x1024                        9.8 us
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "dense_ops.h"
#include "gemm_parts.cuh"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

constexpr int kBK = 64;          // 128 bytes of K: one swizzled row
template <int CT>
constexpr int kPiece = piece_terms(CT) / kBK;  // blocks of K that one TMEM stage sums
constexpr int kOutBytes = 32 * 128;

// K-major tiles lie as rows of 128 bytes (64 of K), MN-major ones as 64 rows of K by 64 elements, one such box of
// 8 KB after the other along MN; both with the 128-byte swizzle.  Their descriptors, and how far a step of
// 16 along K is in units of 16 bytes.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, int t) {
    if (!t) return umma_desc(addr, 128);
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(8192 >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint32_t operand_step(int t) { return t ? 16 * 128 / 16 : 32 / 16; }

// kind::f16, fp32 D, M rows of D and n columns
__device__ __forceinline__ uint32_t idesc_of(int type, int a_t, int b_t, int m, int n) {
    const uint32_t f = type == kBF16 ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | (static_cast<uint32_t>(a_t) << 15) | (static_cast<uint32_t>(b_t) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// The 16 bytes at chunk j of a staging row as numbers.
template <int CT>
__device__ __forceinline__ void add_chunk(uint4 v, float2 (&acc)[32], int j) {
    if constexpr (CT == kF32) {
        acc[2 * j].x += __uint_as_float(v.x), acc[2 * j].y += __uint_as_float(v.y);
        acc[2 * j + 1].x += __uint_as_float(v.z), acc[2 * j + 1].y += __uint_as_float(v.w);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_half<CT>(w[i]);
            acc[4 * j + i].x += f.x, acc[4 * j + i].y += f.y;
        }
    }
}

// Rows of the boxes that each CTA of a pair loads (0: none, the matrix ends before them).
struct PairRows {
    int a[2], b[2];
};
// What the host finds out about the matrices of the epilogue: whether their rows allow TMA.
struct Epi {
    int tma_c, tma_z, tma_r;
};

// ---------------------------------------------------------------------------------------------------------
// One tile is 256 x 256, computed by a pair of CTAs with cta_group::2 MMAs: CTA r holds rows 128 r .. of the
// tile's A and of its B (each operand byte is fetched once per pair, 64 KB for 256 x 256 x 64 products), and rows
// 128 r .. of the result in its TMEM, in two stages of 256 columns: the next tile's (or piece's) MMAs run
// while this one's sums are read.  Warps of each CTA:
//   0-15   epilogue, 32 rows x 64 columns each      16  TMA producer
//   17     TMEM owner; CTA 0's issues the MMAs      18, 19  none
// The epilogue's sums move to registers at once (64 a thread), so a TMEM stage is free again before the
// arithmetic and the stores begin.  Registers: 16 x 32 x 112 + 4 x 32 x 32 = 20 x 32 x 96.
// Barriers: full (CTA 0's, both CTAs' bytes), empty and accFull (both CTAs', by commit), accEmpty (CTA
// 0's, arrivals from the epilogue warps of both), rFull (a warp's residual box).
// ---------------------------------------------------------------------------------------------------------
constexpr int kPairThreads = 640;
constexpr int kPairEpi = 16;
constexpr int kStages = 5;
constexpr int kStageBytes = 2 * 128 * kBK * 2;
constexpr int kOffOut = kStages * kStageBytes;
constexpr int kOffBars = kOffOut + kPairEpi * kOutBytes;
constexpr int kPairSmem = kOffBars + 8 * (2 * kStages + 2 * 2 + kPairEpi) + 16 + 1024;
static_assert(kPairSmem <= 227 * 1024, "shared memory budget");

// Rows m0 .., columns n .. (128 bytes of them) between a staging buffer and a matrix whose rows TMA cannot take.
template <int EL, bool STORE>
__device__ __forceinline__ void copy_rows(uint8_t* buf, void* mat, int64_t ld, int m0, int n, int rows, int cols, int lane) {
    for (int r = 0; r < rows; ++r) {
        uint8_t* g = static_cast<uint8_t*>(mat) + (static_cast<int64_t>(m0 + r) * ld + n) * EL;
        for (int c = lane; c < cols; c += 32) {
            uint8_t* s = buf + swz_offset(r * 128 + c * EL, 128);
            if constexpr (EL == 4) {
                if (STORE) *reinterpret_cast<uint32_t*>(g + c * 4) = *reinterpret_cast<const uint32_t*>(s);
                else *reinterpret_cast<uint32_t*>(s) = *reinterpret_cast<const uint32_t*>(g + c * 4);
            } else {
                if (STORE) *reinterpret_cast<uint16_t*>(g + c * 2) = *reinterpret_cast<const uint16_t*>(s);
                else *reinterpret_cast<uint16_t*>(s) = *reinterpret_cast<const uint16_t*>(g + c * 2);
            }
        }
    }
}

template <int CT>
struct PairEpilogue {
    static constexpr int kEl = CT == kF32 ? 4 : 2;
    static constexpr int kCols = 128 / kEl;  // columns of a box
    static constexpr int kBoxes = 64 / kCols;
    const GemmDenseArgs& p;
    const Epi& e;
    const CUtensorMap *tmC, *tmZ, *tmR;
    uint8_t* buf;
    uint64_t* rbar;
    int lane;
    uint32_t rphase;

    // A TMA store clips a box at 16 bytes, not at the element: a last box whose row ends inside 16 bytes goes
    // out by elements.
    __device__ __forceinline__ bool whole(int n) const { return n + kCols <= p.N || p.N * kEl % 16 == 0; }

    __device__ __forceinline__ void buffer_free() {
        if (lane == 0) tma_store_wait_read<0>();
        __syncwarp();
    }
    __device__ __forceinline__ void fetch_residual(int m0, int n) {
        if (lane == 0) {
            tma_store_wait_read<0>();
            mbar_arrive_expect_tx(rbar, kOutBytes);
            tma_load_2d(buf, tmR, rbar, n, m0);
        }
    }
    __device__ __forceinline__ void put(const float2 (&acc)[32], int b) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(buf + swz_offset(lane * 128 + j * 16, 128)) = pack_chunk<CT, 32>(acc, b * 8 + j);
    }
    // the buffer to rows m0 .., columns n ..
    __device__ __forceinline__ void store(const CUtensorMap* tm, int tma, void* mat, int64_t ld, int m0, int n) {
        if (tma && whole(n)) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                tma_store_2d(tm, buf, n, m0);
                tma_store_commit();
            }
        } else {
            __syncwarp();
            copy_rows<kEl, true>(buf, mat, ld, m0, n, min(32, p.M - m0), min(kCols, p.N - n), lane);
            fence_proxy_async_smem();  // (a residual may land here next)
            __syncwarp();
        }
    }
    // Sums of rows m0 + lane, columns n0 .. n0 + 63; `fetched`: the first residual box is on its way.  False when a
    // residual did not come.
    __device__ __forceinline__ bool finish(float2 (&acc)[32], int m0, int n0, bool fetched, volatile int* abort, uint64_t budget) {
        if (p.bias) {
            float b[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = n0 + j * 32 + lane;
                b[j] = n < p.N ? load_any(p.bias, p.btype, n) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                acc[j].x += __shfl_sync(0xFFFFFFFFu, b[j >> 4], (2 * j) & 31);
                acc[j].y += __shfl_sync(0xFFFFFFFFu, b[j >> 4], (2 * j + 1) & 31);
            }
        }
        if (p.Z) {
#pragma unroll
            for (int b = 0; b < kBoxes; ++b) {
                const int n = n0 + b * kCols;
                if (n >= p.N) break;
                buffer_free();
                put(acc, b);
                store(tmZ, e.tma_z, p.Z, p.ldz, m0, n);
            }
        }
        if (p.act == 1) {
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[j] = gelu_sig2(acc[j]);
        } else if (p.act == 2) {
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[j] = make_float2(relu_ref(acc[j].x), relu_ref(acc[j].y));
        }
#pragma unroll
        for (int b = 0; b < kBoxes; ++b) {
            const int n = n0 + b * kCols;
            if (n >= p.N) break;
            if (p.res) {
                if (e.tma_r) {
                    if (!fetched || b > 0) fetch_residual(m0, n);
                    if (!mbar_wait(rbar, rphase, abort, budget)) return false;
                    rphase ^= 1;
                } else {
                    buffer_free();
                    copy_rows<kEl, false>(buf, const_cast<void*>(p.res), p.ldres, m0, n, min(32, p.M - m0), min(kCols, p.N - n), lane);
                    __syncwarp();
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    add_chunk<CT>(*reinterpret_cast<const uint4*>(buf + swz_offset(lane * 128 + j * 16, 128)), acc, b * 8 + j);
            } else {
                buffer_free();
            }
            put(acc, b);
            store(tmC, e.tma_c, p.C, p.ldc, m0, n);
        }
        return true;
    }
};

// One block of K of a CTA's 128 rows of A and of B into a stage; its bytes count on the barrier `bar`.
__device__ __forceinline__ void load_half(const CUtensorMap& tm, uint8_t* st, uint32_t bar, int t, int mn, int rows, int k) {
    if (t) {
        if (rows > 0) tma_load_2d_pair(st, &tm, bar, mn, k);
        if (rows > 64) tma_load_2d_pair(st + 8192, &tm, bar, mn + 64, k);
    } else if (rows > 0) {
        tma_load_2d_pair(st, &tm, bar, k, mn);
    }
}
__device__ __forceinline__ void load_stage(const GemmDenseArgs& p, const CUtensorMap& tmA, const CUtensorMap& tmB, uint8_t* st, uint32_t bar,
                                           int m, int n, int k, const PairRows& r, uint32_t rank) {
    load_half(tmA, st, bar, p.a_t, m, r.a[rank], k);
    load_half(tmB, st + 16384, bar, p.b_t, n, r.b[rank], k);
}

// LONG: K has more than one piece (5765x1016x192 with GELU: 13.4 us, 13.9 where the epilogue may have to add).
template <int CT, bool LONG>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC,
                 const __grid_constant__ CUtensorMap tmZ, const __grid_constant__ CUtensorMap tmR, const GemmDenseArgs p, const Epi e,
                 const PairRows rows) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOffBars);
    uint64_t* empty = full + kStages;
    uint64_t* accFull = empty + kStages;
    uint64_t* accEmpty = accFull + 2;
    uint64_t* rFull = accEmpty + 2;
    uint32_t* sTmem = reinterpret_cast<uint32_t*>(rFull + kPairEpi);
    volatile int* sAbort = reinterpret_cast<volatile int*>(sTmem + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);  // (known to be the same in all lanes)
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int tm = (p.M + 255) / 256, tn = (p.N + 255) / 256;
    const int tiles = tm * tn;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int KB = (p.K + kBK - 1) / kBK;
    const int piece = LONG ? kPiece<CT> : KB;
    const int pieces = LONG ? (KB + piece - 1) / piece : min(KB, 1);
    const uint64_t budget = p.wait_ns ? p.wait_ns : kWaitNs;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&accFull[s], 1);
            mbar_init(&accEmpty[s], 2 * kPairEpi);
        }
        for (int s = 0; s < kPairEpi; ++s) mbar_init(&rFull[s], 1);
        *sAbort = 0;
        fence_mbar_init();
    }
    if (warp == kPairEpi + 1) tmem_alloc_pair(sTmem, 512);
    if (warp == kPairEpi && lane == 0) prefetch_tmap(&tmA), prefetch_tmap(&tmB);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are ready
    tc_fence_after();
    const uint32_t tmem_base = *sTmem;
    grid_dep_launch();
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on

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
                    const int m = mt * 256 + rank * 128, n = nt * 256 + rank * 128;
                    for (int kb = 0; kb < KB; ++kb, ++it) {
                        const int s = it % kStages;
                        if (!mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, sAbort, budget)) {
                            *sAbort = 1;
                            atomicOr(p.err, kErrWaitSlotFree);
                            ok = false;
                            break;
                        }
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], (rows.a[0] + rows.a[1] + rows.b[0] + rows.b[1]) * kBK * 2);
                        const uint32_t bar = map_rank(smem_u32(&full[s]), 0);
                        uint8_t* st = smem + s * kStageBytes;
                        load_stage(p, tmA, tmB, st, bar, m, n, kb * kBK, rows, rank);
                    }
                }
                // every load that was issued has landed and been read before the CTA exits
                for (int j = it > kStages ? it - kStages : 0; j < it; ++j)
                    if (!mbar_wait_drain(&empty[j % kStages], (j / kStages) & 1)) {
                        atomicOr(p.err, kErrWaitDrain);
                        break;
                    }
            }
            __syncwarp();
        } else if (warp == kPairEpi + 1) {
            // ---------------- MMA issuer
            if (rank == 0 && elect_one()) {
                const uint32_t idesc = idesc_of(p.abtype, p.a_t, p.b_t, 256, 256);
                const uint32_t astep = operand_step(p.a_t), bstep = operand_step(p.b_t);
                int it = 0, acc = 0;  // blocks of K, TMEM stages handed over
                bool ok = true;
                for (int t = first; ok && t < tiles; t += step) {
                    for (int kb = 0; kb < KB; ++kb, ++it) {
                        const int s = it % kStages, in = kb % piece;
                        const bool free = in > 0 || mbar_wait(&accEmpty[acc & 1], ((acc >> 1) & 1) ^ 1, sAbort, budget);
                        if (!free || !mbar_wait(&full[s], (it / kStages) & 1, sAbort, budget)) {
                            *sAbort = 1;
                            atomicOr(p.err, free ? kErrWaitTmaFull : kErrWaitAccFree);
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t ab = smem_u32(smem + s * kStageBytes);
                        const uint64_t ad = operand_desc(ab, p.a_t), bd = operand_desc(ab + 16384, p.b_t);
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k)
                            mma_f16_pair(tmem_base + (acc & 1) * 256, ad + k * astep, bd + k * bstep, idesc, in > 0 || k > 0 ? 1u : 0u);
                        mma_commit_pair(&empty[s]);
                        if (in == piece - 1 || kb == KB - 1) {
                            mma_commit_pair(&accFull[acc & 1]);
                            ++acc;
                        }
                    }
                }
                // the last commit completes before TMEM is released: the last block's stage is empty
                if (it > 0 && !mbar_wait_drain(&empty[(it - 1) % kStages], ((it - 1) / kStages) & 1)) atomicOr(p.err, kErrWaitDrain);
            }
            __syncwarp();
        }
    } else {
        // ---------------- epilogue
        reg_inc<112>();
        const uint32_t accEmpty0 = map_rank(smem_u32(accEmpty), 0);
        const uint32_t tmem0 = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + (warp >> 2) * 64;
        PairEpilogue<CT> epi{p, e, &tmC, &tmZ, &tmR, smem + kOffOut + warp * kOutBytes, &rFull[warp], lane, 0};
        int acc_i = 0;
        bool ok = true;
        for (int t = first; ok && t < tiles; t += step) {
            int mt, nt;
            tile_at(t, tm, tn, mt, nt);
            const int m0 = mt * 256 + rank * 128 + (warp & 3) * 32, n0 = nt * 256 + (warp >> 2) * 64;
            const bool live = m0 < p.M && n0 < p.N;
            const bool fetched = p.res && e.tma_r && !p.Z && live;
            if (fetched) epi.fetch_residual(m0, n0);  // it comes while the tile's sums are formed
            float2 acc[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[j] = make_float2(0.0f, 0.0f);
            for (int i = 0; i < pieces; ++i, ++acc_i) {
                const int st = acc_i & 1;
                if (!mbar_wait(&accFull[st], (acc_i >> 1) & 1, sAbort, budget)) {
                    *sAbort = 1;
                    atomicOr(p.err, kErrWaitAccFull);
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t r[32];
                    tmem_read(tmem0 + st * 256 + c * 32, r);
                    if (c == 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(accEmpty0 + st * 8);
                    }
                    if (!LONG || (CT != kF32 && i == 0)) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[c * 16 + j] = make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            acc[c * 16 + j] = add2_rn(acc[c * 16 + j], make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])));
                    }
                }
            }
            bool coming = fetched;  // a residual box that has not been waited for
            if (ok && live) {
                coming = !epi.finish(acc, m0, n0, fetched, sAbort, budget);
                if (coming) {
                    *sAbort = 1;
                    atomicOr(p.err, kErrWaitTmaFull);
                    ok = false;
                }
            }
            if (coming && lane == 0 && !mbar_wait_drain(&rFull[warp], epi.rphase)) atomicOr(p.err, kErrWaitDrain);
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

CUtensorMapDataType map_type(int t) {
    return t == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : t == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}
// Rows of an operand's box, of which `most` would be a tile's: fewer where the whole matrix has fewer (rows that the
// copy engine fills with zeros are as slow as ones that it reads).  Of MN-major operands whole boxes of 64 are left out.
int box_rows(int t, int64_t mn, int most) { return static_cast<int>(mn >= most ? most : (t ? (mn + 63) / 64 * 64 : (mn + 7) / 8 * 8)); }
// Boxes of an operand: `rows` x 64 of K, or 64 of K by 64 along MN.
bool operand_map(CUtensorMap* tm, int type, const void* base, int t, int64_t mn, int64_t k, int64_t ld, int rows) {
    if (t) return encode_2d(tm, map_type(type), base, mn, k, ld * 2, 64, kBK, 128);
    return encode_2d(tm, map_type(type), base, k, mn, ld * 2, kBK, rows, 128);
}
PairRows pair_rows(const GemmDenseArgs& p) {
    // (a matrix of at most 128 rows has none for the second CTA; of more, the boxes are whole)
    const int a = box_rows(p.a_t, p.M, 128), b = box_rows(p.b_t, p.N, 128);
    return {{a, p.M > 128 ? a : 0}, {b, p.N > 128 ? b : 0}};
}
bool tma_rows(const void* p, int64_t ld, int type) {
    return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * type_bytes(type) % 16 == 0;
}

template <int CT>
cudaError_t launch_pair(const GemmDenseArgs& p, cudaStream_t stream) {
    CUtensorMap tmA{}, tmB{}, tmC{}, tmZ{}, tmR{};
    const PairRows rows = pair_rows(p);
    if (p.K > 0 && (!operand_map(&tmA, p.abtype, p.A, p.a_t, p.M, p.K, p.lda, rows.a[0]) || !operand_map(&tmB, p.abtype, p.B, p.b_t, p.N, p.K, p.ldb, rows.b[0])))
        return cudaErrorInvalidValue;
    constexpr int kEl = CT == kF32 ? 4 : 2;
    // (a matrix of one row has no row stride to speak of)
    const auto pitch = [&](int64_t ld) { return p.M == 1 ? (static_cast<int64_t>(p.N) + 7) / 8 * 8 : ld; };
    Epi e{};
    const auto map = [&](CUtensorMap* tm, const void* m, int64_t ld, int* on) {
        *on = tma_rows(m, pitch(ld), CT);
        return !*on || encode_2d(tm, map_type(CT), m, p.N, p.M, pitch(ld) * kEl, 128 / kEl, 32, 128);
    };
    if (!map(&tmC, p.C, p.ldc, &e.tma_c) || !map(&tmZ, p.Z, p.ldz, &e.tma_z) || !map(&tmR, p.res, p.ldres, &e.tma_r)) return cudaErrorInvalidValue;
    auto kern = CT == kF32 || p.K > piece_terms(CT) ? gemm_pair_kernel<CT, true> : gemm_pair_kernel<CT, CT == kF32>;
    const cudaError_t err = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kPairSmem);
    if (err != cudaSuccess) return err;
    const int64_t tiles = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + 255) / 256);
    const int pairs = device_sm_count() / 2;
    return launch_early(kern, 2 * static_cast<int>(tiles < pairs ? tiles : pairs), kPairThreads, kPairSmem, 2, stream, tmA, tmB, tmC, tmZ, tmR, p, e, rows);
}

// ---------------------------------------------------------------------------------------------------------
// Few tiles and a long K: a cluster of 2 S CTAs for one 256 x 256 tile, each of its S pairs summing a share of K.
// A CTA puts its 128 x 256 partial sums where the operands were, and after a cluster barrier every CTA adds the
// partials of its 256 / S columns in the order of the pairs, applies the epilogue and stores, each lane a
// row.  Warps as in the kernel of pairs, without the idle ones.
// ---------------------------------------------------------------------------------------------------------
constexpr int kSplitThreads = 32 * (kPairEpi + 2);
constexpr int kSplitSmem = kOffOut + 8 * (2 * kStages + 2 * 2) + 16 + 1024;
static_assert(128 * 256 * 4 <= kOffOut, "the partial sums take the place of the operands");

// W columns of a row, from column n on, element `at` of `mat` being the first: stored there (row_store) or added to v
// (row_add).  `vec`: rows start on 16-byte boundaries.
template <int CT, int W>
__device__ __forceinline__ void row_store(void* mat, int64_t at, bool vec, int n, int N, const float (&v)[W]) {
    constexpr int kEl = CT == kF32 ? 4 : 2, kVec = 16 / kEl;
    if (vec && n + W <= N) {
#pragma unroll
        for (int j = 0; j < W; j += kVec) {
            uint4 u;
            if constexpr (CT == kF32) {
                u = make_uint4(__float_as_uint(v[j]), __float_as_uint(v[j + 1]), __float_as_uint(v[j + 2]), __float_as_uint(v[j + 3]));
            } else {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = pack_half<CT>(make_float2(v[j + 2 * i], v[j + 2 * i + 1]));
                u = make_uint4(w[0], w[1], w[2], w[3]);
            }
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(mat) + (at + j) * kEl) = u;
        }
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (n + j < N) store_any(mat, CT, at + j, v[j]);
    }
}
template <int CT, int W>
__device__ __forceinline__ void row_add(const void* mat, int64_t at, bool vec, int n, int N, float (&v)[W]) {
    constexpr int kEl = CT == kF32 ? 4 : 2, kVec = 16 / kEl;
    if (vec && n + W <= N) {
#pragma unroll
        for (int j = 0; j < W; j += kVec) {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(mat) + (at + j) * kEl);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (CT == kF32) {
                    v[j + i] += __uint_as_float(w[i]);
                } else {
                    const float2 f = unpack_half<CT>(w[i]);
                    v[j + 2 * i] += f.x, v[j + 2 * i + 1] += f.y;
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (n + j < N) v[j] += plain_load<CT>(mat, at + j);
    }
}

template <int CT, int S>
__global__ void __launch_bounds__(kSplitThreads, 1)
gemm_split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmDenseArgs p, const PairRows rows) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOffOut);
    uint64_t* empty = full + kStages;
    uint64_t* accFull = empty + kStages;
    uint64_t* accEmpty = accFull + 2;
    uint32_t* sTmem = reinterpret_cast<uint32_t*>(accEmpty + 2);
    volatile int* sAbort = reinterpret_cast<volatile int*>(sTmem + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);  // (known to be the same in all lanes)
    const int lane = threadIdx.x & 31;
    const uint32_t crank = cluster_ctarank(), rank = crank & 1, lead = crank & ~1u;
    const int pair = static_cast<int>(crank >> 1), tn = (p.N + 255) / 256, tile = blockIdx.x / (2 * S);
    const int mt = tile / tn, nt = tile % tn;
    const int KB = (p.K + kBK - 1) / kBK;
    const int kb0 = static_cast<int>(static_cast<int64_t>(KB) * pair / S), count = static_cast<int>(static_cast<int64_t>(KB) * (pair + 1) / S) - kb0;
    constexpr int piece = kPiece<CT>;
    const uint64_t budget = p.wait_ns ? p.wait_ns : kWaitNs;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&accFull[s], 1);
            mbar_init(&accEmpty[s], 2 * kPairEpi);
        }
        *sAbort = 0;
        fence_mbar_init();
    }
    if (warp == kPairEpi + 1) tmem_alloc_pair(sTmem, 512);
    if (warp == kPairEpi && lane == 0) prefetch_tmap(&tmA), prefetch_tmap(&tmB);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the barriers of all CTAs are ready
    tc_fence_after();
    const uint32_t tmem_base = *sTmem;
    float* part = reinterpret_cast<float*>(smem);  // four columns, 128 rows of them, and so on
    grid_dep_launch();
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on

    if (warp == kPairEpi) {
        // ---------------- TMA producer
        if (elect_one()) {
            const int m = mt * 256 + rank * 128, n = nt * 256 + rank * 128;
            int it = 0;
            for (; it < count; ++it) {
                const int s = it % kStages, k = (kb0 + it) * kBK;
                if (!mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, sAbort, budget)) {
                    *sAbort = 1;
                    atomicOr(p.err, kErrWaitSlotFree);
                    break;
                }
                if (rank == 0) mbar_arrive_expect_tx(&full[s], (rows.a[0] + rows.a[1] + rows.b[0] + rows.b[1]) * kBK * 2);
                load_stage(p, tmA, tmB, smem + s * kStageBytes, map_rank(smem_u32(&full[s]), lead), m, n, k, rows, rank);
            }
            // every load that was issued has landed and been read before the partial sums take its place
            for (int j = it > kStages ? it - kStages : 0; j < it; ++j)
                if (!mbar_wait_drain(&empty[j % kStages], (j / kStages) & 1)) {
                    *sAbort = 1;
                    atomicOr(p.err, kErrWaitDrain);
                    break;
                }
        }
        __syncwarp();
    } else if (warp == kPairEpi + 1) {
        // ---------------- MMA issuer
        if (rank == 0 && elect_one()) {
            const uint32_t idesc = idesc_of(p.abtype, p.a_t, p.b_t, 256, 256);
            const uint32_t astep = operand_step(p.a_t), bstep = operand_step(p.b_t);
            int it = 0, acc = 0;
            for (; it < count; ++it) {
                const int s = it % kStages, in = it % piece;
                const bool free = in > 0 || mbar_wait(&accEmpty[acc & 1], ((acc >> 1) & 1) ^ 1, sAbort, budget);
                if (!free || !mbar_wait(&full[s], (it / kStages) & 1, sAbort, budget)) {
                    *sAbort = 1;
                    atomicOr(p.err, free ? kErrWaitTmaFull : kErrWaitAccFree);
                    break;
                }
                tc_fence_after();
                const uint32_t ab = smem_u32(smem + s * kStageBytes);
                const uint64_t ad = operand_desc(ab, p.a_t), bd = operand_desc(ab + 16384, p.b_t);
#pragma unroll
                for (int k = 0; k < kBK / 16; ++k)
                    mma_f16_pair(tmem_base + (acc & 1) * 256, ad + k * astep, bd + k * bstep, idesc, in > 0 || k > 0 ? 1u : 0u);
                mma_commit_pair(&empty[s], 3u << lead);
                if (in == piece - 1 || it == count - 1) {
                    mma_commit_pair(&accFull[acc & 1], 3u << lead);
                    ++acc;
                }
            }
            // the last commit completes before TMEM is released
            if (it > 0 && !mbar_wait_drain(&empty[(it - 1) % kStages], ((it - 1) / kStages) & 1)) atomicOr(p.err, kErrWaitDrain);
        }
        __syncwarp();
    } else {
        // ---------------- the sums to registers, then to shared memory
        const uint32_t accEmpty0 = map_rank(smem_u32(accEmpty), lead);
        const uint32_t tmem0 = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + (warp >> 2) * 64;
        float2 acc[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[j] = make_float2(0.0f, 0.0f);
        bool ok = true;
        for (int i = 0, done = 0; done < count; ++i, done += piece) {
            if (!mbar_wait(&accFull[i & 1], (i >> 1) & 1, sAbort, budget)) {
                *sAbort = 1;
                atomicOr(p.err, kErrWaitAccFull);
                ok = false;
                break;
            }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t r[32];
                tmem_read(tmem0 + (i & 1) * 256 + c * 32, r);
                if (c == 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(accEmpty0 + (i & 1) * 8);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    acc[c * 16 + j] = add2_rn(acc[c * 16 + j], make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])));
            }
        }
        // the last block's MMAs have read every stage of both CTAs
        if (ok) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                *reinterpret_cast<float4*>(part + (((warp >> 2) * 16 + j) * 128 + (warp & 3) * 32 + lane) * 4) =
                    make_float4(acc[2 * j].x, acc[2 * j].y, acc[2 * j + 1].x, acc[2 * j + 1].y);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the partial sums of all pairs are there

    // ---------------- join: 256 / S columns of this CTA's rows, 64 / S of them and 32 rows a warp
    if (warp < kPairEpi && *sAbort == 0) {
        constexpr int W = 64 / S;
        const int r = (warp & 3) * 32 + lane, c0 = pair * (256 / S) + (warp >> 2) * W;
        const int m = mt * 256 + rank * 128 + r, n = nt * 256 + c0;
        float v[W];
        float4 u[S][W / 4];
#pragma unroll
        for (int q = 0; q < S; ++q)
#pragma unroll
            for (int j = 0; j < W / 4; ++j) u[q][j] = ld_cluster4(map_rank(smem_u32(part + ((c0 / 4 + j) * 128 + r) * 4), 2 * q + rank));
#pragma unroll
        for (int j = 0; j < W / 4; ++j) {
            float4 t = u[0][j];
#pragma unroll
            for (int q = 1; q < S; ++q) t.x += u[q][j].x, t.y += u[q][j].y, t.z += u[q][j].z, t.w += u[q][j].w;
            v[4 * j] = t.x, v[4 * j + 1] = t.y, v[4 * j + 2] = t.z, v[4 * j + 3] = t.w;
        }
        if (p.bias) {
            const float b = n + (lane % W) < p.N ? load_any(p.bias, p.btype, n + (lane % W)) : 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) v[j] += __shfl_sync(0xFFFFFFFFu, b, j);
        }
        if (m < p.M && n < p.N) {
            const auto vec_of = [&](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (p.M == 1 || ld * (CT == kF32 ? 4 : 2) % 16 == 0); };
            if (p.Z) row_store<CT, W>(p.Z, static_cast<int64_t>(m) * p.ldz + n, vec_of(p.Z, p.ldz), n, p.N, v);
            if (p.act == 1) {
#pragma unroll
                for (int j = 0; j < W; j += 2) {
                    const float2 g = gelu_sig2(make_float2(v[j], v[j + 1]));
                    v[j] = g.x, v[j + 1] = g.y;
                }
            } else if (p.act == 2) {
#pragma unroll
                for (int j = 0; j < W; ++j) v[j] = relu_ref(v[j]);
            }
            if (p.res) row_add<CT, W>(p.res, static_cast<int64_t>(m) * p.ldres + n, vec_of(p.res, p.ldres), n, p.N, v);
            row_store<CT, W>(p.C, static_cast<int64_t>(m) * p.ldc + n, vec_of(p.C, p.ldc), n, p.N, v);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while another may still reach its shared memory
    if (warp == kPairEpi + 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

template <int CT, int S>
cudaError_t launch_split(const GemmDenseArgs& p, cudaStream_t stream) {
    CUtensorMap tmA{}, tmB{};
    const PairRows rows = pair_rows(p);
    if (!operand_map(&tmA, p.abtype, p.A, p.a_t, p.M, p.K, p.lda, rows.a[0]) || !operand_map(&tmB, p.abtype, p.B, p.b_t, p.N, p.K, p.ldb, rows.b[0]))
        return cudaErrorInvalidValue;
    auto kern = gemm_split_kernel<CT, S>;
    const cudaError_t err = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kSplitSmem);
    if (err != cudaSuccess) return err;
    const int64_t tiles = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + 255) / 256);
    return launch_early(kern, tiles * 2 * S, kSplitThreads, kSplitSmem, 2 * S, stream, tmA, tmB, p, rows);
}

// ---------------------------------------------------------------------------------------------------------
// The narrow kernel, for few rows of A (a token to a few hundred): rows of B (weights) on the 128 lanes of the
// MMA and NT rows of A as its columns, and K split over the CTAs of a cluster so that all SMs read weights.  Each
// CTA sums its share of K, puts the partial tile into its shared memory, and after a cluster barrier every
// CTA adds the partials of its columns in the order of the ranks (deterministic; no atomics, no
// workspace), applies the epilogue and stores.  Up to NT = 64 two CTAs fit an SM; a grid that has no more CTAs
// than SMs takes the memory of both for its own ring instead (DEEP).  Warps: four of epilogue for each 32
// columns, then one TMA producer, one TMEM owner and MMA issuer.
// ---------------------------------------------------------------------------------------------------------
template <int NT, bool DEEP>
struct NarrowCfg {
    static constexpr int kPart = NT < 32 ? NT : 32;  // columns of an epilogue warp
    static constexpr int kEpi = 4 * (NT / kPart);
    static constexpr int kThreads = 32 * (kEpi + 2);
    static constexpr int kPerSm = DEEP || NT > 64 ? 1 : 2;
    static constexpr int kWBytes = 128 * kBK * 2;
    static constexpr int kStageBytes = kWBytes + NT * kBK * 2;
    static constexpr int kStages = (NT > 64 ? 196608 : (DEEP ? 204800 : 98304)) / kStageBytes;
    static constexpr int kTmem = NT * 2 < 32 ? 32 : NT * 2;
    static constexpr int kOffBars = kStages * kStageBytes;
    static constexpr int kSmemBytes = kOffBars + 8 * (2 * kStages + 4) + 16 + 1024;
    static_assert(kPerSm * (kSmemBytes + 1024) <= 228 * 1024, "CTAs per SM");
    static_assert(128 * NT * 4 <= kStages * kStageBytes, "the partial tile takes the place of the stages");
};

template <int NT, int CT, bool DEEP>
__global__ void __launch_bounds__(NarrowCfg<NT, DEEP>::kThreads, NarrowCfg<NT, DEEP>::kPerSm)
gemm_narrow_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const GemmDenseArgs p, const int split,
                   const int wrows, const int xrows) {
    using C = NarrowCfg<NT, DEEP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
    uint64_t* empty = full + C::kStages;
    uint64_t* accFull = empty + C::kStages;
    uint64_t* accEmpty = accFull + 2;
    uint32_t* sTmem = reinterpret_cast<uint32_t*>(accEmpty + 2);
    volatile int* sAbort = reinterpret_cast<volatile int*>(sTmem + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);  // (known to be the same in all lanes)
    const int lane = threadIdx.x & 31;
    const int rank = blockIdx.x % split, all = blockIdx.x / split;  // a cluster is `split` blocks in a row
    const int tx = (p.M + NT - 1) / NT, tiles = tx * ((p.N + 127) / 128);
    const int tile = all % tiles, run = all / tiles;  // run: of K, one of p.runs, each with a C of its own
    const int n0 = tile / tx * 128, m0 = tile % tx * NT;
    const int KB = (p.K + kBK - 1) / kBK, parts = split * p.runs, part_i = run * split + rank;
    const int kb0 = static_cast<int>(static_cast<int64_t>(KB) * part_i / parts);
    const int count = static_cast<int>(static_cast<int64_t>(KB) * (part_i + 1) / parts) - kb0;
    constexpr int piece = kPiece<CT>;
    const uint64_t budget = p.wait_ns ? p.wait_ns : kWaitNs;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&accFull[s], 1);
            mbar_init(&accEmpty[s], C::kEpi);
        }
        *sAbort = 0;
        fence_mbar_init();
    }
    if (warp == C::kEpi + 1) tmem_alloc(sTmem, C::kTmem);
    if (warp == C::kEpi && lane == 0) prefetch_tmap(&tmW), prefetch_tmap(&tmX);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *sTmem;
    grid_dep_launch();
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on
    float* part = reinterpret_cast<float*>(smem);  // (NT, 128) partial sums, after the last block

    if (warp == C::kEpi) {
        // ---------------- TMA producer
        if (elect_one()) {
            int it = 0;
            for (; it < count; ++it) {
                const int s = it % C::kStages, k = (kb0 + it) * kBK;
                if (!mbar_wait(&empty[s], ((it / C::kStages) & 1) ^ 1, sAbort, budget)) {
                    *sAbort = 1;
                    atomicOr(p.err, kErrWaitSlotFree);
                    break;
                }
                mbar_arrive_expect_tx(&full[s], (wrows + xrows) * kBK * 2);
                uint8_t* st = smem + s * C::kStageBytes;
                if (p.b_t) {
                    tma_load_2d(st, &tmW, &full[s], n0, k);
                    if (wrows > 64) tma_load_2d(st + 8192, &tmW, &full[s], n0 + 64, k);
                } else {
                    tma_load_2d(st, &tmW, &full[s], k, n0);
                }
                if (NT >= 64 && p.a_t) {
#pragma unroll
                    for (int j = 0; j < NT / 64; ++j)
                        if (j * 64 < xrows) tma_load_2d(st + C::kWBytes + j * 8192, &tmX, &full[s], m0 + j * 64, k);
                } else {
                    tma_load_2d(st + C::kWBytes, &tmX, &full[s], k, m0);
                }
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
            const uint32_t idesc = idesc_of(p.abtype, p.b_t, p.a_t, 128, NT);
            const uint32_t wstep = operand_step(p.b_t), xstep = operand_step(p.a_t);
            int it = 0, acc = 0;
            for (; it < count; ++it) {
                const int s = it % C::kStages, in = it % piece;
                const bool free = in > 0 || mbar_wait(&accEmpty[acc & 1], ((acc >> 1) & 1) ^ 1, sAbort, budget);
                if (!free || !mbar_wait(&full[s], (it / C::kStages) & 1, sAbort, budget)) {
                    *sAbort = 1;
                    atomicOr(p.err, free ? kErrWaitTmaFull : kErrWaitAccFree);
                    break;
                }
                tc_fence_after();
                const uint32_t wb = smem_u32(smem + s * C::kStageBytes);
                const uint64_t wd = operand_desc(wb, p.b_t), xd = operand_desc(wb + C::kWBytes, p.a_t);
#pragma unroll
                for (int k = 0; k < kBK / 16; ++k)
                    mma_f16(tmem_base + (acc & 1) * NT, wd + k * wstep, xd + k * xstep, idesc, in > 0 || k > 0 ? 1u : 0u);
                mma_commit(&empty[s]);
                if (in == piece - 1 || it == count - 1) {
                    mma_commit(&accFull[acc & 1]);
                    ++acc;
                }
            }
            // the last commit completes before TMEM is released
            if (it > 0 && !mbar_wait_drain(&empty[(it - 1) % C::kStages], ((it - 1) / C::kStages) & 1)) atomicOr(p.err, kErrWaitDrain);
        }
        __syncwarp();
    } else {
        // ---------------- the sums to registers, then to shared memory
        constexpr int W = C::kPart;
        const int quad = warp & 3, col0 = (warp >> 2) * W;
        float2 acc[W / 2];
#pragma unroll
        for (int j = 0; j < W / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
        bool ok = true;
        for (int i = 0, done = 0; done < count; ++i, done += piece) {
            if (!mbar_wait(&accFull[i & 1], (i >> 1) & 1, sAbort, budget)) {
                *sAbort = 1;
                atomicOr(p.err, kErrWaitAccFull);
                ok = false;
                break;
            }
            tc_fence_after();
            uint32_t r[W];
            tmem_read(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + (i & 1) * NT + col0, r);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&accEmpty[i & 1]);
#pragma unroll
            for (int j = 0; j < W / 2; ++j)
                acc[j] = add2_rn(acc[j], make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])));
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
    // (a matrix of one row has no row stride to speak of, a run's C has: it is one of p.runs, M rows apart)
    const bool one_row = p.M == 1 && p.runs == 1;
    const auto vec_of = [&](const void* m, int64_t ld) { return reinterpret_cast<uintptr_t>(m) % (4 * kEl) == 0 && (one_row || ld % 4 == 0); };
    const bool vec_c = vec_of(p.C, p.ldc), vec_z = vec_of(p.Z, p.ldz), vec_r = vec_of(p.res, p.ldres);
    const auto store4 = [&](void* mat, int64_t at, bool vec, int n, const float (&o)[4]) {
        if (vec && n + 4 <= p.N) {
            if constexpr (CT == kF32) {
                *reinterpret_cast<float4*>(static_cast<float*>(mat) + at) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(mat) + at) =
                    make_uint2(pack_half<CT>(make_float2(o[0], o[1])), pack_half<CT>(make_float2(o[2], o[3])));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < p.N) store_any(mat, CT, at + i, o[i]);
        }
    };
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
        if (p.Z) store4(p.Z, static_cast<int64_t>(m) * p.ldz + n, vec_z, n, o);
        if (p.act == 1) {
            const float2 g0 = gelu_sig2(make_float2(o[0], o[1])), g1 = gelu_sig2(make_float2(o[2], o[3]));
            o[0] = g0.x, o[1] = g0.y, o[2] = g1.x, o[3] = g1.y;
        } else if (p.act == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = relu_ref(o[i]);
        }
        if (p.res) {
            const int64_t at = static_cast<int64_t>(m) * p.ldres + n;
            if (vec_r && n + 4 <= p.N) {
                if constexpr (CT == kF32) {
                    const float4 r = *reinterpret_cast<const float4*>(static_cast<const float*>(p.res) + at);
                    o[0] += r.x, o[1] += r.y, o[2] += r.z, o[3] += r.w;
                } else {
                    const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.res) + at);
                    const float2 f0 = unpack_half<CT>(r.x), f1 = unpack_half<CT>(r.y);
                    o[0] += f0.x, o[1] += f0.y, o[2] += f1.x, o[3] += f1.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.N) o[i] += plain_load<CT>(p.res, at + i);
            }
        }
        store4(p.C, (static_cast<int64_t>(run) * p.M + m) * p.ldc + n, vec_c, n, o);
    }

    if (warp == C::kEpi + 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmem);
    }
    if (split > 1) cluster_sync();  // no CTA leaves while another may still read its partial tile
}

template <int NT, int CT, bool DEEP>
cudaError_t launch_narrow(const GemmDenseArgs& p, int split, cudaStream_t stream) {
    using C = NarrowCfg<NT, DEEP>;
    CUtensorMap tmW{}, tmX{};
    const int wrows = box_rows(p.b_t, p.N, 128), xrows = box_rows(p.a_t, p.M, NT);
    if (p.K > 0 && (!operand_map(&tmW, p.abtype, p.B, p.b_t, p.N, p.K, p.ldb, wrows) || !operand_map(&tmX, p.abtype, p.A, p.a_t, p.M, p.K, p.lda, xrows)))
        return cudaErrorInvalidValue;
    auto kern = gemm_narrow_kernel<NT, CT, DEEP>;
    const cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), C::kSmemBytes);
    if (e != cudaSuccess) return e;
    const int64_t tiles = static_cast<int64_t>((p.N + 127) / 128) * ((p.M + NT - 1) / NT);
    return launch_early(kern, tiles * split * p.runs, C::kThreads, C::kSmemBytes, split, stream, tmW, tmX, p, split, wrows, xrows);
}

template <int CT>
cudaError_t narrow(const GemmDenseArgs& p, const DensePlan& c, cudaStream_t stream) {
    if (c.columns == 16) return c.deep ? launch_narrow<16, CT, true>(p, c.split, stream) : launch_narrow<16, CT, false>(p, c.split, stream);
    if (c.columns == 32) return c.deep ? launch_narrow<32, CT, true>(p, c.split, stream) : launch_narrow<32, CT, false>(p, c.split, stream);
    if (c.columns == 64) return c.deep ? launch_narrow<64, CT, true>(p, c.split, stream) : launch_narrow<64, CT, false>(p, c.split, stream);
    return launch_narrow<128, CT, true>(p, c.split, stream);
}

// Joins the sums of the runs of K, in their order, and applies the epilogue; four columns a thread.
template <int CT>
__global__ void __launch_bounds__(256) gemm_join_kernel(const GemmDenseArgs p, const float* sums, int runs, bool vec) {
    grid_dep_launch();
    grid_dep_wait();
    const int64_t per = (p.N + 3) / 4, all = per * p.M, plane = static_cast<int64_t>(p.M) * p.N;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t m = i / per;
        const int n = static_cast<int>(i % per) * 4, cols = min(4, p.N - n);
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float* at = sums + m * p.N + n;
        if (vec) {
            for (int r = 0; r < runs; ++r, at += plane) {
                const float4 f = *reinterpret_cast<const float4*>(at);
                v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
            }
        } else {
            for (int r = 0; r < runs; ++r, at += plane)
                for (int c = 0; c < cols; ++c) v[c] += at[c];
        }
        for (int c = 0; c < cols; ++c) {
            float z = v[c];
            if (p.bias) z += load_any(p.bias, p.btype, n + c);
            if (p.Z) store_any(p.Z, CT, m * p.ldz + n + c, z);
            if (p.act == 1) z = gelu_sig2(make_float2(z, 0.0f)).x;
            else if (p.act == 2) z = relu_ref(z);
            if (p.res) z += plain_load<CT>(p.res, m * p.ldres + n + c);
            store_any(p.C, CT, m * p.ldc + n + c, z);
        }
    }
}

template <int CT>
cudaError_t dispatch(const GemmDenseArgs& p, float* sums, cudaStream_t stream) {
    const DensePlan c = gemm_dense_plan(p.M, p.N, p.K, p.a_t, device_sm_count());
    if (c.runs > 1) {
        GemmDenseArgs q = p;
        q.runs = c.runs, q.C = sums, q.ctype = kF32, q.ldc = p.N, q.bias = nullptr, q.act = 0, q.res = nullptr, q.Z = nullptr;
        const cudaError_t e = narrow<kF32>(q, c, stream);
        if (e != cudaSuccess) return e;
        const int64_t blocks = ((p.N + 3ll) / 4 * p.M + 255) / 256, most = 4ll * device_sm_count();
        return launch_early(gemm_join_kernel<CT>, blocks < most ? blocks : most, 256, 0, 1, stream, p, static_cast<const float*>(sums), c.runs, p.N % 4 == 0);
    }
    if (c.columns == 0) return c.split == 1 ? launch_pair<CT>(p, stream) : (c.split == 2 ? launch_split<CT, 2>(p, stream) : launch_split<CT, 4>(p, stream));
    return narrow<CT>(p, c, stream);
}

// ---------------------------------------------------------------------------------------------------------
// Operands that TMA cannot read (base or row stride no multiple of 16 bytes) are copied first, rows on the boundaries
// that copy_stride() gives.
// ---------------------------------------------------------------------------------------------------------
struct AlignJob {
    const uint16_t* src;
    int64_t ld, rows, cols;
    uint16_t* dst;
    int64_t ldd, per, packs;  // packs of eight elements: in a row, in all
};

// Eight elements of the result a thread, from the two 16-byte words that hold them where both lie inside the matrix.
__global__ void __launch_bounds__(256) align_rows_kernel(const AlignJob a, const AlignJob b) {
    grid_dep_launch();
    grid_dep_wait();
    for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < a.packs + b.packs; e += static_cast<int64_t>(gridDim.x) * 256) {
        const bool second = e >= a.packs;
        const AlignJob& j = second ? b : a;
        const int64_t i = second ? e - a.packs : e, per = j.per;
        int64_t r, c;
        if (j.packs < (1ll << 31)) {
            const uint32_t q = static_cast<uint32_t>(i) / static_cast<uint32_t>(per);
            r = q, c = (static_cast<uint32_t>(i) - q * static_cast<uint32_t>(per)) * 8;
        } else {
            r = i / per, c = i % per * 8;
        }
        const uint16_t* p = j.src + r * j.ld + c;
        const int q = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 7;
        uint32_t w[4];
        if (c + 8 <= j.cols && p - q >= j.src && p - q + 16 <= j.src + (j.rows - 1) * j.ld + j.cols) {
            load8<false>(p, w);
        } else {
            load_single<8>(p, 0, static_cast<int>(j.cols - c < 8 ? j.cols - c : 8), w);
        }
        *reinterpret_cast<uint4*>(j.dst + r * j.ldd + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
// The row stride of a copy: whole lines of 128 bytes, save for short rows (5826x1616x10152 with A along K: 168 us with rows
// on 128-byte boundaries, 181 on 16-byte ones).
int64_t copy_stride(int64_t cols) { return cols > 256 ? (cols + 63) / 64 * 64 : up8(cols); }

}  // namespace

// Which kernel, and how it is cut: the cheapest by a model fitted to 590 measurements (us, graphs of launches over
// operands that do not fit L2 together); KB blocks of 64 along K, rounds of the CTAs (pairs) that run at a time.
//   narrow, NT columns, split s   base + rounds ceil(KB / s) c + further per further round + join (s > 1)
//       NT = 16, 32, 64, 128: base 3.3, 4.6, 5.4, 6.0; c 0.22, 0.22, 0.24, 0.27, where two CTAs share an SM 0.32, 0.36,
//       0.40; further 3.7, 4.2, 5.2, 7.4; join 1.0, 0.6, 0.7, 0.8
//   pairs, split s                5.6 + rounds ceil(KB / s) 0.32 + 1.4 per further round + 0, 1.9, 3.5 (s = 1, 2, 4)
// Clusters do not fill every processor cluster's SMs: 132 CTAs at a time in fours, 112 in eights, 66 and 56 pairs
// (440x4304x11248 as 34 tiles of two pairs each: 79 us, twice what one round takes).  Over
// the 61 measured shapes the choice takes 1.9 % longer than the best one.  E.g. 512x4096x4096: 19.5 with pairs and a
// split of 2, 22.7 with 128/1, 25.7 with pairs alone; 355x3616x7136: 26.6, 36.0, 40.6; 64x1024x1024: 5.2 with 16/4,
// 5.5 with 64/8, 8.5 with 64/1; 1024x1024x1024: 9.4 with 64/1, 9.8 with 128/2, 10.6 pairs.
DensePlan gemm_dense_plan(int64_t M, int64_t N, int64_t K, int a_t, int64_t sms) {
    const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const int64_t KB = up(K, kBK);
    constexpr int kBase[4] = {327, 459, 537, 603}, kCost[4] = {22, 22, 24, 27}, kShared[4] = {32, 36, 40, 0};  // hundredths of a microsecond
    constexpr int kFurther[4] = {366, 424, 520, 735}, kJoin[4] = {100, 60, 73, 75};
    DensePlan plan{a_t ? 64 : 16, 1, false, 1};
    int64_t best = -1;
    for (int i = a_t ? 2 : 0; i < 4; ++i) {  // (boxes of an MN-major A are 64 wide)
        const int w = 16 << i;
        if (w > plan.columns && best >= 0 && w / 2 >= M) break;
        for (int s = 1; s <= 8 && (s == 1 || 2 * s <= KB); s *= 2) {
            const int64_t ctas = up(N, 128) * up(M, w) * s, cap = s == 8 ? up(sms * 3, 4) : (s == 4 ? up(sms * 7, 8) : sms);
            const bool shared = w <= 64 && ctas > sms;
            const int64_t rounds = up(ctas, shared ? 2 * cap : cap);
            const int64_t cost = kBase[i] + rounds * up(KB, s) * (shared ? kShared[i] : kCost[i]) + (rounds - 1) * kFurther[i] + (s > 1 ? kJoin[i] : 0);
            if (best < 0 || cost < best) best = cost, plan = {w, s, w == 128 || ctas <= sms, 1};
        }
    }
    // a long K for a result of a few tiles: runs of K for as many clusters of eight as there are, joined by a second kernel
    // (2.5 us, and some 4 MB of sums a microsecond); 64x64x65536: 34.6 us in one run
    for (int i = a_t ? 2 : 0; i < 4; ++i) {
        const int w = 16 << i;
        if (w > 16 && w / 2 >= M && w > (a_t ? 64 : 16)) break;
        const int64_t ctas = up(N, 128) * up(M, w) * 8, runs = std::min(up(sms * 3, 4) / ctas, KB / 32);
        if (runs < 2) continue;
        const int64_t cost = kBase[i] + up(KB, 8 * runs) * kCost[i] + kJoin[i] + 250 + M * N * runs / 10000;
        if (cost < best) best = cost, plan = {w, 8, true, static_cast<int>(runs)};
    }
    const int64_t tiles = up(M, 256) * up(N, 256), pairs = sms / 2;
    for (int s = 1; s <= 4 && pairs > 0 && (s == 1 || 2 * s <= KB); s *= 2) {
        const int64_t at_a_time = s == 1 ? pairs : (s == 2 ? pairs * 9 / 10 : pairs * 3 / 4);
        if (s > 1 && tiles * s > at_a_time) break;
        const int64_t rounds = up(tiles * s, at_a_time), cost = 560 + rounds * up(KB, s) * 32 + (rounds - 1) * 143 + (s == 1 ? 0 : (s == 2 ? 187 : 351));
        if (cost < best) best = cost, plan = {0, s, false, 1};
    }
    return plan;
}

// The kernel for few rows (gemm_few.cu): CTAs of a cluster share K until each warp has no more steps than it keeps in
// flight, as far as the SMs hold them, two each (1x1024x1024: 2.4 us with one CTA for K, 2.9 with 2, 3.1 with 4;
// 16x4096x4096: 13.4, 10.0, 13.9).
int gemm_few_split(int64_t M, int64_t N, int64_t K, int b_t, int64_t sms) {
    const int64_t cols = b_t ? 64 : (M <= 8 ? 16 : 32), tiles = (N + cols - 1) / cols;
    const int64_t share = b_t ? 384 : (M <= 8 ? 2048 : (M <= 16 ? 768 : 256));
    int split = 1;
    while (split < 8 && K > share * split && tiles * split * 2 <= 2 * sms) split *= 2;
    return split;
}

int64_t gemm_dense_workspace(const void* A, int64_t lda, int a_t, const void* B, int64_t ldb, int b_t, int64_t M, int64_t N, int64_t K) {
    if (few_rows(A, lda, a_t, B, ldb, b_t, M, N, K)) return 0;  // read as they lie
    const int64_t ra = a_t ? K : M, ca = a_t ? M : K, rb = b_t ? K : N, cb = b_t ? N : K;
    const int64_t runs = gemm_dense_plan(M, N, K, a_t, device_sm_count()).runs;
    return (tma_operand(A, lda, ra) ? 0 : 2 * ra * copy_stride(ca)) + (tma_operand(B, ldb, rb) ? 0 : 2 * rb * copy_stride(cb)) + (runs > 1 ? runs * M * N * 4 : 0);
}

cudaError_t gemm_dense_launch(const GemmDenseArgs& args, cudaStream_t stream) {
    GemmDenseArgs p = args;
    p.wait_ns = debug_wait_budget_ns();
    if (few_rows(p.A, p.lda, p.a_t, p.B, p.ldb, p.b_t, p.M, p.N, p.K)) return gemm_few_launch(p, gemm_few_split(p.M, p.N, p.K, p.b_t, device_sm_count()), stream);
    uint16_t* room = static_cast<uint16_t*>(p.ws);
    AlignJob job[2]{};
    const auto align = [&](const void*& base, int64_t& ld, int64_t rows, int64_t cols, AlignJob& j) {
        if (p.K == 0) return;
        if (tma_operand(base, ld, rows)) {
            if (rows <= 1) ld = up8(cols);
            return;
        }
        const int64_t ldd = copy_stride(cols), per = up8(cols) / 8;
        j = {static_cast<const uint16_t*>(base), ld, rows, cols, room, ldd, per, rows * per};
        base = room, ld = ldd, room += rows * ldd;
    };
    align(p.A, p.lda, p.a_t ? p.K : p.M, p.a_t ? p.M : p.K, job[0]);
    align(p.B, p.ldb, p.b_t ? p.K : p.N, p.b_t ? p.N : p.K, job[1]);
    if (const int64_t blocks = (job[0].packs + job[1].packs + 255) / 256; blocks > 0) {
        const int64_t most = 16ll * device_sm_count();
        const cudaError_t e = launch_early(align_rows_kernel, blocks < most ? blocks : most, 256, 0, 1, stream, job[0], job[1]);
        if (e != cudaSuccess) return e;
    }
    p.runs = 1;
    float* sums = reinterpret_cast<float*>(room);  // (rows of eight elements: on a 16-byte boundary)
    if (p.ctype == kF32) return dispatch<kF32>(p, sums, stream);
    return p.ctype == kBF16 ? dispatch<kBF16>(p, sums, stream) : dispatch<kF16>(p, sums, stream);
}

}  // namespace nfx
