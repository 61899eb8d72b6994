// gemm_few.cu -- the 16-bit product for few rows of A (few_rows in dense_ops.h), contiguous ones: a few tokens against a weight, where reading B is
// what has to be done.
//
//   Z = A B^T + bias,  C = act(Z) + R
//
// B goes from memory straight into the registers of mma.sync instructions: no tensor maps, barriers, TMEM or
// copies to set up and wait for, which is most of a small product's time on tcgen05, and the arithmetic is a
// fraction of the time that the bytes take.  A sum does not care about the order of its terms, so each
// lane takes whole 16-byte words and the instruction's k positions are dealt out accordingly:
//   rows of B contiguous: rows of B are the instruction's 16 rows, rows of A its 8 columns.  Lane (g, t) loads 8
//     elements of rows g and g + 8 from k0 + 8 t on, and of row g of A; they feed two instructions.
//   columns of B contiguous: rows of A are the 16 rows, and lane (g, t) loads 8 columns from n0 + 8 g on in the
//     rows k0 + 4 t .. + 3; pairs of rows are joined by byte permutations, and instruction j takes column
//     8 g + j as its column g.
// The eight warps of a block share K by turns, blocks of a cluster by parts; partial sums are joined in a fixed
// order through shared memory, where a warp also adds up the pieces of a long K (piece_terms()).
//
// Measured (one B200, weights from HBM): 1x4096x4096 8.1 to 8.4 us, 4.1 TB/s (narrow kernel 10.0), 1x4096x16384 23 us, 5.8 TB/s,
// 16x4096x4096 9.8 us, 1x1024x1024 2.4 us (4.3), 1x64x64 1.6 us.  Small ones are bound by the launch and one trip to
// memory, large ones by HBM.
#include <cuda_runtime.h>

#include <cstdint>

#include "dense_ops.h"
#include "gemm_parts.cuh"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Rows of A (NT groups of 8) and of B (MT groups of 16, 64 where B's columns are contiguous) of a block, and steps of K
// that a warp has in flight: what 128 registers hold.
template <bool KMAJOR, bool VEC, int NT>
struct Few {
    static constexpr int kMT = NT == 1 ? 1 : 2;
    static constexpr int kRows = KMAJOR ? 8 * NT : 16;
    static constexpr int kCols = KMAJOR ? 16 * kMT : 64;
    static constexpr int kU = KMAJOR ? (NT == 1 ? (VEC ? 8 : 4) : (NT == 2 && VEC ? 3 : 2)) : 3;
    static constexpr int kOut = kRows * kCols;
    static constexpr int kPart = KMAJOR ? kOut : kRows * 66;  // a warp's sums
    static constexpr int kSmem = (kWarps * kPart + kOut) * 4;
    // turns of a warp's loop to a piece of K
    template <int CT>
    __host__ __device__ static constexpr int turns() { return piece_terms(CT) / ((KMAJOR ? 32 : 16) * kU); }
    // where the sum of row m of A and row n of B is among a warp's: a warp's lanes, and 32 columns, lie in unlike banks
    __device__ static constexpr int place(int m, int n) {
        return KMAJOR ? m * kCols + (NT > 1 ? n ^ ((m & 6) << 2) : n) : m * 66 + n + (n >> 5);
    }
};

// LONG: a warp may have more than one piece of K.  Ordinary lengths go without the loop and the sums for that (1x64x64: 1.6 us,
// 1.75 with them; 8x1023x1023 3.8, 4.1), save for the widest form, where that makes no difference.
template <typename T, int CT, bool KMAJOR, bool VEC, int NT, bool LONG>
__global__ void __launch_bounds__(kThreads, 2) gemm_few_kernel(const GemmDenseArgs p, const int split) {
    using F = Few<KMAJOR, VEC, NT>;
    constexpr int kCols = F::kCols, kOut = F::kOut, kPart = F::kPart, kU = F::kU, kMT = F::kMT;
    extern __shared__ float part[];  // (warp, row of A, row of B) sums, then the block's
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % split, n0 = blockIdx.x / split * kCols;
    const uint16_t* A = static_cast<const uint16_t*>(p.A);
    const uint16_t* B = static_cast<const uint16_t*>(p.B);
    constexpr int kStep = KMAJOR ? 32 : 16;  // of K, for a warp
    // Whole steps are dealt out to the ranks in runs and to a block's warps in turn.  What is left of K goes by elements,
    // and without VEC so do the first and the last step, whose words could lie outside the matrix.
    const int steps = p.K / kStep, from = VEC ? 0 : 1, to = VEC ? steps : max(steps - 1, from);
    const int s0 = from + static_cast<int>(static_cast<int64_t>(to - from) * rank / split);
    const int s1 = from + static_cast<int>(static_cast<int64_t>(to - from) * (rank + 1) / split);
    const int single[3] = {steps, 0, steps - 1};  // done by elements, each by another warp of the last rank
    const int which = rank == split - 1 ? kWarps - 1 - warp : 3;
    const bool by_elements = which == 0 ? p.K % kStep != 0 : (!VEC && which < 3 && steps >= which);
    const int64_t arow = p.lda;
    constexpr int kTurns = F::template turns<CT>();

    grid_dep_launch();
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on

    // rows beyond the matrices' ends read the last one: what comes of them is not stored
    if constexpr (KMAJOR) {
        float c[kMT][NT][4];
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) c[i][j][0] = c[i][j][1] = c[i][j][2] = c[i][j][3] = 0.0f;
        const uint16_t* br[2 * kMT];
#pragma unroll
        for (int i = 0; i < 2 * kMT; ++i) br[i] = B + static_cast<int64_t>(min(n0 + g + 8 * i, p.N - 1)) * p.ldb;
        const uint16_t* ar[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) ar[j] = A + min(j * 8 + g, p.M - 1) * arow;
        const auto step = [&](const uint32_t (&wb)[2 * kMT][4], const uint32_t (&wa)[NT][4]) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < kMT; ++i) {
                    mma16<T>(c[i][j], wb[2 * i][0], wb[2 * i + 1][0], wb[2 * i][1], wb[2 * i + 1][1], wa[j][0], wa[j][1]);
                    mma16<T>(c[i][j], wb[2 * i][2], wb[2 * i + 1][2], wb[2 * i][3], wb[2 * i + 1][3], wa[j][2], wa[j][3]);
                }
        };
        const auto put = [&](auto add) {  // to this lane's places
            float* mine = part + warp * kPart;
#pragma unroll
            for (int i = 0; i < kMT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& m = mine[F::place(j * 8 + 2 * t + (e & 1), i * 16 + g + 8 * (e >> 1))];
                        m = add ? m + c[i][j][e] : c[i][j][e];
                        if (LONG) c[i][j][e] = 0.0f;
                    }
        };
        int s = s0 + warp;
        bool first = true;
        for (;;) {
            const int end = LONG ? min(s1, s + kWarps * kU * kTurns) : s1;
            for (; s < end; s += kWarps * kU) {
                uint32_t wb[kU][2 * kMT][4], wa[kU][NT][4];
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    if (s + u * kWarps < s1) {
                        const int k = (s + u * kWarps) * kStep + t * 8;
#pragma unroll
                        for (int i = 0; i < 2 * kMT; ++i) load8<VEC>(br[i] + k, wb[u][i]);
#pragma unroll
                        for (int j = 0; j < NT; ++j) load8<VEC>(ar[j] + k, wa[u][j]);
                    }
                }
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    if (s + u * kWarps < s1) step(wb[u], wa[u]);
            }
            if (!LONG || s >= s1) [[likely]] break;
            if (first) put(std::false_type{});
            else put(std::true_type{});
            first = false;
        }
        if (by_elements) {
            uint32_t wb[2 * kMT][4], wa[NT][4];
            const int k = single[which] * kStep + t * 8;
#pragma unroll
            for (int i = 0; i < 2 * kMT; ++i) load_single<8>(br[i], k, p.K, wb[i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) load_single<8>(ar[j], k, p.K, wa[j]);
            step(wb, wa);
        }
        if (!LONG || first) [[likely]] put(std::false_type{});
        else put(std::true_type{});
    } else {
        float c[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
        const bool whole = n0 + g * 8 + 8 <= p.N;  // else by elements
        const uint16_t* bg = B + (whole ? n0 + g * 8 : 0);
        const uint16_t* ar[2] = {A + min(g, p.M - 1) * arow, A + min(g + 8, p.M - 1) * arow};
        const auto row = [&](int k, uint32_t (&w)[4]) {
            if (whole) load8<VEC>(bg + static_cast<int64_t>(k) * p.ldb, w);
            else load_single<8>(B + static_cast<int64_t>(k) * p.ldb, n0 + g * 8, p.N, w);
        };
        const auto step = [&](const uint32_t (&wb)[4][4], const uint32_t (&wa)[2][2]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t sel = (j & 1) ? 0x7632 : 0x5410;
                const uint32_t lo = __byte_perm(wb[0][j >> 1], wb[1][j >> 1], sel), hi = __byte_perm(wb[2][j >> 1], wb[3][j >> 1], sel);
                mma16<T>(c[j], wa[0][0], wa[1][0], wa[0][1], wa[1][1], lo, hi);
            }
        };
        const auto put = [&](auto add) {
            float* mine = part + warp * kPart;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float& m = mine[F::place(g + 8 * (i >> 1), (2 * t + (i & 1)) * 8 + j)];
                    m = add ? m + c[j][i] : c[j][i];
                    if (LONG) c[j][i] = 0.0f;
                }
        };
        int s = s0 + warp;
        bool first = true;
        for (;;) {
            const int end = LONG ? min(s1, s + kWarps * kU * kTurns) : s1;
            for (; s < end; s += kWarps * kU) {
                uint32_t wb[kU][4][4], wa[kU][2][2];
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    if (s + u * kWarps < s1) {
                        const int k = (s + u * kWarps) * kStep + t * 4;
#pragma unroll
                        for (int r = 0; r < 4; ++r) row(k + r, wb[u][r]);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if constexpr (VEC) {
                                const uint2 v = __ldg(reinterpret_cast<const uint2*>(ar[h] + k));
                                wa[u][h][0] = v.x, wa[u][h][1] = v.y;
                            } else {
                                load_single<4>(ar[h], k, p.K, wa[u][h]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    if (s + u * kWarps < s1) step(wb[u], wa[u]);
            }
            if (!LONG || s >= s1) [[likely]] break;
            if (first) put(std::false_type{});
            else put(std::true_type{});
            first = false;
        }
        if (by_elements) {
            uint32_t wb[4][4], wa[2][2];
            const int k = single[which] * kStep + t * 4;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (k + r < p.K) load_single<8>(B + static_cast<int64_t>(k + r) * p.ldb, n0 + g * 8, p.N, wb[r]);
                else wb[r][0] = wb[r][1] = wb[r][2] = wb[r][3] = 0;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) load_single<4>(ar[h], k, p.K, wa[h]);
            step(wb, wa);
        }
        if (!LONG || first) [[likely]] put(std::false_type{});
        else put(std::true_type{});
    }
    __syncthreads();
    float* sum = part + kWarps * kPart;
    const auto joined = [&](int e) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += part[w * kPart + F::place(e / kCols, e % kCols)];
        return v;
    };
    if (split > 1) {
        for (int e = threadIdx.x; e < kOut; e += kThreads) sum[e] = joined(e);
        cluster_sync();
    }
    const int share = (kOut + split - 1) / split;
    for (int e = rank * share + threadIdx.x; e < min(kOut, (rank + 1) * share); e += kThreads) {
        const int m = e / kCols, n = n0 + e % kCols;
        if (m >= p.M || n >= p.N) continue;
        float v;
        if (split == 1) {
            v = joined(e);
        } else {
            v = 0.0f;
            float w[8];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < split) w[r] = ld_cluster(map_rank(smem_u32(sum + e), r));
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < split) v += w[r];
        }
        if (p.bias) v += load_any(p.bias, p.btype, n);
        if (p.Z) store_any(p.Z, CT, static_cast<int64_t>(m) * p.ldz + n, v);
        if (p.act == 1) v = gelu_sig2(make_float2(v, 0.0f)).x;
        else if (p.act == 2) v = relu_ref(v);
        if (p.res) v += plain_load<CT>(p.res, static_cast<int64_t>(m) * p.ldres + n);
        store_any(p.C, CT, static_cast<int64_t>(m) * p.ldc + n, v);
    }
    if (split > 1) cluster_sync();  // no CTA leaves while another may still read its sums
}

template <typename T, int CT, bool KMAJOR, bool VEC, int NT>
cudaError_t few_go(const GemmDenseArgs& p, int split, cudaStream_t s) {
    using F = Few<KMAJOR, VEC, NT>;
    // (a block has at most one step more than this, a warp then at most turns() turns)
    const bool more = NT == 4 || p.K / (KMAJOR ? 32 : 16) / split >= kWarps * F::kU * F::template turns<CT>();
    auto kern = more ? gemm_few_kernel<T, CT, KMAJOR, VEC, NT, true> : gemm_few_kernel<T, CT, KMAJOR, VEC, NT, NT == 4>;
    constexpr int kSmem = Few<KMAJOR, VEC, NT>::kSmem;
    const cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kSmem);
    if (e != cudaSuccess) return e;
    constexpr int kCols = Few<KMAJOR, VEC, NT>::kCols;
    return launch_early(kern, (p.N + kCols - 1) / kCols * split, kThreads, kSmem, split, s, p, split);
}
template <typename T, int CT, bool KMAJOR, bool VEC>
cudaError_t few_width(const GemmDenseArgs& p, int split, cudaStream_t s) {
    if constexpr (!KMAJOR) return few_go<T, CT, false, VEC, 2>(p, split, s);
    if (p.M <= 8) return few_go<T, CT, true, VEC, 1>(p, split, s);
    if (VEC || p.M <= 16) return few_go<T, CT, true, VEC, 2>(p, split, s);
    return few_go<T, CT, true, false, 4>(p, split, s);
}
template <typename T, int CT>
cudaError_t few_form(const GemmDenseArgs& p, int split, cudaStream_t s) {
    const bool vec = tma_operand(p.A, p.lda, p.M) && tma_operand(p.B, p.ldb, p.b_t ? p.K : p.N);
    if (!p.b_t) return vec ? few_width<T, CT, true, true>(p, split, s) : few_width<T, CT, true, false>(p, split, s);
    return vec ? few_width<T, CT, false, true>(p, split, s) : few_width<T, CT, false, false>(p, split, s);
}

}  // namespace

cudaError_t gemm_few_launch(const GemmDenseArgs& p, int split, cudaStream_t s) {
    if (p.abtype == kBF16) return p.ctype == kF32 ? few_form<__nv_bfloat16, kF32>(p, split, s) : few_form<__nv_bfloat16, kBF16>(p, split, s);
    return p.ctype == kF32 ? few_form<__half, kF32>(p, split, s) : few_form<__half, kF16>(p, split, s);
}

}  // namespace nfx
