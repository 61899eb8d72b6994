// rms_norm_grad.cu -- gradient of the RMS norm, joined with the one that reaches its input from elsewhere.
//
//   a = gamma dy,  xh = h r,  dh = r (a - xh mean(a xh)) + dsum
//   dgamma = sum over rows of dy xh
//
// All sums are fp32; dgamma's are joined in a fixed order by a second kernel (3 us).
//
// Bound by HBM.  Measured (one B200; GPU time, both kernels): 16384x4096 bf16 with dsum 85.6 us, 6.3 TB/s; bf16 with an fp32
// stream 169 us, 6.3 TB/s; 65536x512 bf16 44 us, 6.1 TB/s; 8192x2048 bf16 27.4 us, 4.9 TB/s, 8192x2047 35.2 us; 5003x1031
// fp16 17.8 us; 4096x16384 bf16 137 us, 3.9 TB/s; 2048x20000 256 us.
#include <atomic>

#include "dense_ops.h"
#include "launch.cuh"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "rms_parts.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

// Wider rows than the registers hold: a block of 512 threads takes every gridDim.x-th row in two sweeps, the second from
// L2, and adds its rows' parameter gradients, in their order, to its own row of partial sums (each column always by one
// thread: the launcher makes gridDim.x rows a whole number of boundaries).
constexpr int kWideThreads = 512;

template <typename T, typename H, int VE>
__global__ void __launch_bounds__(kWideThreads, 2) rms_grad_wide_kernel(RmsGradArgs a, Shift sh) {
    __shared__ float red[2][kWideThreads / 32];
    const int tid = threadIdx.x;
    float* pg = a.part + static_cast<int64_t>(blockIdx.x) * a.d;
    const Split<VE> sp(a.d, static_cast<int>((sh.base + static_cast<int64_t>(blockIdx.x) * sh.step) % VE), tid);
    const uint32_t packs = sp.packs;  // (up to 2^31: the number of the next one has no sign)
    const auto gamma = [&](int c) { return a.gamma ? load_any(a.gamma, a.ptype, c) : 1.0f; };
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on
    int buf = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, buf ^= 1) {
        const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
        const H* h = static_cast<const H*>(a.h) + r * a.ldh;
        const H* ds = static_cast<const H*>(a.dsum) + r * a.lddsum;
        const float rs = a.rstd[r];
        const bool begin = r == blockIdx.x;
        float t = 0.0f;
        const auto term = [&](int c, float g, float hv) {
            const float dyx = g * (hv * rs);
            t = fmaf(gamma(c), dyx, t);
            return dyx;
        };
        for (uint32_t k = tid; k < packs; k += kWideThreads) {
            const int c = sp.head + static_cast<int>(k) * VE;
            Elems<T, VE> y;
            Elems<H, VE> x;
            y.load(dy + c), x.load(h + c);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float p = term(c + i, y.at(i), x.at(i));
                if (a.part) pg[c + i] = p + (begin ? 0.0f : pg[c + i]);
            }
        }
        if (VE > 1 && sp.edge >= 0) {
            const float p = term(sp.edge, to_f32(dy[sp.edge]), to_f32(h[sp.edge]));
            if (a.part) pg[sp.edge] = p + (begin ? 0.0f : pg[sp.edge]);
        }
        const float m = __fdiv_rn(row_sum<false>(t, red[buf], kWideThreads / 32), static_cast<float>(a.d)) * rs;
        T* dx = static_cast<T*>(a.dx) + r * a.lddx;
        H* dr = static_cast<H*>(a.dres) + r * a.lddres;
        for (uint32_t k = tid; k < packs; k += kWideThreads) {
            const int c = sp.head + static_cast<int>(k) * VE;
            Elems<T, VE> y;
            Elems<H, VE> x, s;
            y.load(dy + c), x.load(h + c);
            if (a.dsum) s.load(ds + c);
            float o[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                o[i] = rs * fmaf(-x.at(i), m, y.at(i) * gamma(c + i));
                if (a.dsum) o[i] += s.at(i);
            }
            if (a.dx) y.set(o), y.store(dx + c);
            if (a.dres) x.set(o), x.store(dr + c);
        }
        if (VE > 1 && sp.edge >= 0) {
            const int c = sp.edge;
            float o = rs * fmaf(-to_f32(h[c]), m, to_f32(dy[c]) * gamma(c));
            if (a.dsum) o += to_f32(ds[c]);
            if (a.dx) dx[c] = from_f32<T>(o);
            if (a.dres) dr[c] = from_f32<H>(o);
        }
    }
}

template <typename T, typename H, int VE>
cudaError_t rms_grad_wide_go(RmsGradArgs& a, cudaStream_t s) {
    if (VE > 1 && a.parts < a.rows) a.parts = a.parts / VE * VE;  // steps of whole boundaries (a.parts is VE at least)
    return launch_early(rms_grad_wide_kernel<T, H, VE>, a.parts, kWideThreads, 0, 1, s, a, shift_of(a.dy, a.lddy, sizeof(T), VE));
}

// ---------------------------------------------------------------------------------------------------------
// The rows of dy, h and dsum in registers as they were read, each unpacked where it is used; layout as in the
// forward kernel.  Blocks walk over the rows; a thread's columns are the same in every row, so dgamma's sums are
// in its registers and written once per block (with 1,024 threads, 64 registers each, gamma and the sums are in
// shared memory and nothing is fetched ahead).
// ---------------------------------------------------------------------------------------------------------
constexpr int grad_blocks(int most) { return most >= 512 ? 1 : 512 / most; }

template <typename T, typename H, int VE, int VPT, int MOST, bool ONE, bool EDGE>
__global__ void __launch_bounds__(MOST, grad_blocks(MOST)) rms_grad_row_kernel(RmsGradArgs a, Shift sh, bool gvec) {
    __shared__ float red[2][MOST / 32];
    constexpr bool kShared = MOST == 1024, kEdges = EDGE && VE > 1;
    constexpr int kRows = ONE ? MOST / 32 : 1, E = VPT * VE;
    // ONE: element e of lane l at e 32 + l, to join the rows' sums; kShared: the sums, element e of thread t at e
    // threads + t (no bank conflicts), then gamma in the same way
    extern __shared__ float room[];
    const int lane = threadIdx.x & 31, warps = ONE ? 1 : blockDim.x >> 5, threads = blockDim.x;
    const int sub = ONE ? lane : threadIdx.x, mine = ONE ? threadIdx.x >> 5 : 0;
    const int first = (sub >> 5) * VPT * 32 + lane;
    const float inv_d = __frcp_rn(static_cast<float>(a.d));
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    const int s = EDGE ? static_cast<int>((sh.base + (static_cast<int64_t>(blockIdx.x) * kRows + mine) * sh.step) % VE) : 0;
    const Split<VE> sp(a.d, s, sub);
    const auto column = [&](int j) { return (EDGE ? sp.head : 0) + (first + j * 32) * VE; };
    const auto inside = [&](int j) { return EDGE ? first + j * 32 < sp.packs : (first + j * 32) * VE < a.d; };

    Elems<T, VE> ny[VPT];
    Elems<H, VE> nh[VPT], ns[VPT];
    Elems<T, 1> ey;  // the edge element
    Elems<H, 1> eh, es;
    ey.zero(), eh.zero(), es.zero();
    float next_rs = 0.0f;
    const auto fetch = [&](int64_t r) {
        const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
        const H* h = static_cast<const H*>(a.h) + r * a.ldh;
        const H* ds = static_cast<const H*>(a.dsum) + r * a.lddsum;
        if (r < a.rows) next_rs = __ldg(a.rstd + r);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = column(j);
            if (r < a.rows && inside(j)) {
                ny[j].load(dy + c);
                nh[j].load(h + c);
                if (a.dsum) ns[j].load(ds + c);
            } else {
                ny[j].zero(), nh[j].zero(), ns[j].zero();
            }
        }
        if (kEdges && sp.edge >= 0) {
            if (r < a.rows) {
                ey.load(dy + sp.edge);
                eh.load(h + sp.edge);
                if (a.dsum) es.load(ds + sp.edge);
            } else {
                ey.zero(), eh.zero();
            }
        }
    };
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on
    float gam[kShared ? 1 : VPT][VE], pg[kShared ? 1 : VPT][VE];
    float* const sums = room;
    float* const gams = room + E * threads;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = column(j);
        float g[VE];
        if (!EDGE && c < a.d) {
            load_params<T, VE>(a.gamma, a.ptype, gvec, c, 1.0f, g);
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) g[i] = EDGE && a.gamma && c + i < a.d ? load_any(a.gamma, a.ptype, c + i) : 1.0f;
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            if constexpr (kShared) gams[(j * VE + i) * threads + sub] = g[i], sums[(j * VE + i) * threads + sub] = 0.0f;
            else gam[j][i] = g[i], pg[j][i] = 0.0f;
        }
    }
    const float egam = kEdges && a.gamma && sp.edge >= 0 ? load_any(a.gamma, a.ptype, sp.edge) : 1.0f;
    float epg = 0.0f;
    int buf = 0;
    if (!kShared) fetch(static_cast<int64_t>(blockIdx.x) * kRows + mine);
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += step, buf ^= 1) {
        const int64_t r = base + mine;
        const bool live = r < a.rows;
        if (kShared) fetch(r);
        Elems<T, VE> y[VPT];
        Elems<H, VE> h[VPT], ds[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) y[j] = ny[j], h[j] = nh[j], ds[j] = ns[j];
        const float rs = next_rs, fy = ey.at(0), fh = eh.at(0), fs = es.at(0);
        if (!kShared) fetch(r + step);
        float t = 0.0f;
        if (kEdges) {
            const float dyx = fy * (fh * rs);
            t = egam * dyx;
            epg += dyx;
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const int e = (j * VE + i) * threads + sub;
                const float dyx = y[j].at(i) * (h[j].at(i) * rs);
                if constexpr (kShared) {
                    t = fmaf(gams[e], dyx, t);
                    sums[e] += dyx;
                } else {
                    t = fmaf(gam[j][i], dyx, t);
                    pg[j][i] += dyx;
                }
            }
        const float m = row_sum<ONE>(t, red[buf], warps) * inv_d * rs;
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            if (!inside(j)) continue;
            const int c = column(j);
            float o[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float g = kShared ? gams[(j * VE + i) * threads + sub] : gam[j][i];
                o[i] = rs * fmaf(-h[j].at(i), m, y[j].at(i) * g);
                if (a.dsum) o[i] += ds[j].at(i);
            }
            if (a.dx) {
                T* dx = static_cast<T*>(a.dx) + r * a.lddx;
                Elems<T, VE> w;
                w.set(o);
                w.store(dx + c);
            }
            if (a.dres) {
                H* dr = static_cast<H*>(a.dres) + r * a.lddres;
                Elems<H, VE> w;
                w.set(o);
                w.store(dr + c);
            }
        }
        if (kEdges && sp.edge >= 0) {
            float o = rs * fmaf(-fh, m, fy * egam);
            if (a.dsum) o += fs;
            if (a.dx) static_cast<T*>(a.dx)[r * a.lddx + sp.edge] = from_f32<T>(o);
            if (a.dres) static_cast<H*>(a.dres)[r * a.lddres + sp.edge] = from_f32<H>(o);
        }
    }
    if (!a.part) return;
    grid_dep_launch();  // the kernel that joins the blocks' sums may be placed
    if constexpr (ONE) {
        // the block's rows join their sums, one warp after the other (with EDGE each warp's columns are its own: by column)
        if constexpr (EDGE) {
            for (int i = threadIdx.x; i < a.d; i += threads) room[i] = 0.0f;
            __syncthreads();
            for (int k = 0; k < kRows; ++k) {
                if (mine == k) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (inside(e / VE)) room[column(e / VE) + e % VE] += pg[e / VE][e % VE];
                    if (kEdges && sp.edge >= 0) room[sp.edge] += epg;
                }
                __syncthreads();
            }
            for (int c = threadIdx.x; c < a.d; c += threads) a.part[static_cast<int64_t>(blockIdx.x) * a.d + c] = room[c];
            return;
        } else {
            for (int k = 1; k < kRows; ++k) {
                if (mine == k) {
#pragma unroll
                    for (int e = 0; e < E; ++e) room[e * 32 + lane] = pg[e / VE][e % VE];
                }
                __syncthreads();
                if (mine == 0) {
#pragma unroll
                    for (int e = 0; e < E; ++e) pg[e / VE][e % VE] += room[e * 32 + lane];
                }
                __syncthreads();
            }
            if (mine != 0) return;
        }
    }
    float* out = a.part + static_cast<int64_t>(blockIdx.x) * a.d;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = column(j);
        float o[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) o[i] = kShared ? sums[(j * VE + i) * threads + sub] : pg[j][i];
        if (!inside(j)) continue;
        if constexpr (!EDGE) {  // (d is a multiple of VE, the workspace 16-byte aligned)
#pragma unroll
            for (int i = 0; i < VE; i += 4) *reinterpret_cast<float4*>(out + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) out[c + i] = o[i];
        }
    }
    if (kEdges && sp.edge >= 0) out[sp.edge] = epg;
}

// Launches as many blocks as are resident, at most a.parts, and leaves their number there.
template <typename T, typename H, int VE, int VPT, int MOST, bool ONE, bool EDGE>
cudaError_t rms_grad_go(RmsGradArgs& a, cudaStream_t s) {
    auto kern = rms_grad_row_kernel<T, H, VE, VPT, MOST, ONE, EDGE>;
    constexpr int E = VPT * VE;
    // (a row's packs are d / VE at most, its edges go beside them)
    const int packs = a.d / VE, threads = ONE ? MOST : (packs < 1 ? 1 : (packs + 32 * VPT - 1) / (32 * VPT)) * 32, rows = ONE ? MOST / 32 : 1;
    const int smem = MOST == 1024 ? 2 * E * threads * 4 : (ONE ? (E * 32 + VE) * 4 : 0);
    const cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), MOST == 1024 ? 2 * E * 1024 * 4 : smem);
    if (e != cudaSuccess) return e;
    static std::atomic<int> known[64][MOST / 32];  // asked for once per kernel, device and size of block
    std::atomic<int>& at = known[current_device() & 63][threads / 32 - 1];
    int most = at.load(std::memory_order_relaxed);
    if (most == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&most, kern, threads, smem) != cudaSuccess || most < 1) most = 1;
        most *= device_sm_count();
        at.store(most, std::memory_order_relaxed);
    }
    const int64_t want = (a.rows + rows - 1) / rows;
    int64_t grid = want < most ? want : most;
    if (grid > a.parts) grid = a.parts;
    if (EDGE && VE > 1 && grid < want) grid = grid >= VE ? grid / VE * VE : VE;  // steps of whole boundaries (a.parts is VE at least)
    a.parts = static_cast<int>(grid);
    return launch_early(kern, grid, threads, smem, 1, s, a, shift_of(a.dy, a.lddy, sizeof(T), VE), aligned16(a.gamma) && (a.ptype == kF32 || VE == 8));
}

// Sixteen elements a thread where a row's three numbers have 16 bits, eight where some have 32.
template <typename T, typename H, int VE, bool EDGE>
cudaError_t rms_grad_width(RmsGradArgs& a, cudaStream_t s) {
    const int d = a.d / VE * VE;  // (edges need no packs)
    if constexpr (sizeof(H) == 2 && VE > 1) {
        if (d <= 512) return rms_grad_go<T, H, VE, 16 / VE, 256, true, EDGE>(a, s);
        if (d <= 4096) return rms_grad_go<T, H, VE, 16 / VE, 256, false, EDGE>(a, s);
        if (d <= 8192) return rms_grad_go<T, H, VE, 16 / VE, 512, false, EDGE>(a, s);
    } else {
        if constexpr (VE > 1) {
            if (d <= 256) return rms_grad_go<T, H, VE, 8 / VE, 256, true, EDGE>(a, s);
        }
        if (d <= 2048) return rms_grad_go<T, H, VE, 8 / VE, 256, false, EDGE>(a, s);
        if (d <= 4096) return rms_grad_go<T, H, VE, 8 / VE, 512, false, EDGE>(a, s);
    }
    return rms_grad_go<T, H, VE, 16 / VE, 1024, false, EDGE>(a, s);
}

template <typename T, typename H>
cudaError_t rms_grad_t(RmsGradArgs& a, cudaStream_t s) {
    if (a.rows == 0) return cudaSuccess;
    constexpr int VE = 16 / sizeof(T);
    const Shift sy = shift_of(a.dy, a.lddy, sizeof(T), VE);
    const auto like = [&](const void* p, int64_t ld, int64_t el) { return !p || same_shift(sy, shift_of(p, ld, el, VE), a.rows); };
    if (like(a.h, a.ldh, sizeof(H)) && like(a.dsum, a.lddsum, sizeof(H)) && like(a.dx, a.lddx, sizeof(T)) && like(a.dres, a.lddres, sizeof(H))) {
        if (a.d <= 16384 && sy.base == 0 && (a.rows == 1 || sy.step == 0) && a.d % VE == 0) return rms_grad_width<T, H, VE, false>(a, s);
        return a.d <= 16384 ? rms_grad_width<T, H, VE, true>(a, s) : rms_grad_wide_go<T, H, VE>(a, s);
    }
    if (a.d <= 16384) return rms_grad_width<T, H, 1, true>(a, s);
    return rms_grad_wide_go<T, H, 1>(a, s);
}

}  // namespace

// The most blocks that the kernels launch, each with its own partial sums: as many as the SMs hold of narrow rows,
// fewer of wide ones, so that the partial sums stay small against the rows; VE at least.
int rms_norm_parts(int64_t rows, int64_t d) {
    const int64_t sms = device_sm_count(), cap = (d <= 1024 ? 6 : (d <= 2048 ? 4 : 2)) * (sms < 4 ? 4 : sms);
    return static_cast<int>(rows < cap ? rows : cap);
}

cudaError_t rms_norm_backward_launch(const RmsGradArgs& args, int dytype, int htype, cudaStream_t s) {
    RmsGradArgs a = args;
    cudaError_t e;
    if (dytype == kF32) e = rms_grad_t<float, float>(a, s);
    else if (dytype == kBF16) e = htype == kF32 ? rms_grad_t<__nv_bfloat16, float>(a, s) : rms_grad_t<__nv_bfloat16, __nv_bfloat16>(a, s);
    else e = htype == kF32 ? rms_grad_t<__half, float>(a, s) : rms_grad_t<__half, __half>(a, s);
    if (e == cudaSuccess && a.dgamma) e = column_reduce_launch(a.part, a.parts, a.d, a.dgamma, nullptr, a.ptype, s);
    return e;
}

}  // namespace nfx
