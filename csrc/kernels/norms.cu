// Layer norm and RMS norm over the last dimension, forward and backward.
//
//   xh = (x - mean) * rstd,  y = xh * w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g = dy * w,  dx = rstd * (g - mean(g) - xh * mean(g * xh)),  dw = sum_rows dy * xh,  db = sum_rows dy
//   (RMS norm: mean = 0 and no mean(g) term)
//
// A row stays on the chip, in the registers of one warp (short rows) or one block, so x is read
// once; the variance is the mean of squared distances from the mean, not a difference of large
// sums. Backward blocks walk several rows: a thread keeps the same columns for every row and adds
// dw and db up in registers; each block then writes one row of partial sums and a second kernel adds
// them in a fixed order (no atomics).
// Bound by memory: x in and y out; x and dy in and dx out.
#include "kernels/ops.h"
#include "kernels/ops_common.cuh"

#include <algorithm>

namespace bccl {
namespace ops {
namespace {

constexpr int kWarpRows = 8;  // rows of a block whose warps work on a row each

// Columns of access v of a thread: accesses of neighbouring threads are adjacent.
template <int E> __device__ __forceinline__ long long col_of(int v, int tx, int g) {
    return static_cast<long long>(v * g + tx) * E;
}

// WARP: blockDim = (32, kWarpRows), a row per warp; else blockDim = (g, 1), a row per block.
template <int D, int WD, int E, int NV, bool LAYER, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 512) norm_forward_kernel(const NormForwardArgs a) {
    __shared__ float buf[2][32];
    const int tx = threadIdx.x, g = blockDim.x;
    const long long step = WARP ? static_cast<long long>(gridDim.x) * kWarpRows : gridDim.x;
    long long row = WARP ? static_cast<long long>(blockIdx.x) * kWarpRows + threadIdx.y : blockIdx.x;
    const int warps = g >> 5;
    const float inv_h = 1.0f / static_cast<float>(a.h);
    const Bits<D>* x = static_cast<const Bits<D>*>(a.x);
    int parity = 0;
    auto sum = [&](float v) {
        if constexpr (WARP) return warp_sum(v);
        const float s = block_sum(v, buf, parity, tx, warps);
        parity ^= 1;
        return s;
    };
    Raw<D, E> next[NV];
    auto fetch = [&](long long r) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const long long c = col_of<E>(v, tx, g);
            next[v] = c < a.h && r < a.rows ? load_raw_cs<D, E>(x + r * a.x_stride + c) : zero_raw<D, E>();
        }
    };
    fetch(row);
    for (; row < a.rows; row += step) {
        float f[NV][E];
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            unpack<D, E>(next[v], f[v]);
#pragma unroll
            for (int e = 0; e < E; ++e) s += LAYER ? f[v][e] : f[v][e] * f[v][e];
        }
        fetch(row + step);
        // Asked for before the sums, so that they wait for x and the weights together.
        float w[NV][E];
        if (a.w != nullptr) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const long long c = col_of<E>(v, tx, g);
                if (c < a.h) load_f<WD, E>(static_cast<const Bits<WD>*>(a.w) + c, w[v]);
            }
        }
        float mean = 0.0f;
        if constexpr (LAYER) {
            mean = sum(s) * inv_h;
            s = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (col_of<E>(v, tx, g) < a.h) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        f[v][e] -= mean;
                        s = fmaf(f[v][e], f[v][e], s);
                    }
                }
            }
        }
        const float rstd = 1.0f / sqrtf(sum(s) * inv_h + a.eps);
        if (tx == 0) {
            if (LAYER) a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        Bits<D>* y = static_cast<Bits<D>*>(a.y) + row * a.y_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const long long c = col_of<E>(v, tx, g);
            if (c >= a.h) continue;
            float b[E];
            if (LAYER && a.b != nullptr) load_f<WD, E>(static_cast<const Bits<WD>*>(a.b) + c, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                f[v][e] *= rstd;
                if (a.w != nullptr) f[v][e] *= w[v][e];
                if (LAYER && a.b != nullptr) f[v][e] += b[e];
            }
            store_f_cs<D, E>(y + c, f[v]);
        }
    }
}

__device__ __forceinline__ void copy16_async(void* smem, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))),
                 "l"(global)
                 : "memory");
}

// Parameters of a thread's columns in shared memory (its own place, so no barrier), read back as floats.
template <int WD, int E>
__device__ __forceinline__ void keep_params(Bits<WD>* smem, const void* params, long long c) {
    float w[E];
    load_f<WD, E>(static_cast<const Bits<WD>*>(params) + c, w);
    store_f<WD, E>(smem + c, w);
}
template <int WD, int E>
__device__ __forceinline__ void read_params(const Bits<WD>* smem, long long c, float (&w)[E]) {
    constexpr int W = Vec<WD>::E;
#pragma unroll
    for (int i = 0; i < E / W; ++i) {
        float t[W];
        Vec<WD>::unpack(reinterpret_cast<const uint4*>(smem + c)[i], t);
#pragma unroll
        for (int e = 0; e < W; ++e) w[i * W + e] = t[e];
    }
}

// Many rows of 16-byte accesses too long for a warp. Every thread copies its own columns of the next
// STAGES - 1 rows into shared memory with cp.async and only reads what it copied itself, so the copies
// need no barrier and stay in flight whatever the row at hand waits for; a row costs one barrier
// per sum.
template <int D, int WD, int NV, bool LAYER, int STAGES>
__global__ void __launch_bounds__(512, NV <= 2 ? 2 : 1) norm_forward_ring_kernel(const NormForwardArgs a) {
    constexpr int E = Vec<D>::E;
    extern __shared__ uint4 ring[];  // [STAGES][NV][threads], then the parameters
    __shared__ float buf[2][32];
    const int tx = threadIdx.x, g = blockDim.x, warps = g >> 5;
    const float inv_h = 1.0f / static_cast<float>(a.h);
    const Bits<D>* x = static_cast<const Bits<D>*>(a.x);
    Bits<WD>* w_smem = reinterpret_cast<Bits<WD>*>(ring + static_cast<size_t>(STAGES) * NV * g);
    Bits<WD>* b_smem = w_smem + a.h;
    auto issue = [&](long long row, int slot) {
        if (row < a.rows) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const long long c = col_of<E>(v, tx, g);
                if (c < a.h) copy16_async(ring + (static_cast<size_t>(slot) * NV + v) * g + tx, x + row * a.x_stride + c);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const long long c = col_of<E>(v, tx, g);
        if (c >= a.h) continue;
        if (a.w != nullptr) keep_params<WD, E>(w_smem, a.w, c);
        if (LAYER && a.b != nullptr) keep_params<WD, E>(b_smem, a.b, c);
    }
    int slot = 0, parity = 0;
    auto sum = [&](float v) {
        const float s = block_sum(v, buf, parity, tx, warps);
        parity ^= 1;
        return s;
    };
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        issue(row + static_cast<long long>(STAGES - 1) * gridDim.x, slot == 0 ? STAGES - 1 : slot - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        float f[NV][E], s = 0.0f, mean = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (col_of<E>(v, tx, g) >= a.h) continue;
            Vec<D>::unpack(ring[(static_cast<size_t>(slot) * NV + v) * g + tx], f[v]);
#pragma unroll
            for (int e = 0; e < E; ++e) s += LAYER ? f[v][e] : f[v][e] * f[v][e];
        }
        if constexpr (LAYER) {
            mean = sum(s) * inv_h;
            s = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (col_of<E>(v, tx, g) >= a.h) continue;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    f[v][e] -= mean;
                    s = fmaf(f[v][e], f[v][e], s);
                }
            }
        }
        const float rstd = 1.0f / sqrtf(sum(s) * inv_h + a.eps);
        if (tx == 0) {
            if (LAYER) a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        Bits<D>* y = static_cast<Bits<D>*>(a.y) + row * a.y_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const long long c = col_of<E>(v, tx, g);
            if (c >= a.h) continue;
            float p[E];
#pragma unroll
            for (int e = 0; e < E; ++e) f[v][e] *= rstd;
            if (a.w != nullptr) {
                read_params<WD, E>(w_smem, c, p);
#pragma unroll
                for (int e = 0; e < E; ++e) f[v][e] *= p[e];
            }
            if (LAYER && a.b != nullptr) {
                read_params<WD, E>(b_smem, c, p);
#pragma unroll
                for (int e = 0; e < E; ++e) f[v][e] += p[e];
            }
            store_f_cs<D, E>(y + c, f[v]);
        }
        slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
}

// Rows longer than a block's registers hold: three passes over the row, the later ones from L2.
template <int D, int WD, int E, bool LAYER>
__global__ void __launch_bounds__(1024) norm_forward_long_kernel(const NormForwardArgs a) {
    __shared__ float buf[2][32];
    const int tx = threadIdx.x;
    const long long step = static_cast<long long>(blockDim.x) * E;
    const float inv_h = 1.0f / static_cast<float>(a.h);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Bits<D>* x = static_cast<const Bits<D>*>(a.x) + row * a.x_stride;
        Bits<D>* y = static_cast<Bits<D>*>(a.y) + row * a.y_stride;
        float mean = 0.0f;
        if constexpr (LAYER) {
            float s = 0.0f;
            for (long long c = static_cast<long long>(tx) * E; c < a.h; c += step) {
                float f[E];
                unpack<D, E>(load_raw<D, E>(x + c), f);
#pragma unroll
                for (int e = 0; e < E; ++e) s += f[e];
            }
            mean = block_sum(s, buf, 0, tx, blockDim.x >> 5) * inv_h;
        }
        float s = 0.0f;
        for (long long c = static_cast<long long>(tx) * E; c < a.h; c += step) {
            float f[E];
            unpack<D, E>(load_raw<D, E>(x + c), f);
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(f[e] - mean, f[e] - mean, s);
        }
        const float rstd = 1.0f / sqrtf(block_sum(s, buf, 1, tx, blockDim.x >> 5) * inv_h + a.eps);
        __syncthreads();  // RMS norm sums once per row: its buffer is free only now
        if (tx == 0) {
            if (LAYER) a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        for (long long c = static_cast<long long>(tx) * E; c < a.h; c += step) {
            float f[E], w[E], b[E];
            unpack<D, E>(load_raw<D, E>(x + c), f);
            if (a.w != nullptr) load_f<WD, E>(static_cast<const Bits<WD>*>(a.w) + c, w);
            if (LAYER && a.b != nullptr) load_f<WD, E>(static_cast<const Bits<WD>*>(a.b) + c, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                f[e] = (f[e] - mean) * rstd;
                if (a.w != nullptr) f[e] *= w[e];
                if (LAYER && a.b != nullptr) f[e] += b[e];
            }
            store_f_cs<D, E>(y + c, f);
        }
    }
}

template <int D, int WD, int E, int NV, bool LAYER, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 512) norm_backward_kernel(const NormBackwardArgs a) {
    extern __shared__ float rows_sum[];  // WARP: one row of partial sums per warp
    __shared__ float2 buf[2][32];
    const int tx = threadIdx.x, g = blockDim.x;
    const long long step = WARP ? static_cast<long long>(gridDim.x) * kWarpRows : gridDim.x;
    long long row = WARP ? static_cast<long long>(blockIdx.x) * kWarpRows + threadIdx.y : blockIdx.x;
    const int warps = g >> 5;
    const float inv_h = 1.0f / static_cast<float>(a.h);
    const Bits<D>* x = static_cast<const Bits<D>*>(a.x);
    const Bits<D>* dy = static_cast<const Bits<D>*>(a.dy);
    int parity = 0;
    float dw[NV][E], db[LAYER ? NV : 1][LAYER ? E : 1];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dw[v][e] = 0.0f;
            if (LAYER) db[v][e] = 0.0f;
        }
    Raw<D, E> nx[NV], ny[NV];
    auto fetch = [&](long long r) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const long long c = col_of<E>(v, tx, g);
            const bool in = c < a.h && r < a.rows;
            nx[v] = in ? load_raw_cs<D, E>(x + r * a.x_stride + c) : zero_raw<D, E>();
            ny[v] = in ? load_raw_cs<D, E>(dy + r * a.dy_stride + c) : zero_raw<D, E>();
        }
    };
    fetch(row);
    for (; row < a.rows; row += step) {
        const float mean = LAYER ? __ldg(a.mean + row) : 0.0f;
        const float rstd = __ldg(a.rstd + row);
        float xh[NV][E], gr[NV][E];
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const long long c = col_of<E>(v, tx, g);
            unpack<D, E>(nx[v], xh[v]);
            unpack<D, E>(ny[v], gr[v]);
            if (c >= a.h) continue;
            float w[E];
            if (a.w != nullptr) load_f<WD, E>(static_cast<const Bits<WD>*>(a.w) + c, w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[v][e] = (xh[v][e] - mean) * rstd;
                dw[v][e] = fmaf(gr[v][e], xh[v][e], dw[v][e]);
                if (LAYER) db[v][e] += gr[v][e];
                if (a.w != nullptr) gr[v][e] *= w[e];
                s.x += gr[v][e];
                s.y = fmaf(gr[v][e], xh[v][e], s.y);
            }
        }
        fetch(row + step);
        if constexpr (WARP) {
            s = warp_sum(s);
        } else {
            s = block_sum(s, buf, parity, tx, warps);
            parity ^= 1;
        }
        const float m1 = LAYER ? s.x * inv_h : 0.0f, m2 = s.y * inv_h;
        Bits<D>* dx = static_cast<Bits<D>*>(a.dx) + row * a.dx_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const long long c = col_of<E>(v, tx, g);
            if (c >= a.h) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) gr[v][e] = rstd * (gr[v][e] - m1 - xh[v][e] * m2);
            store_f_cs<D, E>(dx + c, gr[v]);
        }
    }
    if (a.partials == nullptr) return;
    // partials: [blocks][h] of dw, then of db.
    float* pw = a.partials + blockIdx.x * a.h;
    float* pb = a.partials + (static_cast<long long>(gridDim.x) + blockIdx.x) * a.h;
    auto put = [&](float* to, float (&sum)[NV][E]) {
        if constexpr (WARP) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const long long c = col_of<E>(v, tx, g) + e;
                    if (c < a.h) rows_sum[threadIdx.y * a.h + c] = sum[v][e];
                }
            __syncthreads();
            for (long long c = threadIdx.y * 32 + tx; c < a.h; c += 32 * kWarpRows) {
                float t = 0.0f;
#pragma unroll
                for (int r = 0; r < kWarpRows; ++r) t += rows_sum[r * a.h + c];
                to[c] = t;
            }
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const long long c = col_of<E>(v, tx, g);
                if (c < a.h) {
#pragma unroll
                    for (int e = 0; e < E; ++e) to[c + e] = sum[v][e];
                }
            }
        }
    };
    if (a.dw != nullptr) put(pw, dw);
    if constexpr (LAYER) {
        if (a.db != nullptr) put(pb, db);
    }
}

// Rows of 16-byte accesses too long for a warp. Every thread copies its own columns of the next
// STAGES - 1 rows of x and dy into shared memory with cp.async, and only reads what it copied
// itself, so the copies need no barrier and keep 2 blocks' rings of up to 112 KiB in flight per SM; a
// row costs one barrier, for its sums. The second use of a row reads it from shared memory again
// instead of holding it in registers.
template <int D, int WD, int NV, bool LAYER, int STAGES>
__global__ void __launch_bounds__(512, NV <= 2 ? 2 : 1) norm_backward_ring_kernel(const NormBackwardArgs a) {
    constexpr int E = Vec<D>::E;
    extern __shared__ uint4 ring[];  // [STAGES][x, dy][NV][threads], then the weights' accesses
    __shared__ float2 buf[2][32];
    const int tx = threadIdx.x, g = blockDim.x, warps = g >> 5;
    const float inv_h = 1.0f / static_cast<float>(a.h);
    const Bits<D>* x = static_cast<const Bits<D>*>(a.x);
    const Bits<D>* dy = static_cast<const Bits<D>*>(a.dy);
    Bits<WD>* weights = reinterpret_cast<Bits<WD>*>(ring + static_cast<size_t>(STAGES) * 2 * NV * g);
    auto issue = [&](long long row, int slot) {
        if (row < a.rows) {
            uint4* to = ring + static_cast<size_t>(slot) * 2 * NV * g + tx;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const long long c = col_of<E>(v, tx, g);
                if (c < a.h) {
                    copy16_async(to + v * g, x + row * a.x_stride + c);
                    copy16_async(to + (NV + v) * g, dy + row * a.dy_stride + c);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
    float dw[NV][E], db[LAYER ? NV : 1][E];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const long long c = col_of<E>(v, tx, g);
        if (a.w != nullptr && c < a.h) keep_params<WD, E>(weights, a.w, c);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dw[v][e] = 0.0f;
            if constexpr (LAYER) db[v][e] = 0.0f;
        }
    }
    int slot = 0, parity = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        issue(row + static_cast<long long>(STAGES - 1) * gridDim.x, slot == 0 ? STAGES - 1 : slot - 1);
        const float mean = LAYER ? __ldg(a.mean + row) : 0.0f;
        const float rstd = __ldg(a.rstd + row);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        const uint4* from = ring + static_cast<size_t>(slot) * 2 * NV * g + tx;
        auto load = [&](int v, float (&xh)[E], float (&gr)[E], float (&w)[E]) {
            Vec<D>::unpack(from[v * g], xh);
            Vec<D>::unpack(from[(NV + v) * g], gr);
#pragma unroll
            for (int e = 0; e < E; ++e) xh[e] = (xh[e] - mean) * rstd;
            if (a.w == nullptr) {
#pragma unroll
                for (int e = 0; e < E; ++e) w[e] = 1.0f;
            } else {
                read_params<WD, E>(weights, col_of<E>(v, tx, g), w);
            }
        };
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (col_of<E>(v, tx, g) >= a.h) continue;
            float xh[E], gr[E], w[E];
            load(v, xh, gr, w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dw[v][e] = fmaf(gr[e], xh[e], dw[v][e]);
                if constexpr (LAYER) db[v][e] += gr[e];
                const float gw = gr[e] * w[e];
                if (LAYER) s.x += gw;
                s.y = fmaf(gw, xh[e], s.y);
            }
        }
        s = block_sum(s, buf, parity, tx, warps);
        parity ^= 1;
        const float m1 = LAYER ? s.x * inv_h : 0.0f, m2 = s.y * inv_h;
        Bits<D>* dx = static_cast<Bits<D>*>(a.dx) + row * a.dx_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const long long c = col_of<E>(v, tx, g);
            if (c >= a.h) continue;
            float xh[E], gr[E], w[E];
            load(v, xh, gr, w);
#pragma unroll
            for (int e = 0; e < E; ++e) gr[e] = rstd * (gr[e] * w[e] - m1 - xh[e] * m2);
            store_f_cs<D, E>(dx + c, gr);
        }
        slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
    if (a.partials == nullptr) return;
    float* pw = a.partials + blockIdx.x * a.h;
    float* pb = a.partials + (static_cast<long long>(gridDim.x) + blockIdx.x) * a.h;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const long long c = col_of<E>(v, tx, g);
        if (c >= a.h) continue;
        if (a.dw != nullptr) store_f<kF32, E>(reinterpret_cast<Bits<kF32>*>(pw + c), dw[v]);
        if constexpr (LAYER) {
            if (a.db != nullptr) store_f<kF32, E>(reinterpret_cast<Bits<kF32>*>(pb + c), db[v]);
        }
    }
}

// Rows longer than a block's registers hold: dx in two passes over the row, and dw / db by a
// second kernel that reads x and dy again by columns.
template <int D, int WD, int E, bool LAYER>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(const NormBackwardArgs a) {
    __shared__ float2 buf[2][32];
    const int tx = threadIdx.x;
    const long long step = static_cast<long long>(blockDim.x) * E;
    const float inv_h = 1.0f / static_cast<float>(a.h);
    int parity = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
        const Bits<D>* x = static_cast<const Bits<D>*>(a.x) + row * a.x_stride;
        const Bits<D>* dy = static_cast<const Bits<D>*>(a.dy) + row * a.dy_stride;
        Bits<D>* dx = static_cast<Bits<D>*>(a.dx) + row * a.dx_stride;
        const float mean = LAYER ? __ldg(a.mean + row) : 0.0f;
        const float rstd = __ldg(a.rstd + row);
        float2 s = make_float2(0.0f, 0.0f);
        auto load = [&](long long c, float (&xh)[E], float (&gr)[E]) {
            float w[E];
            unpack<D, E>(load_raw<D, E>(x + c), xh);
            unpack<D, E>(load_raw<D, E>(dy + c), gr);
            if (a.w != nullptr) load_f<WD, E>(static_cast<const Bits<WD>*>(a.w) + c, w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[e] = (xh[e] - mean) * rstd;
                if (a.w != nullptr) gr[e] *= w[e];
            }
        };
        for (long long c = static_cast<long long>(tx) * E; c < a.h; c += step) {
            float xh[E], gr[E];
            load(c, xh, gr);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s.x += gr[e];
                s.y = fmaf(gr[e], xh[e], s.y);
            }
        }
        s = block_sum(s, buf, parity, tx, blockDim.x >> 5);
        const float m1 = LAYER ? s.x * inv_h : 0.0f, m2 = s.y * inv_h;
        for (long long c = static_cast<long long>(tx) * E; c < a.h; c += step) {
            float xh[E], gr[E];
            load(c, xh, gr);
#pragma unroll
            for (int e = 0; e < E; ++e) gr[e] = rstd * (gr[e] - m1 - xh[e] * m2);
            store_f_cs<D, E>(dx + c, gr);
        }
    }
}

template <int D, int E, bool LAYER>
__global__ void __launch_bounds__(256) norm_columns_kernel(const NormBackwardArgs a) {
    __shared__ float part[8][32 * E];
    const long long c = (static_cast<long long>(blockIdx.x) * 32 + threadIdx.x) * E;
    float dw[E] = {}, db[E] = {};
    if (c < a.h) {
        for (long long row = static_cast<long long>(blockIdx.y) * 8 + threadIdx.y; row < a.rows;
             row += static_cast<long long>(gridDim.y) * 8) {
            float x[E], dy[E];
            unpack<D, E>(load_raw_cs<D, E>(static_cast<const Bits<D>*>(a.x) + row * a.x_stride + c), x);
            unpack<D, E>(load_raw_cs<D, E>(static_cast<const Bits<D>*>(a.dy) + row * a.dy_stride + c), dy);
            const float mean = LAYER ? __ldg(a.mean + row) : 0.0f, rstd = __ldg(a.rstd + row);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dw[e] = fmaf(dy[e], (x[e] - mean) * rstd, dw[e]);
                db[e] += dy[e];
            }
        }
    }
    auto put = [&](float* to, const float (&sum)[E]) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) part[threadIdx.y][threadIdx.x * E + e] = sum[e];
        __syncthreads();
        for (int i = threadIdx.y * 32 + threadIdx.x; i < 32 * E; i += 256) {
            const long long col = static_cast<long long>(blockIdx.x) * 32 * E + i;
            if (col >= a.h) continue;
            float t = 0.0f;
#pragma unroll
            for (int r = 0; r < 8; ++r) t += part[r][i];
            to[col] = t;
        }
    };
    if (a.dw != nullptr) put(a.partials + blockIdx.y * a.h, dw);
    if (LAYER && a.db != nullptr) put(a.partials + (static_cast<long long>(gridDim.y) + blockIdx.y) * a.h, db);
}

// Sums `blocks` rows of partials: 32 columns per block, 32 threads down each column.
// blockIdx.y: 0 dw, 1 db.
template <int WD>
__global__ void __launch_bounds__(1024) norm_weights_kernel(const float* __restrict__ partials, int blocks, long long h,
                                                            void* dw, void* db) {
    __shared__ float part[32][33];
    void* out = blockIdx.y == 0 ? dw : db;
    if (out == nullptr) return;
    const float* p = partials + (blockIdx.y == 0 ? 0 : blocks * h);
    const long long c = static_cast<long long>(blockIdx.x) * 32 + threadIdx.x;
    float t = 0.0f;
    if (c < h) {
#pragma unroll 4
        for (int b = threadIdx.y; b < blocks; b += 32) t += p[b * h + c];
    }
    part[threadIdx.y][threadIdx.x] = t;
    __syncthreads();
    t = warp_sum(part[threadIdx.x][threadIdx.y]);
    const long long col = static_cast<long long>(blockIdx.x) * 32 + threadIdx.y;
    if (threadIdx.x == 0 && col < h) static_cast<Bits<WD>*>(out)[col] = Ty<WD>::store(t);
}

// How a row is spread: accesses per thread and threads per row (32: a warp). Zero threads: long.
struct Shape {
    int nv, threads;
};
// Widths tried in order, the first that fits; more accesses per thread mean fewer warps to
// synchronise per row, fewer accesses more rows in flight.
Shape forward_shape(long long h, int e) {
    const long long n = ceil_div(h, e);
    if (e > 1) {
        for (int nv : {1, 2, 4})
            if (n <= 32 * nv) return {nv, 32};
        if (n <= 512) return {1, round32(n)};
        if (n <= 1024) return {2, round32(ceil_div(n, 2))};
        if (n <= 2048) return {4, round32(ceil_div(n, 4))};
        if (n <= 4096 && e == 4) return {8, round32(ceil_div(n, 8))};
    } else {
        for (int nv : {4, 16})
            if (n <= 32 * nv) return {nv, 32};
        if (n <= 8192) return {16, round32(ceil_div(n, 16))};
    }
    return {0, 0};
}
// Blocks of at most 512 threads, two on an SM, or one where a thread has four accesses.
Shape ring_shape(long long h, int e) {
    const long long n = ceil_div(h, e);
    if (n <= 64 || n > 2048) return {0, 0};
    return n <= 1024 ? Shape{2, round32(ceil_div(n, 2))} : Shape{4, round32(ceil_div(n, 4))};
}
Shape backward_shape(long long h, int e) {
    const long long n = ceil_div(h, e);
    if (e > 1) {
        for (int nv : {1, 2})
            if (n <= 32 * nv) return {nv, 32};
        return ring_shape(h, e);
    } else {
        for (int nv : {4, 16})
            if (n <= 32 * nv) return {nv, 32};
        if (n <= 4096) return {8, round32(ceil_div(n, 8))};
        if (n <= 8192) return {16, round32(ceil_div(n, 16))};
    }
    return {0, 0};
}

// Backward blocks that are resident at once: 1024 threads per SM at 64 registers (512 where a
// thread holds 4 accesses), but 8 rows each where that still fills the SMs, since each block costs
// a row of partial sums.
int row_blocks(long long rows, int threads, int nv, int e) {
    const bool warp = threads == 32;
    const int block = warp ? 32 * kWarpRows : threads;
    const int per_sm = std::max(1, std::min(8, (e > 1 && nv > 2 ? 512 : 1024) / block));
    const long long work = warp ? ceil_div(rows, kWarpRows) : rows;
    return static_cast<int>(std::min(std::min(work, static_cast<long long>(sm_count()) * per_sm),
                                     std::max<long long>(sm_count(), ceil_div(work, 8))));
}

constexpr int kColumnChunks = 64;  // row chunks of norm_columns_kernel at most

template <int D, int WD, int E, int NV, bool LAYER>
cudaError_t forward(const NormForwardArgs& a, int threads, cudaStream_t s) {
    // A row per block (or warp) and no persistent grid: with all SMs' blocks resident the rows in
    // flight hide each other's latency.
    const int grid = static_cast<int>(std::min<long long>(threads == 32 ? ceil_div(a.rows, kWarpRows) : a.rows, 1 << 20));
    if (threads == 32)
        norm_forward_kernel<D, WD, E, NV, LAYER, true><<<grid, dim3(32, kWarpRows), 0, s>>>(a);
    else
        norm_forward_kernel<D, WD, E, NV, LAYER, false><<<grid, threads, 0, s>>>(a);
    return cudaGetLastError();
}

// The deepest ring of 2 to 4 rows that leaves the SM room for `per_sm` blocks (228 KiB; a block takes
// 1 KiB for the system and 512 bytes for its sums besides). Launches f(Int<stages>, bytes).
template <typename F>
cudaError_t with_ring(size_t row, size_t params, int per_sm, F&& f) {
    const size_t room = std::min<size_t>(228 * 1024 / per_sm, 227 * 1024) - 1024 - 512;
    if (params + 4 * row <= room) return f(Int<4>{}, params + 4 * row);
    if (params + 3 * row <= room) return f(Int<3>{}, params + 3 * row);
    return f(Int<2>{}, params + 2 * row);
}

template <int D, int WD, int NV, bool LAYER>
cudaError_t forward_ring(const NormForwardArgs& a, int threads, cudaStream_t s) {
    const int per_sm = std::min(8, (NV > 2 ? 512 : 1024) / threads);
    const int grid = static_cast<int>(std::min<long long>(a.rows, static_cast<long long>(sm_count()) * per_sm));
    const int vectors = (a.w != nullptr) + (a.b != nullptr);
    return with_ring(static_cast<size_t>(NV) * threads * 16, static_cast<size_t>(vectors) * a.h * sizeof(Bits<WD>), per_sm,
                     [&](auto S, size_t smem) {
                         auto* kernel = &norm_forward_ring_kernel<D, WD, NV, LAYER, decltype(S)::value>;
                         const cudaError_t e = cudaFuncSetAttribute(
                             kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
                         if (e != cudaSuccess) return e;
                         kernel<<<grid, threads, smem, s>>>(a);
                         return cudaGetLastError();
                     });
}

template <int D, int WD, int E, bool LAYER>
cudaError_t forward_any(const NormForwardArgs& a, cudaStream_t s) {
    if constexpr (E > 1) {
        const Shape ring = ring_shape(a.h, E);
        static const int mode = getenv("BCCL_X") ? atoi(getenv("BCCL_X")) : 0;
        if (mode < 8 && ring.threads != 0 && a.rows > (mode ? 0 : 2ll * sm_count() * ((ring.nv > 2 ? 512 : 1024) / ring.threads))) {
            if (ring.nv == 2) return forward_ring<D, WD, 2, LAYER>(a, ring.threads, s);
            return forward_ring<D, WD, 4, LAYER>(a, ring.threads, s);
        }
    }
    const Shape sh = forward_shape(a.h, E);
    if constexpr (E > 1) {
        if (sh.nv == 1) return forward<D, WD, E, 1, LAYER>(a, sh.threads, s);
        if (sh.nv == 2) return forward<D, WD, E, 2, LAYER>(a, sh.threads, s);
        if (sh.nv == 4) return forward<D, WD, E, 4, LAYER>(a, sh.threads, s);
        if constexpr (E == 4) {
            if (sh.nv == 8) return forward<D, WD, E, 8, LAYER>(a, sh.threads, s);
        }
    } else {
        if (sh.nv == 4) return forward<D, WD, E, 4, LAYER>(a, sh.threads, s);
        if (sh.nv == 16) return forward<D, WD, E, 16, LAYER>(a, sh.threads, s);
    }
    const int grid = static_cast<int>(std::min<long long>(a.rows, sm_count() * 2));
    norm_forward_long_kernel<D, WD, E, LAYER><<<grid, 1024, 0, s>>>(a);
    return cudaGetLastError();
}

template <int D, int WD, int E, int NV, bool LAYER, bool WARP>
cudaError_t backward(const NormBackwardArgs& a, int threads, int grid, cudaStream_t s) {
    if (WARP)
        norm_backward_kernel<D, WD, E, NV, LAYER, true>
            <<<grid, dim3(32, kWarpRows), sizeof(float) * kWarpRows * a.h, s>>>(a);
    else
        norm_backward_kernel<D, WD, E, NV, LAYER, false><<<grid, threads, 0, s>>>(a);
    return cudaGetLastError();
}

template <int D, int WD, int NV, bool LAYER>
cudaError_t backward_ring(const NormBackwardArgs& a, int threads, int grid, cudaStream_t s) {
    const int per_sm = std::max(1, std::min(static_cast<int>(ceil_div(grid, sm_count())), (NV > 2 ? 512 : 1024) / threads));
    return with_ring(static_cast<size_t>(2) * NV * threads * 16, a.w != nullptr ? a.h * sizeof(Bits<WD>) : 0, per_sm,
                     [&](auto S, size_t smem) {
                         auto* kernel = &norm_backward_ring_kernel<D, WD, NV, LAYER, decltype(S)::value>;
                         const cudaError_t e = cudaFuncSetAttribute(
                             kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
                         if (e != cudaSuccess) return e;
                         kernel<<<grid, threads, smem, s>>>(a);
                         return cudaGetLastError();
                     });
}

// Rows of partial sums that the backward pass of this shape writes.
int partial_rows(long long rows, long long h, int e) {
    const Shape sh = backward_shape(h, e);
    if (sh.threads != 0) return row_blocks(rows, sh.threads, sh.nv, e);
    return static_cast<int>(std::max(1ll, std::min<long long>(ceil_div(rows, 8), kColumnChunks)));
}

template <int D, int WD, int E, bool LAYER>
cudaError_t backward_any(const NormBackwardArgs& a, cudaStream_t s) {
    const Shape sh = backward_shape(a.h, E);
    const int parts = partial_rows(a.rows, a.h, E);
    cudaError_t e = cudaSuccess;
    if (sh.threads != 0) {
        if constexpr (E > 1) {
            if (sh.threads == 32)
                e = sh.nv == 1 ? backward<D, WD, E, 1, LAYER, true>(a, sh.threads, parts, s)
                               : backward<D, WD, E, 2, LAYER, true>(a, sh.threads, parts, s);
            else
                e = sh.nv == 2 ? backward_ring<D, WD, 2, LAYER>(a, sh.threads, parts, s)
                               : backward_ring<D, WD, 4, LAYER>(a, sh.threads, parts, s);
        } else {
            if (sh.threads == 32)
                e = sh.nv == 4 ? backward<D, WD, E, 4, LAYER, true>(a, sh.threads, parts, s)
                               : backward<D, WD, E, 16, LAYER, true>(a, sh.threads, parts, s);
            else
                e = sh.nv == 8 ? backward<D, WD, E, 8, LAYER, false>(a, sh.threads, parts, s)
                               : backward<D, WD, E, 16, LAYER, false>(a, sh.threads, parts, s);
        }
    } else {
        norm_backward_long_kernel<D, WD, E, LAYER>
            <<<static_cast<int>(std::min<long long>(a.rows, sm_count() * 2)), 1024, 0, s>>>(a);
        e = cudaGetLastError();
        if (e == cudaSuccess && a.partials != nullptr) {
            const dim3 grid(static_cast<unsigned>(ceil_div(a.h, 32 * E)), parts);
            norm_columns_kernel<D, E, LAYER><<<grid, dim3(32, 8), 0, s>>>(a);
            e = cudaGetLastError();
        }
    }
    if (e != cudaSuccess || a.partials == nullptr) return e;
    const dim3 grid(static_cast<unsigned>(ceil_div(a.h, 32)), a.db != nullptr ? 2 : 1);
    norm_weights_kernel<WD><<<grid, dim3(32, 32), 0, s>>>(a.partials, parts, a.h, a.dw, a.db);
    return cudaGetLastError();
}

}  // namespace
}  // namespace ops

cudaError_t LaunchNormForward(bool layer, const NormForwardArgs& a, int dtype, int wdtype, cudaStream_t stream) {
    using namespace ops;
    if (a.rows == 0) return cudaSuccess;
    const int size = size_of(dtype);
    const bool wide = rows16(a.x, a.x_stride, a.h, size) && rows16(a.y, a.y_stride, a.h, size) &&
                      (a.w == nullptr || on16(a.w)) && (a.b == nullptr || on16(a.b));
    return with_types(dtype, wdtype, [&](auto D, auto W) {
        constexpr int kD = decltype(D)::value, kW = decltype(W)::value, kE = Vec<kD>::E;
        if (layer)
            return wide ? forward_any<kD, kW, kE, true>(a, stream) : forward_any<kD, kW, 1, true>(a, stream);
        return wide ? forward_any<kD, kW, kE, false>(a, stream) : forward_any<kD, kW, 1, false>(a, stream);
    });
}

size_t NormBackwardWorkspace(bool layer, long long rows, long long h, int dtype) {
    using namespace ops;
    if (rows == 0 || h == 0) return 0;
    // Either width may run, by the alignment of the call's pointers.
    const int parts = std::max(partial_rows(rows, h, 16 / size_of(dtype)), partial_rows(rows, h, 1));
    return sizeof(float) * (layer ? 2 : 1) * static_cast<size_t>(parts) * static_cast<size_t>(h);
}

cudaError_t LaunchNormBackward(bool layer, NormBackwardArgs a, int dtype, int wdtype, cudaStream_t stream) {
    using namespace ops;
    if (a.dw == nullptr && a.db == nullptr) a.partials = nullptr;
    if (a.rows == 0) {  // sums over no rows
        const size_t bytes = static_cast<size_t>(a.h) * size_of(wdtype);
        cudaError_t e = a.dw != nullptr ? cudaMemsetAsync(a.dw, 0, bytes, stream) : cudaSuccess;
        if (e == cudaSuccess && a.db != nullptr) e = cudaMemsetAsync(a.db, 0, bytes, stream);
        return e;
    }
    const int size = size_of(dtype);
    const bool wide = rows16(a.x, a.x_stride, a.h, size) && rows16(a.dy, a.dy_stride, a.h, size) &&
                      rows16(a.dx, a.dx_stride, a.h, size) && (a.w == nullptr || on16(a.w));
    return with_types(dtype, wdtype, [&](auto D, auto W) {
        constexpr int kD = decltype(D)::value, kW = decltype(W)::value, kE = Vec<kD>::E;
        if (layer)
            return wide ? backward_any<kD, kW, kE, true>(a, stream) : backward_any<kD, kW, 1, true>(a, stream);
        return wide ? backward_any<kD, kW, kE, false>(a, stream) : backward_any<kD, kW, 1, false>(a, stream);
    });
}

}  // namespace bccl
