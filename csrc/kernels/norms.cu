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
#include <type_traits>

namespace bccl {
namespace ops {
namespace {

constexpr int kWarpRows = 8;  // rows of a block whose warps work on a row each

// WARP: blockDim = (32, kWarpRows), a row per warp; else blockDim = (g, 1), a row per block. Access v of a
// thread covers columns (v * g + tx) * E - shift and on; accesses of neighbouring threads are adjacent.
template <int D, int WD, int NV, bool LAYER, bool WARP, bool ODD>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 512) norm_forward_kernel(const NormForwardArgs a) {
    constexpr int E = Vec<D>::E;
    __shared__ float buf[2][32];
    const int tx = threadIdx.x, g = blockDim.x, warps = g >> 5, h = static_cast<int>(a.h);
    const long long step = WARP ? static_cast<long long>(gridDim.x) * kWarpRows : gridDim.x;
    long long row = WARP ? static_cast<long long>(blockIdx.x) * kWarpRows + threadIdx.y : blockIdx.x;
    const float inv_h = 1.0f / static_cast<float>(h);
    const Bits<D>* x = static_cast<const Bits<D>*>(a.x);
    const Bits<WD>*weight = static_cast<const Bits<WD>*>(a.w), *bias = static_cast<const Bits<WD>*>(a.b);
    int parity = 0;
    auto sum = [&](float v) {
        if constexpr (WARP) return warp_sum(v);
        const float s = block_sum(v, buf, parity, tx, warps);
        parity ^= 1;
        return s;
    };
    auto out = [&](long long r) { return static_cast<Bits<D>*>(a.y) + r * a.y_stride; };
    Raw<D, E> next[NV];
    auto fetch = [&](long long r) {
        const int c0 = tx * E - shift_of<ODD, D>(out(r));
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = c0 + v * g * E;
            next[v] = c < h && r < a.rows ? get_row<ODD, D>(x + r * a.x_stride, c, h) : zero_raw<D, E>();
        }
    };
    fetch(row);
    for (; row < a.rows; row += step) {
        const int c0 = tx * E - shift_of<ODD, D>(out(row));
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
        if (weight != nullptr) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = c0 + v * g * E;
                if (c < h) get_params<ODD, WD, E>(weight, c, h, w[v]);
            }
        }
        float mean = 0.0f;
        if constexpr (LAYER) {
            mean = sum(s) * inv_h;
            s = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = c0 + v * g * E;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    f[v][e] -= mean;
                    if (c + e < h && (!ODD || c + e >= 0)) s = fmaf(f[v][e], f[v][e], s);
                }
            }
        }
        const float rstd = inv_sqrt(sum(s) * inv_h + a.eps);
        if (tx == 0) {
            if (LAYER) a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = c0 + v * g * E;
            if (c >= h) continue;
            float b[E];
            if (LAYER && bias != nullptr) get_params<ODD, WD, E>(bias, c, h, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                f[v][e] *= rstd;
                if (weight != nullptr) f[v][e] *= w[v][e];
                if (LAYER && bias != nullptr) f[v][e] += b[e];
            }
            put_row<ODD, D, E>(out(row), c, h, f[v]);
        }
    }
}

__device__ __forceinline__ void copy16_async(void* smem, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))),
                 "l"(global)
                 : "memory");
}

// The parameters of E columns from c on in shared memory at `place` (the thread's own, so no barrier),
// and back.
template <bool ODD, int WD, int E>
__device__ __forceinline__ void keep_params(Bits<WD>* place, const Bits<WD>* params, int c, int h) {
    if constexpr (!ODD) {
#pragma unroll
        for (int i = 0; i < E / Vec<WD>::E; ++i)
            reinterpret_cast<uint4*>(place)[i] = __ldg(reinterpret_cast<const uint4*>(params + c) + i);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) place[e] = c + e >= 0 && c + e < h ? __ldg(params + c + e) : 0;
    }
}
template <int WD, int E>
__device__ __forceinline__ void read_params(const Bits<WD>* place, F2 (&w)[E / 2]) {
    constexpr int W = Vec<WD>::E;
#pragma unroll
    for (int i = 0; i < E / W; ++i) {
        F2 t[W / 2];
        unpack2<WD>(reinterpret_cast<const uint4*>(place)[i], t);
#pragma unroll
        for (int e = 0; e < W / 2; ++e) w[i * (W / 2) + e] = t[e];
    }
}
// Zeros where columns [c, c + E) are not the row's: an ODD row's first and last group hold its
// neighbours' elements too.
template <int P>
__device__ __forceinline__ void mask_row(F2 (&a)[P], int c, int h) {
    if (c >= 0 && c + 2 * P <= h) return;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const float2 t = split(a[i]);
        a[i] = f2(c + 2 * i >= 0 && c + 2 * i < h ? t.x : 0.0f, c + 2 * i + 1 >= 0 && c + 2 * i + 1 < h ? t.y : 0.0f);
    }
}
template <bool ODD, int D, int P>
__device__ __forceinline__ void put_row2(Bits<D>* row, int c, int h, const F2 (&a)[P]) {
    if (!ODD || (c >= 0 && c + 2 * P <= h)) {
        __stcs(reinterpret_cast<uint4*>(row + c), pack2<D>(a));
    } else {
        float f[2 * P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float2 t = split(a[i]);
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
        put_row<true, D, 2 * P>(row, c, h, f);
    }
}

// Many rows of 16-byte accesses. ODD: every row of x begins at the same distance from a 16-byte boundary as
// its row of y, and the grid makes a block's rows all begin at the same. Blocks are persistent. Every thread copies its
// own columns of the next STAGES - 1 rows into shared memory with cp.async and only reads what it
// copied itself, so the copies need no barrier and stay in flight whatever the row at hand waits for;
// a row costs one barrier per sum. A thread takes two accesses and 64 registers, so that an SM holds
// 1024 threads (of rows too long for that, four and 128): measured on the backward pass of 8192 x 8192
// bf16, one access per thread took 132 us, two 97, four 96 to 102; f32 rows of 4096 77, 77 and 91.
template <int D> constexpr int ring_max_threads() { return D == kF32 ? 1024 : 512; }

template <int D, int WD, bool LAYER, bool ODD, int STAGES, int NV>
__global__ void __launch_bounds__(ring_max_threads<D>(), NV == 2 && D != kF32 ? 2 : 1) norm_forward_ring_kernel(const NormForwardArgs a) {
    constexpr int E = Vec<D>::E, P = E / 2;
    extern __shared__ uint4 ring[];  // [STAGES][NV][threads], then the weights and biases that there are
    __shared__ float buf[2][32];
    const int tx = threadIdx.x, g = blockDim.x, warps = g >> 5, h = static_cast<int>(a.h);
    const float inv_h = 1.0f / static_cast<float>(h);
    const int shift = shift_of<ODD, D>(static_cast<const Bits<D>*>(a.y) + blockIdx.x * a.y_stride);
    const int c0 = tx * E - shift, dc = g * E;  // columns of access v: c0 + v * dc
    Bits<WD>* w_smem = reinterpret_cast<Bits<WD>*>(ring + STAGES * NV * g) + tx * E;
    Bits<WD>* b_smem = w_smem + (a.w != nullptr ? NV * dc : 0);
    const long long x_step = static_cast<long long>(gridDim.x) * a.x_stride, y_step = static_cast<long long>(gridDim.x) * a.y_stride;
    const Bits<D>* x = static_cast<const Bits<D>*>(a.x) + blockIdx.x * a.x_stride + c0;  // of the next row to copy
    Bits<D>* y = static_cast<Bits<D>*>(a.y) + blockIdx.x * a.y_stride;
    int left = static_cast<int>((a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);  // rows to copy
    int todo = left;
    auto issue = [&](int slot) {
        if (left > 0) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (c0 + v * dc < h) copy16_async(ring + (slot * NV + v) * g + tx, x + v * dc);
            x += x_step;
            --left;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = c0 + v * dc;
        if (c >= h) continue;
        if (a.w != nullptr) keep_params<ODD, WD, E>(w_smem + v * dc, static_cast<const Bits<WD>*>(a.w), c, h);
        if (LAYER && a.b != nullptr) keep_params<ODD, WD, E>(b_smem + v * dc, static_cast<const Bits<WD>*>(a.b), c, h);
    }
    int slot = 0, parity = 0;
    auto sum = [&](F2 v) {
        const float2 t = split(v);
        const float s = block_sum(t.x + t.y, buf, parity, tx, warps);
        parity ^= 1;
        return s;
    };
    for (long long row = blockIdx.x; todo > 0; --todo, row += gridDim.x) {
        issue(slot == 0 ? STAGES - 1 : slot - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        F2 f[NV][P], s = f2(0.0f, 0.0f);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (c0 + v * dc >= h) continue;
            unpack2<D>(ring[(slot * NV + v) * g + tx], f[v]);
            if (ODD) mask_row(f[v], c0 + v * dc, h);
#pragma unroll
            for (int e = 0; e < P; ++e) s = LAYER ? add2(f[v][e], s) : fma2(f[v][e], f[v][e], s);
        }
        float mean = 0.0f;
        if constexpr (LAYER) {
            mean = sum(s) * inv_h;
            const F2 minus = f2(-mean, -mean);
            s = f2(0.0f, 0.0f);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (c0 + v * dc >= h) continue;
#pragma unroll
                for (int e = 0; e < P; ++e) f[v][e] = add2(f[v][e], minus);
                if (ODD) mask_row(f[v], c0 + v * dc, h);
#pragma unroll
                for (int e = 0; e < P; ++e) s = fma2(f[v][e], f[v][e], s);
            }
        }
        const float rstd = inv_sqrt(sum(s) * inv_h + a.eps);
        if (tx == 0) {
            if (LAYER) a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        const F2 scale = f2(rstd, rstd);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = c0 + v * dc;
            if (c >= h) continue;
            F2 w[P];
#pragma unroll
            for (int e = 0; e < P; ++e) f[v][e] = mul2(f[v][e], scale);
            if (a.w != nullptr) {
                read_params<WD, E>(w_smem + v * dc, w);
                if (LAYER && a.b != nullptr) {
                    F2 b[P];
                    read_params<WD, E>(b_smem + v * dc, b);
#pragma unroll
                    for (int e = 0; e < P; ++e) f[v][e] = fma2(f[v][e], w[e], b[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < P; ++e) f[v][e] = mul2(f[v][e], w[e]);
                }
            } else if (LAYER && a.b != nullptr) {
                read_params<WD, E>(b_smem + v * dc, w);
#pragma unroll
                for (int e = 0; e < P; ++e) f[v][e] = add2(f[v][e], w[e]);
            }
            put_row2<ODD, D>(y, c, h, f[v]);
        }
        y += y_step;
        slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
}

// Rows longer than a block's registers hold: three passes over the row, the later ones from L2.
template <int D, int WD, bool LAYER, bool ODD>
__global__ void __launch_bounds__(1024) norm_forward_long_kernel(const NormForwardArgs a) {
    constexpr int E = Vec<D>::E;
    __shared__ float buf[2][32];
    const int tx = threadIdx.x, step = blockDim.x * E, h = static_cast<int>(a.h);
    const float inv_h = 1.0f / static_cast<float>(h);
    const Bits<WD>*weight = static_cast<const Bits<WD>*>(a.w), *bias = static_cast<const Bits<WD>*>(a.b);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Bits<D>* x = static_cast<const Bits<D>*>(a.x) + row * a.x_stride;
        Bits<D>* y = static_cast<Bits<D>*>(a.y) + row * a.y_stride;
        const int c0 = tx * E - shift_of<ODD, D>(y);
        float mean = 0.0f;
        if constexpr (LAYER) {
            float s = 0.0f;
            for (int c = c0; c < h; c += step) {
                float f[E];
                unpack<D, E>(get_row<ODD, D>(x, c, h), f);
#pragma unroll
                for (int e = 0; e < E; ++e) s += f[e];
            }
            mean = block_sum(s, buf, 0, tx, blockDim.x >> 5) * inv_h;
        }
        float s = 0.0f;
        for (int c = c0; c < h; c += step) {
            float f[E];
            unpack<D, E>(get_row<ODD, D>(x, c, h), f);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (!ODD || (c + e >= 0 && c + e < h)) s = fmaf(f[e] - mean, f[e] - mean, s);
        }
        const float rstd = inv_sqrt(block_sum(s, buf, 1, tx, blockDim.x >> 5) * inv_h + a.eps);
        __syncthreads();  // RMS norm sums once per row: its buffer is free only now
        if (tx == 0) {
            if (LAYER) a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        for (int c = c0; c < h; c += step) {
            float f[E], w[E], b[E];
            unpack<D, E>(get_row<ODD, D>(x, c, h), f);
            if (weight != nullptr) get_params<ODD, WD, E>(weight, c, h, w);
            if (LAYER && bias != nullptr) get_params<ODD, WD, E>(bias, c, h, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                f[e] = (f[e] - mean) * rstd;
                if (weight != nullptr) f[e] *= w[e];
                if (LAYER && bias != nullptr) f[e] += b[e];
            }
            put_row<ODD, D, E>(y, c, h, f);
        }
    }
}

// Rows of 16-byte accesses short enough for a warp, and ODD rows. ODD: the caller's grid makes a block's (or
// warp's) rows all begin at the same shift, so that a thread's columns stay the same.
template <int D, int WD, int NV, bool LAYER, bool WARP, bool ODD>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 512) norm_backward_kernel(const NormBackwardArgs a) {
    constexpr int E = Vec<D>::E;
    extern __shared__ float rows_sum[];  // WARP: one row of partial sums per warp
    __shared__ float2 buf[2][32];
    const int tx = threadIdx.x, g = blockDim.x, warps = g >> 5, h = static_cast<int>(a.h);
    const long long step = WARP ? static_cast<long long>(gridDim.x) * kWarpRows : gridDim.x;
    long long row = WARP ? static_cast<long long>(blockIdx.x) * kWarpRows + threadIdx.y : blockIdx.x;
    const float inv_h = 1.0f / static_cast<float>(h);
    const Bits<D>*x = static_cast<const Bits<D>*>(a.x), *dy = static_cast<const Bits<D>*>(a.dy);
    const Bits<WD>* weight = static_cast<const Bits<WD>*>(a.w);
    const int c0 = tx * E - shift_of<ODD, D>(static_cast<const Bits<D>*>(a.dx) + row * a.dx_stride);
    int parity = 0;
    float dw[NV][E], db[LAYER ? NV : 1][E];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dw[v][e] = 0.0f;
            if constexpr (LAYER) db[v][e] = 0.0f;
        }
    Raw<D, E> nx[NV], ny[NV];
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto fetch = [&](long long r) {
        if (r < a.rows) {
            if (LAYER) next_mean = __ldg(a.mean + r);
            next_rstd = __ldg(a.rstd + r);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = c0 + v * g * E;
            const bool in = c < h && r < a.rows;
            nx[v] = in ? get_row<ODD, D>(x + r * a.x_stride, c, h) : zero_raw<D, E>();
            ny[v] = in ? get_row<ODD, D>(dy + r * a.dy_stride, c, h) : zero_raw<D, E>();
        }
    };
    fetch(row);
    for (; row < a.rows; row += step) {
        const float mean = next_mean, rstd = next_rstd;
        float xh[NV][E], gr[NV][E];
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = c0 + v * g * E;
            unpack<D, E>(nx[v], xh[v]);
            unpack<D, E>(ny[v], gr[v]);
            if (c >= h) continue;
            float w[E];
            if (weight != nullptr) get_params<ODD, WD, E>(weight, c, h, w);
#pragma unroll
            for (int e = 0; e < E; ++e) {  // outside the row dy is zero
                xh[v][e] = (xh[v][e] - mean) * rstd;
                dw[v][e] = fmaf(gr[v][e], xh[v][e], dw[v][e]);
                if constexpr (LAYER) db[v][e] += gr[v][e];
                if (weight != nullptr) gr[v][e] *= w[e];
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
            const int c = c0 + v * g * E;
            if (c >= h) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) gr[v][e] = rstd * (gr[v][e] - m1 - xh[v][e] * m2);
            put_row<ODD, D, E>(dx, c, h, gr[v]);
        }
    }
    if (a.partials == nullptr) return;
    // partials: [blocks][h] of dw, then of db.
    float* pw = a.partials + blockIdx.x * a.h;
    float* pb = a.partials + (static_cast<long long>(gridDim.x) + blockIdx.x) * a.h;
    auto put = [&](float* to, float (&sum)[NV][E]) {
        float* mine = WARP ? rows_sum + threadIdx.y * h : to;
        if (WARP) __syncthreads();
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = c0 + v * g * E + e;
                if (c < h && (!ODD || c >= 0)) mine[c] = sum[v][e];
            }
        if constexpr (WARP) {
            __syncthreads();
            for (int c = threadIdx.y * 32 + tx; c < h; c += 32 * kWarpRows) {
                float t = 0.0f;
#pragma unroll
                for (int r = 0; r < kWarpRows; ++r) t += rows_sum[r * h + c];
                to[c] = t;
            }
        }
    };
    if (a.dw != nullptr) put(pw, dw);
    if constexpr (LAYER) {
        if (a.db != nullptr) put(pb, db);
    }
}

// As norm_forward_ring_kernel, with x and dy in the ring. With g = dy * w:
//   sums g and g * (x - mean);  dx = rstd * (g - m1) - (x - mean) * (rstd^2 * m2),  m2 = mean(g (x - mean)) * rstd
// The second use of a row reads it from shared memory again; RMS norm, which has registers left where
// layer norm adds up db, keeps g (8192 x 8192 bf16: 81 us, 86 without; floor 61). Pairs of floats share an
// instruction: issuing them fills 70% of the slots, the rest waits for the barrier and shared memory.
template <int D, int WD, bool LAYER, bool ODD, int STAGES, int NV>
__global__ void __launch_bounds__(ring_max_threads<D>(), NV == 2 && D != kF32 ? 2 : 1) norm_backward_ring_kernel(const NormBackwardArgs a) {
    constexpr int E = Vec<D>::E, P = E / 2;
    using Sum = typename std::conditional<LAYER, float2, float>::type;
    extern __shared__ uint4 ring[];  // [STAGES][x, dy][NV][threads], then the weights
    __shared__ Sum buf[2][32];
    const int tx = threadIdx.x, g = blockDim.x, warps = g >> 5, h = static_cast<int>(a.h);
    const float inv_h = 1.0f / static_cast<float>(h);
    const int shift = shift_of<ODD, D>(static_cast<const Bits<D>*>(a.dx) + blockIdx.x * a.dx_stride);
    const int c0 = tx * E - shift, dc = g * E;
    Bits<WD>* w_smem = reinterpret_cast<Bits<WD>*>(ring + STAGES * 2 * NV * g) + tx * E;
    const Bits<D>* x = static_cast<const Bits<D>*>(a.x) + blockIdx.x * a.x_stride + c0;  // of the next row to copy
    const Bits<D>* dy = static_cast<const Bits<D>*>(a.dy) + blockIdx.x * a.dy_stride + c0;
    Bits<D>* dx = static_cast<Bits<D>*>(a.dx) + blockIdx.x * a.dx_stride;
    int left = static_cast<int>((a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);  // rows to copy
    int todo = left;
    auto issue = [&](int slot) {
        if (left > 0) {
            uint4* to = ring + slot * 2 * NV * g + tx;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (c0 + v * dc < h) {
                    copy16_async(to + v * g, x + v * dc);
                    copy16_async(to + (NV + v) * g, dy + v * dc);
                }
            }
            x += gridDim.x * a.x_stride;
            dy += gridDim.x * a.dy_stride;
            --left;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s);
    const F2 zero = f2(0.0f, 0.0f);
    F2 dw[NV][P], db[LAYER ? NV : 1][P];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = c0 + v * dc;
        if (a.w != nullptr && c < h) keep_params<ODD, WD, E>(w_smem + v * dc, static_cast<const Bits<WD>*>(a.w), c, h);
#pragma unroll
        for (int e = 0; e < P; ++e) {
            dw[v][e] = zero;
            if constexpr (LAYER) db[v][e] = zero;
        }
    }
    int slot = 0, parity = 0;
    float next_mean = LAYER ? __ldg(a.mean + blockIdx.x) : 0.0f, next_rstd = __ldg(a.rstd + blockIdx.x);
    for (long long row = blockIdx.x; todo > 0; --todo) {
        issue(slot == 0 ? STAGES - 1 : slot - 1);
        const float mean = next_mean, rstd = next_rstd;
        row += gridDim.x;
        if (todo > 1) {  // a row ahead, like the row itself
            if (LAYER) next_mean = __ldg(a.mean + row);
            next_rstd = __ldg(a.rstd + row);
        }
        const F2 scale = f2(rstd, rstd), minus = f2(-mean, -mean);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        const uint4* from = ring + slot * 2 * NV * g + tx;
        F2 s1 = zero, s2 = zero, gw[LAYER ? 1 : NV][P];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (c0 + v * dc >= h) continue;
            F2 xc[P], gr[P], w[P];
            unpack2<D>(from[v * g], xc);
            unpack2<D>(from[(NV + v) * g], gr);
            if (ODD) {
                mask_row(xc, c0 + v * dc, h);
                mask_row(gr, c0 + v * dc, h);
            }
            if (a.w != nullptr) read_params<WD, E>(w_smem + v * dc, w);
#pragma unroll
            for (int e = 0; e < P; ++e) {  // outside the row gr is zero
                if (LAYER) xc[e] = add2(xc[e], minus);
                dw[v][e] = fma2(gr[e], mul2(xc[e], scale), dw[v][e]);
                if constexpr (LAYER) db[v][e] = add2(gr[e], db[v][e]);
                if (a.w != nullptr) gr[e] = mul2(gr[e], w[e]);
                if (LAYER) s1 = add2(gr[e], s1);
                else gw[v][e] = gr[e];
                s2 = fma2(gr[e], xc[e], s2);
            }
        }
        float m1 = 0.0f, m2;
        const float2 t2 = split(s2);
        if constexpr (LAYER) {
            const float2 t1 = split(s1);
            const float2 t = block_sum(make_float2(t1.x + t1.y, t2.x + t2.y), buf, parity, tx, warps);
            m1 = t.x * inv_h;
            m2 = t.y * inv_h * rstd;
        } else {
            m2 = block_sum(t2.x + t2.y, buf, parity, tx, warps) * inv_h * rstd;
        }
        parity ^= 1;
        const float k1 = -m1 * rstd, k2 = -m2 * rstd * rstd;
        const F2 c1 = f2(k1, k1), c2 = f2(k2, k2);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (c0 + v * dc >= h) continue;
            F2 xc[P], gr[P], w[P];
            unpack2<D>(from[v * g], xc);
            if constexpr (LAYER) {
                unpack2<D>(from[(NV + v) * g], gr);
                if (a.w != nullptr) read_params<WD, E>(w_smem + v * dc, w);
            }
#pragma unroll
            for (int e = 0; e < P; ++e) {
                if constexpr (LAYER) {
                    xc[e] = add2(xc[e], minus);
                    if (a.w != nullptr) gr[e] = mul2(gr[e], w[e]);
                    gr[e] = fma2(gr[e], scale, c1);
                } else {
                    gr[e] = mul2(gw[v][e], scale);
                }
                gr[e] = fma2(xc[e], c2, gr[e]);
            }
            put_row2<ODD, D>(dx, c0 + v * dc, h, gr);
        }
        dx += gridDim.x * a.dx_stride;
        slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
    if (a.partials == nullptr) return;
    float* pw = a.partials + blockIdx.x * a.h;
    float* pb = a.partials + (static_cast<long long>(gridDim.x) + blockIdx.x) * a.h;
    auto put = [&](float* to, int c, const F2 (&sum)[P]) {
#pragma unroll
        for (int e = 0; e < P; e += 2) {
            const float2 lo = split(sum[e]), hi = split(sum[e + 1]);
            const float f[4] = {lo.x, lo.y, hi.x, hi.y};
            if constexpr (!ODD) {
                *reinterpret_cast<float4*>(to + c + 2 * e) = make_float4(f[0], f[1], f[2], f[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = c + 2 * e + i;
                    if (k >= 0 && k < h) to[k] = f[i];
                }
            }
        }
    };
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = c0 + v * dc;
        if (c >= h) continue;
        if (a.dw != nullptr) put(pw, c, dw[v]);
        if constexpr (LAYER) {
            if (a.db != nullptr) put(pb, c, db[v]);
        }
    }
}

// Rows longer than a block's registers hold: dx in two passes over the row, and dw / db by a
// second kernel that reads x and dy again by columns.
template <int D, int WD, bool LAYER, bool ODD>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(const NormBackwardArgs a) {
    constexpr int E = Vec<D>::E;
    __shared__ float2 buf[2][32];
    const int tx = threadIdx.x, step = blockDim.x * E, h = static_cast<int>(a.h);
    const float inv_h = 1.0f / static_cast<float>(h);
    const Bits<WD>* weight = static_cast<const Bits<WD>*>(a.w);
    int parity = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
        const Bits<D>* x = static_cast<const Bits<D>*>(a.x) + row * a.x_stride;
        const Bits<D>* dy = static_cast<const Bits<D>*>(a.dy) + row * a.dy_stride;
        Bits<D>* dx = static_cast<Bits<D>*>(a.dx) + row * a.dx_stride;
        const int c0 = tx * E - shift_of<ODD, D>(dx);
        const float mean = LAYER ? __ldg(a.mean + row) : 0.0f;
        const float rstd = __ldg(a.rstd + row);
        float2 s = make_float2(0.0f, 0.0f);
        auto load = [&](int c, float (&xh)[E], float (&gr)[E]) {
            float w[E];
            unpack<D, E>(get_row<ODD, D>(x, c, h), xh);
            unpack<D, E>(get_row<ODD, D>(dy, c, h), gr);
            if (weight != nullptr) get_params<ODD, WD, E>(weight, c, h, w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[e] = (xh[e] - mean) * rstd;
                if (weight != nullptr) gr[e] *= w[e];
            }
        };
        for (int c = c0; c < h; c += step) {
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
        for (int c = c0; c < h; c += step) {
            float xh[E], gr[E];
            load(c, xh, gr);
#pragma unroll
            for (int e = 0; e < E; ++e) gr[e] = rstd * (gr[e] - m1 - xh[e] * m2);
            put_row<ODD, D, E>(dx, c, h, gr);
        }
    }
}

template <int D, bool LAYER, bool ODD>
__global__ void __launch_bounds__(256) norm_columns_kernel(const NormBackwardArgs a) {
    constexpr int E = Vec<D>::E;
    __shared__ float part[8][32 * E];
    const int c = (blockIdx.x * 32 + threadIdx.x) * E, h = static_cast<int>(a.h);
    float dw[E] = {}, db[E] = {};
    if (c < h) {
        for (long long row = static_cast<long long>(blockIdx.y) * 8 + threadIdx.y; row < a.rows;
             row += static_cast<long long>(gridDim.y) * 8) {
            float x[E], dy[E];
            unpack<D, E>(get_row<ODD, D>(static_cast<const Bits<D>*>(a.x) + row * a.x_stride, c, h), x);
            unpack<D, E>(get_row<ODD, D>(static_cast<const Bits<D>*>(a.dy) + row * a.dy_stride, c, h), dy);
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
            const int col = blockIdx.x * 32 * E + i;
            if (col >= h) continue;
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

// How a row is spread: accesses per thread and threads per row (32: a warp). Zero threads: too long
// for registers. More accesses per thread mean fewer warps to synchronise per row, fewer accesses more
// rows in flight.
struct Shape {
    int nv, threads;
};
Shape forward_shape(long long n) {  // n accesses
    for (int nv : {1, 2, 4})
        if (n <= 32 * nv) return {nv, 32};
    if (n <= 512) return {1, round32(n)};
    if (n <= 1024) return {2, round32(ceil_div(n, 2))};
    if (n <= 2048) return {4, round32(ceil_div(n, 4))};
    return {0, 0};
}
Shape backward_shape(long long n, int e) {
    for (int nv : {1, 2})
        if (n <= 32 * nv) return {nv, 32};
    if (n <= 512) return {1, round32(n)};
    if (n <= 1024) return {2, round32(ceil_div(n, 2))};
    if (n <= 2048 && e == 4) return {4, round32(ceil_div(n, 4))};
    return {0, 0};
}

// Accesses per thread of the ring kernels: 0 where a row is short enough for a warp's registers, or
// so long that two rows of x and dy and the weights do not fit in shared memory.
int ring_accesses(long long h, int e, bool odd) {
    const long long n = odd ? accesses<true>(h, e) : accesses<false>(h, e);
    const int most = e == 4 ? 1024 : 512;
    if (n <= (odd ? 16 : 64)) return 0;
    return n <= 2 * most ? 2 : n <= 4 * most && e != 4 ? 4 : 0;
}
int ring_threads(long long h, int e, int nv, bool odd) {
    return round32(ceil_div(odd ? accesses<true>(h, e) : accesses<false>(h, e), nv));
}
int ring_blocks(int threads, int nv) { return std::min(24, std::max(1, (nv == 2 ? 1024 : 512) / threads)); }

// The deepest ring of 2 to 4 rows that leaves the SM room for `per_sm` blocks (228 KiB; a block takes
// 1 KiB for the system and 512 bytes for its sums besides). Launches f(Int<stages>, bytes).
constexpr size_t kMostRing = 227 * 1024 - 1024 - 512;
template <typename F>
cudaError_t with_ring(size_t row, size_t params, int per_sm, F&& f) {
    const size_t room = std::min<size_t>(228 * 1024 / per_sm - 1024 - 512, kMostRing);
    if (params + 4 * row <= room) return f(Int<4>{}, params + 4 * row);
    if (params + 3 * row <= room) return f(Int<3>{}, params + 3 * row);
    return f(Int<2>{}, params + 2 * row);
}
// The limit belongs to the kernel on the device, not to a launch: every call sets the same one, so that calls
// of other widths, in other threads or captured before, never find it below what they launch with.
template <typename K> cudaError_t allow_ring(K* kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostRing));
}

// Backward blocks: what is resident at once, but 4 rows each where that still fills the SMs, since
// each block costs a row of partial sums. More than a row each: a multiple of 8 blocks, so that a block's
// rows begin at one alignment (16 bytes are at most 8 elements).
int row_blocks(long long rows, int rows_per_block, int per_sm) {
    const long long work = ceil_div(rows, rows_per_block);
    const long long most = std::min(static_cast<long long>(sm_count()) * per_sm,
                                    std::max<long long>(sm_count(), ceil_div(work, 4)));
    return static_cast<int>(work <= most ? work : std::max(8ll, most / 8 * 8));
}
// Rows of partial sums that the backward pass writes, a row per block.
constexpr int kColumnChunks = 64;  // row chunks of norm_columns_kernel at most
int ring_grid(long long rows, long long h, int e, int nv, bool odd) {
    return row_blocks(rows, 1, ring_blocks(ring_threads(h, e, nv, odd), nv));
}
int partial_rows(long long rows, long long h, int e, bool odd, bool ring) {
    const int nv = ring ? ring_accesses(h, e, odd) : 0;
    if (nv != 0) return ring_grid(rows, h, e, nv, odd);
    const Shape sh = backward_shape(odd ? accesses<true>(h, e) : accesses<false>(h, e), e);
    if (sh.threads == 32) return row_blocks(rows, kWarpRows, 1024 / (32 * kWarpRows));
    if (sh.threads != 0) return row_blocks(rows, 1, std::max(1, std::min(8, (sh.nv == 1 ? 1024 : 512) / sh.threads)));
    return static_cast<int>(std::max(1ll, std::min<long long>(ceil_div(rows, 8), kColumnChunks)));
}

template <int D, int WD, int NV, bool LAYER, bool ODD>
cudaError_t forward(const NormForwardArgs& a, int threads, cudaStream_t s) {
    // A row per block (or warp) and no persistent grid: the rows in flight hide each other's latency.
    const int grid = static_cast<int>(std::min<long long>(threads == 32 ? ceil_div(a.rows, kWarpRows) : a.rows, 1 << 20));
    if (threads == 32)
        norm_forward_kernel<D, WD, NV, LAYER, true, ODD><<<grid, dim3(32, kWarpRows), 0, s>>>(a);
    else
        norm_forward_kernel<D, WD, NV, LAYER, false, ODD><<<grid, threads, 0, s>>>(a);
    return cudaGetLastError();
}

template <int D, int WD, bool LAYER, bool ODD, int NV>
cudaError_t forward_ring(const NormForwardArgs& a, cudaStream_t s) {
    constexpr int E = Vec<D>::E;
    const int threads = ring_threads(a.h, E, NV, ODD), per_sm = ring_blocks(threads, NV);
    const long long most = static_cast<long long>(sm_count()) * per_sm;
    const int grid = static_cast<int>(a.rows <= most ? a.rows : most / 8 * 8);  // one alignment per block
    const int vectors = (a.w != nullptr) + (a.b != nullptr);
    return with_ring(static_cast<size_t>(NV) * 16 * threads,
                     static_cast<size_t>(vectors) * NV * threads * E * sizeof(Bits<WD>), per_sm, [&](auto S, size_t smem) {
                         auto* kernel = &norm_forward_ring_kernel<D, WD, LAYER, ODD, decltype(S)::value, NV>;
                         const cudaError_t e = allow_ring(kernel);
                         if (e != cudaSuccess) return e;
                         kernel<<<grid, threads, smem, s>>>(a);
                         return cudaGetLastError();
                     });
}

// Two arrays of rows whose rows lie at the same distance from 16-byte boundaries.
bool congruent(const void* p, long long p_stride, const void* q, long long q_stride, int size) {
    return ((reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(q)) & 15) == 0 &&
           (p_stride - q_stride) * size % 16 == 0;
}

template <int D, int WD, bool LAYER, bool ODD>
cudaError_t forward_any(const NormForwardArgs& a, cudaStream_t s) {
    constexpr int E = Vec<D>::E;
    // Blocks that walk several rows: below that a row per block fills the SMs sooner.
    const int nv = !ODD || congruent(a.x, a.x_stride, a.y, a.y_stride, sizeof(Bits<D>)) ? ring_accesses(a.h, E, ODD) : 0;
    if (nv != 0 && a.rows > static_cast<long long>(sm_count()) * ring_blocks(ring_threads(a.h, E, nv, ODD), nv)) {
        if (nv == 2) return forward_ring<D, WD, LAYER, ODD, 2>(a, s);
        if constexpr (E == 8) return forward_ring<D, WD, LAYER, ODD, 4>(a, s);
    }
    const Shape sh = forward_shape(accesses<ODD>(a.h, E));
    if (sh.nv == 1) return forward<D, WD, 1, LAYER, ODD>(a, sh.threads, s);
    if (sh.nv == 2) return forward<D, WD, 2, LAYER, ODD>(a, sh.threads, s);
    if (sh.nv == 4) return forward<D, WD, 4, LAYER, ODD>(a, sh.threads, s);
    const int grid = static_cast<int>(std::min<long long>(a.rows, sm_count() * 2));
    norm_forward_long_kernel<D, WD, LAYER, ODD><<<grid, 1024, 0, s>>>(a);
    return cudaGetLastError();
}

template <int D, int WD, int NV, bool LAYER, bool ODD>
cudaError_t backward(const NormBackwardArgs& a, int threads, int grid, cudaStream_t s) {
    if (threads == 32) {
        if constexpr (NV <= 2)
            norm_backward_kernel<D, WD, NV, LAYER, true, ODD>
                <<<grid, dim3(32, kWarpRows), sizeof(float) * kWarpRows * a.h, s>>>(a);
    } else if constexpr (ODD) {
        norm_backward_kernel<D, WD, NV, LAYER, false, true><<<grid, threads, 0, s>>>(a);
    }
    return cudaGetLastError();
}

template <int D, int WD, bool LAYER, bool ODD, int NV>
cudaError_t backward_ring(const NormBackwardArgs& a, int grid, cudaStream_t s) {
    constexpr int E = Vec<D>::E;
    const int threads = ring_threads(a.h, E, NV, ODD);
    const int per_sm = std::max(1, std::min(static_cast<int>(ceil_div(grid, sm_count())), ring_blocks(threads, NV)));
    return with_ring(static_cast<size_t>(2) * NV * 16 * threads,
                     a.w != nullptr ? static_cast<size_t>(NV) * threads * E * sizeof(Bits<WD>) : 0, per_sm,
                     [&](auto S, size_t smem) {
                         auto* kernel = &norm_backward_ring_kernel<D, WD, LAYER, ODD, decltype(S)::value, NV>;
                         const cudaError_t e = allow_ring(kernel);
                         if (e != cudaSuccess) return e;
                         kernel<<<grid, threads, smem, s>>>(a);
                         return cudaGetLastError();
                     });
}

template <int D, int WD, bool LAYER, bool ODD>
cudaError_t backward_any(const NormBackwardArgs& a, cudaStream_t s) {
    constexpr int E = Vec<D>::E, kSize = sizeof(Bits<D>);
    const bool by_ring = !ODD || (congruent(a.x, a.x_stride, a.dx, a.dx_stride, kSize) &&
                                  congruent(a.dy, a.dy_stride, a.dx, a.dx_stride, kSize));
    const Shape sh = backward_shape(accesses<ODD>(a.h, E), E);
    const int parts = partial_rows(a.rows, a.h, E, ODD, by_ring);
    const int ring = by_ring ? ring_accesses(a.h, E, ODD) : 0;
    cudaError_t e = cudaSuccess;
    if (ring != 0) {
        if constexpr (E == 8)
            e = ring == 2 ? backward_ring<D, WD, LAYER, ODD, 2>(a, parts, s) : backward_ring<D, WD, LAYER, ODD, 4>(a, parts, s);
        else
            e = backward_ring<D, WD, LAYER, ODD, 2>(a, parts, s);
    } else if (sh.nv == 1) {
        e = backward<D, WD, 1, LAYER, ODD>(a, sh.threads, parts, s);
    } else if (sh.nv == 2) {
        e = backward<D, WD, 2, LAYER, ODD>(a, sh.threads, parts, s);
    } else if (sh.nv == 4) {
        if constexpr (E == 4) e = backward<D, WD, 4, LAYER, ODD>(a, sh.threads, parts, s);
    } else {
        norm_backward_long_kernel<D, WD, LAYER, ODD>
            <<<static_cast<int>(std::min<long long>(a.rows, sm_count() * 2)), 1024, 0, s>>>(a);
        e = cudaGetLastError();
        if (e == cudaSuccess && a.partials != nullptr) {
            const dim3 grid(static_cast<unsigned>(ceil_div(a.h, 32 * E)), parts);
            norm_columns_kernel<D, LAYER, ODD><<<grid, dim3(32, 8), 0, s>>>(a);
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
    const bool odd = !rows16(a.x, a.x_stride, a.h, size) || !rows16(a.y, a.y_stride, a.h, size) || !on16(a.w) || !on16(a.b);
    return with_types(dtype, wdtype, [&](auto D, auto W) {
        constexpr int kD = decltype(D)::value, kW = decltype(W)::value;
        if (layer) return odd ? forward_any<kD, kW, true, true>(a, stream) : forward_any<kD, kW, true, false>(a, stream);
        return odd ? forward_any<kD, kW, false, true>(a, stream) : forward_any<kD, kW, false, false>(a, stream);
    });
}

size_t NormBackwardWorkspace(bool layer, long long rows, long long h, int dtype) {
    using namespace ops;
    if (rows == 0 || h == 0) return 0;
    // Either form may run, by the alignment of the call's pointers.
    const int e = 16 / size_of(dtype);
    const int parts = std::max({partial_rows(rows, h, e, false, true), partial_rows(rows, h, e, true, true),
                                partial_rows(rows, h, e, true, false)});
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
    const bool odd = !rows16(a.x, a.x_stride, a.h, size) || !rows16(a.dy, a.dy_stride, a.h, size) ||
                     !rows16(a.dx, a.dx_stride, a.h, size) || !on16(a.w);
    return with_types(dtype, wdtype, [&](auto D, auto W) {
        constexpr int kD = decltype(D)::value, kW = decltype(W)::value;
        if (layer) return odd ? backward_any<kD, kW, true, true>(a, stream) : backward_any<kD, kW, true, false>(a, stream);
        return odd ? backward_any<kD, kW, false, true>(a, stream) : backward_any<kD, kW, false, false>(a, stream);
    });
}

}  // namespace bccl
