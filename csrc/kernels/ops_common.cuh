// Shared by the compute operators (grad_norm.cu, norms.cu, embedding.cu, experts.cu): loads and
// stores of E adjacent elements as floats, reductions over a block, launch helpers.
//
// Kernels access E elements that fill 16 bytes. Where every row starts on a 16-byte boundary (base
// pointers and row strides) an access covers the columns from a multiple of E on. For all other layouts
// each kernel has an ODD form: accesses start on the 16-byte boundaries of the row that is written,
// `shift` columns before multiples of E; a row read at another alignment is put together from two
// 16-byte groups, and the first and last access of a row go element by element. (Element accesses
// throughout were bound by issuing loads: RMS norm of 16384 x 4097 bf16 took 301 us instead of 59.)
#pragma once

#include "kernels/common.cuh"

#include <algorithm>
#include <climits>

namespace bccl {
namespace ops {

using dev::kBF16;
using dev::kF16;
using dev::kF32;
using dev::Ty;
using dev::Vec;

template <int D> using Bits = typename Ty<D>::Bits;

// What one access of E elements holds before conversion (kept in registers for prefetching).
template <int D, int E> struct Raw {
    static_assert(E == Vec<D>::E, "16 bytes");
    uint4 v;
};

template <int D, int E>
__device__ __forceinline__ Raw<D, E> load_raw(const Bits<D>* p) {
    return {__ldg(reinterpret_cast<const uint4*>(p))};
}
template <int D, int E>
__device__ __forceinline__ void unpack(const Raw<D, E>& r, float (&a)[E]) {
    Vec<D>::unpack(r.v, a);
}
template <int D, int E>
__device__ __forceinline__ Raw<D, E> zero_raw() {
    return {make_uint4(0, 0, 0, 0)};
}

// E elements of a (possibly wider) type: vectors of parameters next to 16-bit activations.
template <int D, int E>
__device__ __forceinline__ void load_f(const Bits<D>* p, float (&a)[E]) {
    constexpr int W = Vec<D>::E;
    static_assert(E % W == 0, "whole 16-byte accesses");
#pragma unroll
    for (int i = 0; i < E / W; ++i) {
        float t[W];
        Vec<D>::unpack(__ldg(reinterpret_cast<const uint4*>(p) + i), t);
#pragma unroll
        for (int e = 0; e < W; ++e) a[i * W + e] = t[e];
    }
}
template <int D, int E>
__device__ __forceinline__ void store_f(Bits<D>* p, const float (&a)[E]) {
    constexpr int W = Vec<D>::E;
    static_assert(E % W == 0, "whole 16-byte accesses");
#pragma unroll
    for (int i = 0; i < E / W; ++i) {
        float t[W];
#pragma unroll
        for (int e = 0; e < W; ++e) t[e] = a[i * W + e];
        *(reinterpret_cast<uint4*>(p) + i) = Vec<D>::pack(t);
    }
}
// Streaming stores for outputs far larger than what is read again soon.
template <int D, int E>
__device__ __forceinline__ void store_f_cs(Bits<D>* p, const float (&a)[E]) {
    constexpr int W = Vec<D>::E;
    static_assert(E % W == 0, "whole 16-byte accesses");
#pragma unroll
    for (int i = 0; i < E / W; ++i) {
        float t[W];
#pragma unroll
        for (int e = 0; e < W; ++e) t[e] = a[i * W + e];
        __stcs(reinterpret_cast<uint4*>(p) + i, Vec<D>::pack(t));
    }
}
template <int D, int E>
__device__ __forceinline__ void store_raw_cs(Bits<D>* p, const Raw<D, E>& r) {
    __stcs(reinterpret_cast<uint4*>(p), r.v);
}

// ---------------------------------------------------------------- rows of any alignment
// 16 bytes from any element boundary are put together from the one or two 16-byte groups that hold them
// (and so lie in the allocation that holds the row, whatever comes before and behind it).
template <int D>
__device__ __forceinline__ uint4 join_groups(const Bits<D>* p, const uint4& lo, const uint4& hi) {
    const unsigned int k = reinterpret_cast<uintptr_t>(p) & 15;
    unsigned int w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (k & 4) {
#pragma unroll
        for (int i = 0; i < 7; ++i) w[i] = w[i + 1];
    }
    if (k & 8) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 2];
    }
    const unsigned int bits = (k & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}
// Columns by which the row's first access starts before its first element.
template <bool ODD, int D>
__device__ __forceinline__ int shift_of(const Bits<D>* row) {
    return ODD ? static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(Bits<D>)) : 0;
}
// Columns [c, c + E) of a row of h; zeros outside it, and everywhere unless `in`. Not ODD: c is a multiple of
// E, below h where `in`. Started and finished apart, so that a thread has the loads of several rows in
// flight: finishing waits for them and, at the ends of an ODD row, loads element by element.
template <bool ODD> struct Started {
    uint4 lo;
};
template <> struct Started<true> {
    uint4 lo, hi;
};
template <bool ODD, int D>
__device__ __forceinline__ Started<ODD> start_row(const Bits<D>* row, int c, int h, bool in) {
    Started<ODD> s;
    if constexpr (!ODD) {
        s.lo = in ? __ldcs(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
    } else {
        const uintptr_t a = reinterpret_cast<uintptr_t>(row + c);
        const uint4* group = reinterpret_cast<const uint4*>(a & ~static_cast<uintptr_t>(15));
        in = in && c >= 0 && c + Vec<D>::E <= h;
        s.lo = in ? __ldg(group) : make_uint4(0, 0, 0, 0);
        s.hi = in ? __ldg(group + ((a & 15) != 0 ? 1 : 0)) : make_uint4(0, 0, 0, 0);
    }
    return s;
}
template <bool ODD, int D>
__device__ __forceinline__ Raw<D, Vec<D>::E> finish_row(const Started<ODD>& s, const Bits<D>* row, int c, int h, bool in) {
    constexpr int E = Vec<D>::E;
    Raw<D, E> r;
    if constexpr (!ODD) {
        r.v = s.lo;
    } else if (!in || (c >= 0 && c + E <= h)) {
        r.v = join_groups<D>(row + c, s.lo, s.hi);
    } else {
        dev::V16<D> v;
#pragma unroll
        for (int e = 0; e < E; ++e) v.b[e] = c + e >= 0 && c + e < h ? __ldg(row + c + e) : 0;
        r.v = v.u;
    }
    return r;
}
template <bool ODD, int D>
__device__ __forceinline__ Raw<D, Vec<D>::E> get_row(const Bits<D>* row, int c, int h) {
    return finish_row<ODD, D>(start_row<ODD, D>(row, c, h, true), row, c, h, true);
}
// The same as floats, of a type that may be wider (parameters next to 16-bit rows).
template <bool ODD, int D, int E>
__device__ __forceinline__ void get_params(const Bits<D>* row, int c, int h, float (&a)[E]) {
    if constexpr (!ODD) {
        load_f<D, E>(row + c, a);
    } else {
        constexpr int W = Vec<D>::E;
#pragma unroll
        for (int i = 0; i < E / W; ++i) {
            float t[W];
            unpack<D, W>(get_row<true, D>(row, c + i * W, h), t);
#pragma unroll
            for (int e = 0; e < W; ++e) a[i * W + e] = t[e];
        }
    }
}
// Stores columns [c, c + E), those inside the row; row + c lies on a 16-byte boundary.
template <bool ODD, int D, int E>
__device__ __forceinline__ void put_row(Bits<D>* row, int c, int h, const float (&a)[E]) {
    if (!ODD || (c >= 0 && c + E <= h)) {
        store_f_cs<D, E>(row + c, a);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (c + e >= 0 && c + e < h) row[c + e] = Ty<D>::store(a[e]);
    }
}
template <bool ODD, int D>
__device__ __forceinline__ void put_raw(Bits<D>* row, int c, int h, const Raw<D, Vec<D>::E>& r) {
    if (!ODD || (c >= 0 && c + Vec<D>::E <= h)) {
        store_raw_cs<D, Vec<D>::E>(row + c, r);
    } else {
        dev::V16<D> v;
        v.u = r.v;
#pragma unroll
        for (int e = 0; e < Vec<D>::E; ++e)
            if (c + e >= 0 && c + e < h) row[c + e] = v.b[e];
    }
}
// Accesses that cover a row of h elements at any shift.
template <bool ODD> __host__ __device__ __forceinline__ long long accesses(long long h, int e) {
    return ODD ? (h + 2 * e - 2) / e : (h + e - 1) / e;
}

// Two floats in one register pair: sm_100 multiplies and adds both in one instruction.
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 split(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
// 16 bytes as pairs of floats, and back.
template <int D>
__device__ __forceinline__ void unpack2(const uint4& u, F2 (&a)[Vec<D>::E / 2]) {
    float f[Vec<D>::E];
    Vec<D>::unpack(u, f);
#pragma unroll
    for (int i = 0; i < Vec<D>::E / 2; ++i) a[i] = f2(f[2 * i], f[2 * i + 1]);
}
template <int D>
__device__ __forceinline__ uint4 pack2(const F2 (&a)[Vec<D>::E / 2]) {
    float f[Vec<D>::E];
#pragma unroll
    for (int i = 0; i < Vec<D>::E / 2; ++i) {
        const float2 t = split(a[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
    }
    return Vec<D>::pack(f);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float2 warp_sum(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}

// Sums over all threads of a block (a multiple of 32, at most 1024) in a fixed order, result in
// every thread. `parity` alternates between calls: a call's buffer is written again only two
// calls later, after the barrier of the call between, so one barrier per sum is enough.
__device__ __forceinline__ float plus(float a, float b) { return a + b; }
__device__ __forceinline__ float2 plus(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
template <typename T>
__device__ __forceinline__ T block_sum(T v, T (&buf)[2][32], int parity, int tid, int warps) {
    v = warp_sum(v);
    if (warps == 1) return v;
    if ((tid & 31) == 0) buf[parity][tid >> 5] = v;
    __syncthreads();
    if (warps <= 8) {  // a few broadcast loads instead of another tree of shuffles
        T s = buf[parity][0];
#pragma unroll
        for (int w = 1; w < 8; ++w)
            if (w < warps) s = plus(s, buf[parity][w]);
        return s;
    }
    return warp_sum((tid & 31) < warps ? buf[parity][tid & 31] : T{});
}

// 1 / sqrt(v) to within an ulp or two: the hardware's approximation and a Newton step, in 6
// instructions where the correctly rounded root and quotient take some 50 in every thread of a row.
__device__ __forceinline__ float inv_sqrt(float v) {
    const float r = rsqrtf(v);
    const float d = fmaf(-v * r, r, 1.0f);
    // Zero, infinity and NaN as they come out of the approximation.
    return fabsf(d) < 1.0f ? fmaf(0.5f * r, d, r) : r;
}

inline int size_of(int d) { return d == kF32 ? 4 : 2; }
inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Rows of `h` elements, `stride` apart from `p`, that all start and end on 16-byte boundaries.
inline bool rows16(const void* p, long long stride, long long h, int size) {
    return on16(p) && (stride * size) % 16 == 0 && (h * size) % 16 == 0;
}
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline int round32(long long v) { return static_cast<int>((v + 31) / 32 * 32); }

// SMs of the current device (148 on a B200); looked up once per device.
int sm_count();

// Threads along a row and rows per block (at most `most` threads in all) for kernels without barriers:
// short rows share a block.
struct BlockShape {
    int x, y;
};
inline BlockShape block_shape(long long accesses, int most) {
    const int x = static_cast<int>(std::min<long long>(accesses, most));
    return {x, most / x};
}

// A kernel's form: one aligned row per block (row indexes are then the same for the whole block, which
// saves registers: 32768 looked-up rows of 8 KiB 63 us, 79 without), several, or ODD ones.
struct Plain {
    static constexpr bool odd = false, many = false;
};
struct Many {
    static constexpr bool odd = false, many = true;
};
struct Odd {
    static constexpr bool odd = true, many = true;
};
template <typename Form> __device__ __forceinline__ int row_in_block() { return Form::many ? threadIdx.y : 0; }
template <typename Form> __device__ __forceinline__ int rows_per_block() { return Form::many ? blockDim.y : 1; }
// f(form, accesses per row, block) for rows of h elements.
template <typename F>
cudaError_t with_form(bool odd, long long h, int e, int threads, F&& f) {
    const long long n = odd ? accesses<true>(h, e) : accesses<false>(h, e);
    const BlockShape b = block_shape(n, threads);
    if (odd) return f(Odd{}, n, b);
    if (b.y > 1) return f(Many{}, n, b);
    return f(Plain{}, n, b);
}

// f(integral_constant<D>) for a floating-point type code.
template <int V> struct Int { static constexpr int value = V; };
template <typename F>
cudaError_t with_type(int d, F&& f) {
    switch (d) {
    case kF32: return f(Int<kF32>{});
    case kBF16: return f(Int<kBF16>{});
    case kF16: return f(Int<kF16>{});
    default: return cudaErrorInvalidValue;
    }
}
// A type and the type of what goes with it: the same, or f32.
template <typename F>
cudaError_t with_types(int d, int w, F&& f) {
    return with_type(d, [&](auto D) {
        constexpr int kD = decltype(D)::value;
        if (w == kD) return f(Int<kD>{}, Int<kD>{});
        if (w == kF32) return f(Int<kD>{}, Int<kF32>{});
        return cudaErrorInvalidValue;
    });
}

}  // namespace ops
}  // namespace bccl
