// What the sequence operators (selective scan, short causal convolution, residual norm) share: element types and
// their conversions, vectors of elements that may or may not be aligned, packed fp32 arithmetic, reductions over lanes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <initializer_list>

#include "../../include/ovl_b200.h"

namespace ovl {

// Host side: records the CUDA error for ovl_last_cuda_error() and returns OVL_ERR_CUDA (ovl_launcher.cu).
__attribute__((visibility("hidden"))) int record_cuda_error(cudaError_t e);

inline int launch_status() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? OVL_OK : record_cuda_error(e);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__host__ __device__ inline bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

// Allows a kernel `smem` bytes of dynamic shared memory and, with `registers` > 0, makes sure that its blocks of `threads`
// start with that many (OVL_ERR_INVALID if not); asked of the driver once per kernel and device.
__attribute__((visibility("hidden"))) int prepare_kernel(const void* kernel, size_t smem, int threads = 0, int registers = 0);

// SM count of the current device (148 on a B200), asked once per device.
__attribute__((visibility("hidden"))) int sequence_sm_count();

// ---------------------------------------------------------------------------------------------------------
// element types

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// one rounding to nearest even
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N elements as loaded, before conversion: N * sizeof(T) bytes in registers
template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
    T v[N];
};

// N consecutive elements; `vec`: the address is aligned to the pack and all N exist; otherwise the first `valid`
// are read one by one and the others are zero.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* __restrict__ p, bool vec, int valid) {
    Pack<T, N> r;
    if (vec) {
        if constexpr (sizeof(T) * N <= 16) {
            r = *reinterpret_cast<const Pack<T, N>*>(p);
        } else {
            constexpr int H = 16 / sizeof(T);
#pragma unroll
            for (int i = 0; i < N; i += H)
                *reinterpret_cast<Pack<T, H>*>(&r.v[i]) = *reinterpret_cast<const Pack<T, H>*>(p + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = i < valid ? p[i] : from_f32<T>(0.0f);
    }
    return r;
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T* __restrict__ p, const float (&x)[N], bool vec, int valid, int width = 0) {
    if (vec) {
        constexpr int H = sizeof(T) * N <= 16 ? N : 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < N; i += H) {
            Pack<T, H> r;
#pragma unroll
            for (int k = 0; k < H; ++k) r.v[k] = from_f32<T>(x[i + k]);
            *reinterpret_cast<Pack<T, H>*>(p + i) = r;
        }
    } else if (width >= 2) {                                             // (then `valid` is even)
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            Pack<T, 2> r;
            r.v[0] = from_f32<T>(x[i]);
            r.v[1] = from_f32<T>(x[i + 1]);
            if (i < valid) *reinterpret_cast<Pack<T, 2>*>(p + i) = r;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < valid) p[i] = from_f32<T>(x[i]);
    }
}

// a parameter vector that is either in the tensors' type or in fp32
template <typename T>
__device__ __forceinline__ float load_param(const void* p, int64_t i, bool f32) {
    return f32 ? reinterpret_cast<const float*>(p)[i] : to_f32(reinterpret_cast<const T*>(p)[i]);
}

// ---------------------------------------------------------------------------------------------------------
// fp32 arithmetic on pairs: one instruction for two values

struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 pack2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(F2 x, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
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
__device__ __forceinline__ F2 same2(float a) { return pack2(a, a); }
__device__ __forceinline__ float sum2(F2 x) {
    float a, b;
    unpack2(x, a, b);
    return a + b;
}

// 2^x: one special-function instruction, at most 2^-22.5 off relatively (measured over [-10, 0]: 1.4e-7 at most,
// 3e-8 on average, 1e-8 of bias), results below 2^-126 flush to zero
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ F2 exp2_pair(F2 x) {
    float a, b;
    unpack2(x, a, b);
    return pack2(exp2_approx(a), exp2_approx(b));
}

__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 1 / (1 + e^-x): two special-function instructions
__device__ __forceinline__ float sigmoid(float x) { return rcp_approx(1.0f + exp2_approx(-kLog2e * x)); }
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
// the same for pairs: one instruction for two values but for the special functions
__device__ __forceinline__ F2 sigmoid2(F2 x) {
    const F2 d = add2(exp2_pair(mul2(x, same2(-kLog2e))), same2(1.0f));
    float a, b;
    unpack2(d, a, b);
    return pack2(rcp_approx(a), rcp_approx(b));
}
__device__ __forceinline__ F2 silu2(F2 x) { return mul2(x, sigmoid2(x)); }

// log(1 + e^x) = max(x, 0) + log1p(e^-|x|), relatively exact to 3e-7 also where it is small (a step size of 0.001 is
// softplus(-6.9)): e = e^-|x| with the product by log2 e in two parts, then log1p(e) = e p(e) with p the polynomial of
// degree 9 that agrees with log1p(e) / e in the Chebyshev points of [0, 1] (5e-9 off).  A NaN stays one.  Two at a time,
// leaving the two e for the derivative.
__device__ __forceinline__ void softplus_pair(float& x0, float& x1, float& e0, float& e1) {
    const F2 t = pack2(fminf(fabsf(x0), 100.0f), fminf(fabsf(x1), 100.0f));
    const F2 hi = mul2(t, same2(-kLog2e));
    const F2 lo = fma2(t, same2(1.925963033e-8f), fma2(t, same2(kLog2e), hi));
    unpack2(hi, e0, e1);
    F2 e = pack2(exp2_approx(e0), exp2_approx(e1));
    e = fma2(e, mul2(lo, same2(-kLn2)), e);
    F2 p = same2(-3.176057013e-03f);
    p = fma2(p, e, same2(1.954252645e-02f));
    p = fma2(p, e, same2(-5.637361109e-02f));
    p = fma2(p, e, same2(1.054362357e-01f));
    p = fma2(p, e, same2(-1.526966691e-01f));
    p = fma2(p, e, same2(1.966327429e-01f));
    p = fma2(p, e, same2(-2.495161593e-01f));
    p = fma2(p, e, same2(3.332971036e-01f));
    p = fma2(p, e, same2(-4.999989271e-01f));
    p = fma2(p, e, same2(1.0f));
    p = fma2(p, e, pack2(x0 < 0.0f ? 0.0f : x0, x1 < 0.0f ? 0.0f : x1));
    unpack2(e, e0, e1);
    unpack2(p, x0, x1);
}
__device__ __forceinline__ float softplus(float x) {
    float y = x, e0, e1;
    softplus_pair(x, y, e0, e1);
    return x;
}

// copies of BYTES (4, 8 or 16) bytes from global to shared memory that the thread does not wait for
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until at most LEFT of the thread's groups of copies are in flight
template <int LEFT>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Slices of the rows whose parts are added up, one after another, for one sum: a block of kSumThreads has fewer sums the
// more slices there are (232 rows: 4.4 us in 32 slices, 21.7 in one; 1672 rows: 4.4 us in 32 slices, 10.4 in 8; up to 8
// rows the one slice's loads are under way together anyhow).
constexpr int kSumThreads = 256;
inline int sum_slices(int64_t rows) { return rows <= 8 ? 1 : rows <= 128 ? 8 : 32; }

// The widest copy, in elements, that all rows allow: 16, 8 or 4 bytes; 0: single 16-bit elements.  `of`: base addresses,
// `strides`: strides and sizes in elements.
template <typename T>
inline int copy_width(std::initializer_list<const void*> of, std::initializer_list<int64_t> strides) {
    for (int bytes = 16; bytes >= 4; bytes /= 2) {
        const int width = bytes / (int)sizeof(T);
        bool fits = true;
        for (const void* p : of) fits = fits && (uintptr_t)p % bytes == 0;
        for (int64_t s : strides) fits = fits && s % width == 0;
        if (fits) return width;
    }
    return 0;
}

// N elements into a slot of shared memory that only this thread reads: in flight while it goes on.  `vec`: all N are
// there, on 16-byte boundaries (or the pack's size); otherwise `valid` of them in copies of `width` elements, or, with
// width 0, one by one.
template <typename T, int N>
__device__ __forceinline__ void fetch_pack(T* slot, const T* __restrict__ p, bool vec, int valid, int width) {
    if (vec) {
        constexpr int BYTES = sizeof(T) * N > 16 ? 16 : (int)sizeof(T) * N, H = BYTES / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < N; i += H) copy_async<BYTES>(slot + i, p + i);
    } else if (width > 0) {
        constexpr int H = sizeof(T) == 2 ? 2 : 1;                        // 4 bytes: every width is a multiple
#pragma unroll
        for (int i = 0; i < N; i += H) {
            if (i < valid) copy_async<4>(slot + i, p + i);
            else if (H == 1) slot[i] = from_f32<T>(0.0f);
            else slot[i] = slot[i + 1] = from_f32<T>(0.0f);
        }
    } else {
        T v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = p[i < valid ? i : valid - 1];
#pragma unroll
        for (int i = 0; i < N; ++i) slot[i] = i < valid ? v[i] : from_f32<T>(0.0f);
    }
}
// the same slot, converted
template <typename T, int N>
__device__ __forceinline__ void read_slot(const T* slot, float (&x)[N]) {
    constexpr int H = sizeof(T) * N > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += H) {
        const Pack<T, H> r = *reinterpret_cast<const Pack<T, H>*>(slot + i);
#pragma unroll
        for (int k = 0; k < H; ++k) x[i + k] = to_f32(r.v[k]);
    }
}

// ---------------------------------------------------------------------------------------------------------
// Sums over lanes.  V values per lane are summed over the R lanes whose numbers differ in R * STRIDE / STRIDE (lane
// bits STRIDE, 2 STRIDE, ...).  While a lane holds several values every exchange sends half of them and keeps the
// other half (V - 1 exchanges for V >= R instead of V log2 R); then whole exchanges.  Afterwards lane l (its number
// among the R) holds max(1, V / R) totals in v[0...]: those of index reduced_index<V, R>(l) and following.
template <int V, int R, int STRIDE>
__device__ __forceinline__ void reduce_lanes(float (&v)[V], int lane) {
    int count = V;
#pragma unroll
    for (int s = R / 2; s >= 1; s >>= 1) {
        if (count > 1) {
            const int half = count / 2;
            const bool upper = lane & (s * STRIDE);
#pragma unroll
            for (int i = 0; i < (V > 1 ? V / 2 : 1); ++i) {
                if (i < half) {
                    const float keep = upper ? v[i + half] : v[i];
                    const float send = upper ? v[i] : v[i + half];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, s * STRIDE);
                }
            }
            count = half;
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], s * STRIDE);
        }
    }
}
template <int V, int R>
__device__ __forceinline__ constexpr int reduced_count() { return V >= R ? V / R : 1; }
template <int V, int R>
__device__ __forceinline__ int reduced_index(int l) { return V >= R ? l * (V / R) : l / (R / V); }
// lanes that hold the same totals when there are more lanes than values: only one of them writes
template <int V, int R>
__device__ __forceinline__ bool reduced_owner(int l) { return V >= R ? true : (l % (R / V)) == 0; }

}  // namespace ovl
