// slideformer_amd: what the model operators share (gfx950, wave64): element
// types, 16-byte row accesses of any alignment, wave reductions, argument checks.
#ifndef SLIDEFORMER_AMD_OPS_COMMON_H
#define SLIDEFORMER_AMD_OPS_COMMON_H

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "hip_ptr.h"
#include "model_ops.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// The target runs with unaligned access on: a 16-byte access needs the
// alignment of an element only, so rows of odd length and views at odd offsets
// take the same instructions.
typedef u32x4_t u32x4_any __attribute__((aligned(2)));

// E elements of one 16-byte access, as fp32
template <typename T> struct Elem;

template <> struct Elem<float> {
    static constexpr int kCount = 4;
    __device__ static float to_f32(float x) { return x; }
    __device__ static float from_f32(float x) { return x; }
    __device__ static void unpack(u32x4_t u, float (&x)[4])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(u[i]);
    }
    __device__ static u32x4_t pack(const float (&x)[4])
    {
        u32x4_t u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(x[i]);
        return u;
    }
};

template <> struct Elem<__bf16> {
    static constexpr int kCount = 8;
    __device__ static float to_f32(__bf16 x) { return static_cast<float>(x); }
    __device__ static __bf16 from_f32(float x) { return static_cast<__bf16>(x); }
    __device__ static void unpack(u32x4_t u, float (&x)[8])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    __device__ static u32x4_t pack(const float (&x)[8])
    {
        typedef __bf16 v8 __attribute__((ext_vector_type(8)));
        v8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<__bf16>(x[i]);
        return __builtin_bit_cast(u32x4_t, v);
    }
};

template <> struct Elem<_Float16> {
    static constexpr int kCount = 8;
    __device__ static float to_f32(_Float16 x) { return static_cast<float>(x); }
    __device__ static _Float16 from_f32(float x) { return static_cast<_Float16>(x); }
    __device__ static void unpack(u32x4_t u, float (&x)[8])
    {
        typedef _Float16 v8 __attribute__((ext_vector_type(8)));
        const v8 v = __builtin_bit_cast(v8, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(v[i]);
    }
    __device__ static u32x4_t pack(const float (&x)[8])
    {
        typedef _Float16 v8 __attribute__((ext_vector_type(8)));
        v8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<_Float16>(x[i]);
        return __builtin_bit_cast(u32x4_t, v);
    }
};

// Vector `vec` of a row of `hidden` elements: 16 bytes where it is whole, its
// elements alone where the row ends inside it, zeros beyond.
template <typename T>
__device__ __forceinline__ void load_vec(const T* row, uint32_t vec, uint32_t hidden, float (&x)[Elem<T>::kCount])
{
    constexpr uint32_t E = Elem<T>::kCount;
    const uint32_t at = vec * E;
    if (at + E <= hidden) {
        Elem<T>::unpack(*reinterpret_cast<const u32x4_any*>(row + at), x);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < E; ++i) x[i] = at + i < hidden ? Elem<T>::to_f32(row[at + i]) : 0.0f;
    }
}

// The same as it lies in memory.
template <typename T> __device__ __forceinline__ u32x4_t load_raw(const T* row, uint32_t vec, uint32_t hidden)
{
    constexpr uint32_t E = Elem<T>::kCount;
    const uint32_t at = vec * E;
    if (at + E <= hidden) return *reinterpret_cast<const u32x4_any*>(row + at);
    T x[E];
#pragma unroll
    for (uint32_t i = 0; i < E; ++i) x[i] = at + i < hidden ? row[at + i] : Elem<T>::from_f32(0.0f);
    return __builtin_bit_cast(u32x4_t, x);
}

template <typename T, int E>
__device__ __forceinline__ void store_vec(T* row, uint32_t vec, uint32_t hidden, const float (&x)[E])
{
    const uint32_t at = vec * E;
    if (at + E <= hidden) {
        if constexpr (E == Elem<T>::kCount) {
            *reinterpret_cast<u32x4_any*>(row + at) = Elem<T>::pack(x);
        } else {
            // fp32 beside 16-bit elements: two accesses
#pragma unroll
            for (int h = 0; h < E; h += 4) {
                const float part[4] = {x[h], x[h + 1], x[h + 2], x[h + 3]};
                *reinterpret_cast<u32x4_any*>(row + at + h) = Elem<float>::pack(part);
            }
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < E; ++i)
            if (at + i < hidden) row[at + i] = Elem<T>::from_f32(x[i]);
    }
}

__device__ __forceinline__ float wave_sum(float x)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint32_t y = __shfl_xor(x, d);
        x = y > x ? y : x;
    }
    return x;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
inline int dtype_bytes(int dtype)
{
    switch (dtype) {
    case LA_F32: case LA_I32: return 4;
    case LA_BF16: case LA_F16: return 2;
    case LA_I64: return 8;
    case LA_I8: case LA_F8E4M3: return 1;
    default: return 0;
    }
}

inline bool is_float_dtype(int dtype) { return dtype == LA_F32 || dtype == LA_BF16 || dtype == LA_F16; }

// A matrix's pointer: there, aligned to its elements, rows that do not overlap.
inline int check_matrix(const void* p, int dtype, uint64_t hidden, uint64_t stride)
{
    if (!p || reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(dtype_bytes(dtype))) return LA_EINVAL;
    return stride < hidden ? LA_EINVAL : LA_OK;
}

inline int check_workspace(const void* ws, uint64_t have, uint64_t need, uintptr_t align)
{
    if (need == 0) return LA_OK;
    return !ws || have < need || reinterpret_cast<uintptr_t>(ws) % align ? LA_EINVAL : LA_OK;
}

// One launch; the returned code is this launch's own, and no earlier call's error is cleared or reported.
template <typename... P, typename... A>
int launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, A... given)
{
    void* ptrs[sizeof...(P)];
    return [&](P... args) {
        int k = 0;
        ((ptrs[k++] = &args), ...);
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, ptrs, 0, stream);
        return e == hipSuccess ? LA_OK : static_cast<int>(e);
    }(static_cast<P>(given)...);
}

template <typename A, typename B> constexpr auto ceil_div(A a, B b) { return (a + b - 1) / b; }

}  // namespace

#endif  // SLIDEFORMER_AMD_OPS_COMMON_H
