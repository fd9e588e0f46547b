// Element types of the sequence-model operators (fp32, bf16, fp16) and vector
// access to them: values are held in fp32 and rounded once, to nearest even,
// when they are stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "lifscan_b200.h"

namespace lifb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v)
{
    return __float2half_rn(v);
}

// Two elements of a 16-bit type in a word.
template <typename T>
__device__ __forceinline__ float2 two_f32(uint32_t w)
{
    if constexpr (sizeof(T) == 2) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value)
            return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
        else
            return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    } else {
        return make_float2(0.0f, 0.0f);
    }
}
template <typename T>
__device__ __forceinline__ uint32_t two_from_f32(float a, float b)
{
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    } else {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
}

// N consecutive elements as they are in memory: one aligned load or store of N *
// sizeof(T) bytes, whole words where it has any.
template <typename T, int N>
struct Pack {
    static constexpr int kBytes = sizeof(T) * N, kWords = kBytes / 4;
    static constexpr bool kWhole = kBytes % 4 == 0;
    struct alignas(kBytes) Words {
        uint32_t w[kWhole ? kWords : 1];
    };
    struct alignas(kBytes) Elems {
        T v[N];
    };
    using Store = typename std::conditional<kWhole, Words, Elems>::type;
    Store s;

    __device__ __forceinline__ void zero()
    {
        if constexpr (kWhole) {
#pragma unroll
            for (int i = 0; i < kWords; i++) s.w[i] = 0;
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) s.v[i] = from_f32<T>(0.0f);
        }
    }
    __device__ __forceinline__ void load(const T *p) { s = *reinterpret_cast<const Store *>(p); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<Store *>(p) = s; }
    __device__ __forceinline__ void get(float (&x)[N]) const
    {
        if constexpr (!kWhole) {
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = to_f32(s.v[i]);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = __uint_as_float(s.w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; i++) {
                const float2 f = two_f32<T>(s.w[i]);
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ void set(const float (&x)[N])
    {
        if constexpr (!kWhole) {
#pragma unroll
            for (int i = 0; i < N; i++) s.v[i] = from_f32<T>(x[i]);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i++) s.w[i] = __float_as_uint(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; i++) s.w[i] = two_from_f32<T>(x[2 * i], x[2 * i + 1]);
        }
    }
};

template <typename T, int N>
__device__ __forceinline__ void load_f32(const T *p, float (&x)[N])
{
    Pack<T, N> q;
    q.load(p);
    q.get(x);
}

template <typename T, int N>
__device__ __forceinline__ void store_f32(T *p, const float (&x)[N])
{
    Pack<T, N> q;
    q.set(x);
    q.store(p);
}

inline int64_t dtype_bytes(int dtype) { return dtype == LIFB_F32 ? 4 : dtype == LIFB_BF16 || dtype == LIFB_F16 ? 2 : 0; }

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace lifb

// Runs the statement with T the element type that `dtype` names (checked before).
#define LIFB_BY_DTYPE(dtype, T, ...)           \
    switch (dtype) {                           \
        case LIFB_F32: {                       \
            using T = float;                   \
            __VA_ARGS__;                       \
            break;                             \
        }                                      \
        case LIFB_BF16: {                      \
            using T = __nv_bfloat16;           \
            __VA_ARGS__;                       \
            break;                             \
        }                                      \
        default: {                             \
            using T = __half;                  \
            __VA_ARGS__;                       \
            break;                             \
        }                                      \
    }
