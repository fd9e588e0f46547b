// Element types of the sequence-model operators (fp32, bf16, fp16) and vector
// access to them: values are held in fp32 and rounded once, to nearest even,
// when they are stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

// N consecutive elements: one aligned load or store of N * sizeof(T) bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f32(const T *p, float (&x)[N])
{
    const Pack<T, N> q = *reinterpret_cast<const Pack<T, N> *>(p);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to_f32(q.v[i]);
}

template <typename T, int N>
__device__ __forceinline__ void store_f32(T *p, const float (&x)[N])
{
    Pack<T, N> q;
#pragma unroll
    for (int i = 0; i < N; i++) q.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Pack<T, N> *>(p) = q;
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
