// Typed vector loads and stores of the recurrence and norm kernels: V
// neighbouring elements of a type as fp32 values.  ALIGNED pieces move as one
// access of V * sizeof(T) bytes (16 at most); others element by element.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace cgdr {

template <int BYTES> struct RawOf;
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// V elements of T as they lie in memory
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> pack_zero()
{
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = from_f32<T>(0.0f);
    return r;
}

template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p, int valid = V)
{
    Pack<T, V> r;
    if constexpr (ALIGNED) {
        using Raw = typename RawOf<sizeof(T) * V>::type;
        *reinterpret_cast<Raw*>(&r) = *reinterpret_cast<const Raw*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.e[i] = i < valid ? p[i] : from_f32<T>(0.0f);
    }
    return r;
}

// Two values at once: one conversion instruction for the 16-bit types.
template <typename T> __device__ __forceinline__ void from_f32x2(float a, float b, T* to)
{
    to[0] = from_f32<T>(a);
    to[1] = from_f32<T>(b);
}
template <> __device__ __forceinline__ void from_f32x2<__nv_bfloat16>(float a, float b, __nv_bfloat16* to)
{
    *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(a, b);
}
template <> __device__ __forceinline__ void from_f32x2<__half>(float a, float b, __half* to)
{
    *reinterpret_cast<__half2*>(to) = __floats2half2_rn(a, b);
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> to_pack(const float* v)
{
    Pack<T, V> r;
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) from_f32x2<T>(v[i], v[i + 1], &r.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.e[i] = from_f32<T>(v[i]);
    }
    return r;
}

template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void store_pack(T* p, const float* v, int valid = V)
{
    const Pack<T, V> r = to_pack<T, V>(v);
    if constexpr (ALIGNED) {
        using Raw = typename RawOf<sizeof(T) * V>::type;
        *reinterpret_cast<Raw*>(p) = *reinterpret_cast<const Raw*>(&r);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < valid) p[i] = r.e[i];
    }
}

}  // namespace cgdr
