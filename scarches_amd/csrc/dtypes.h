// Element types of the entry points that take more than fp32: 0 = fp32, 1 = bf16, 2 = fp16 (gfx950 only).
// A vector of N elements is loaded and stored as ONE access that needs only the element's own alignment (rows with an odd
// pitch start anywhere; unaligned access is on for this target), and is held in fp32 between the two.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

enum { SCA_F32 = 0, SCA_BF16 = 1, SCA_F16 = 2 };

// Storage types; conversions to the 16-bit types round to nearest, ties to even (one rounding of an fp32 result).
struct sca_bf16 { uint16_t bits; };
struct sca_f16 { _Float16 v; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(sca_bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
__device__ __forceinline__ float to_f32(sca_f16 v) { return (float)v.v; }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ sca_bf16 from_f32<sca_bf16>(float v) {
    return sca_bf16{__builtin_bit_cast(uint16_t, (__bf16)v)};
}
template <> __device__ __forceinline__ sca_f16 from_f32<sca_f16>(float v) { return sca_f16{(_Float16)v}; }

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&v)[N]) {
    T t[N];
    __builtin_memcpy(t, p, sizeof(T) * N);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(t[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&v)[N]) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = from_f32<T>(v[i]);
    __builtin_memcpy(p, t, sizeof(T) * N);
}
// The same past the caches, for results that are larger than they are (what reads them next would not find them there).
typedef uint32_t words4 __attribute__((ext_vector_type(4)));
typedef uint32_t words2 __attribute__((ext_vector_type(2)));
template <typename T, int N>
__device__ __forceinline__ void stream_vec(T* __restrict__ p, const float (&v)[N]) {
    typedef words4 words4_at __attribute__((aligned(2)));
    typedef words2 words2_at __attribute__((aligned(2)));
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = from_f32<T>(v[i]);
    static_assert(sizeof(T) * N == 16 || sizeof(T) * N == 8, "one store");
    if constexpr (sizeof(T) * N == 16) {
        words4 w;
        __builtin_memcpy(&w, t, 16);
        __builtin_nontemporal_store(w, (words4_at*)p);
    } else {
        words2 w;
        __builtin_memcpy(&w, t, 8);
        __builtin_nontemporal_store(w, (words2_at*)p);
    }
}
// The first `left` of N elements (the others read as 0 / are not written).
template <typename T, int N>
__device__ __forceinline__ void load_part(const T* __restrict__ p, int left, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < left ? to_f32(p[i]) : 0.f;
}
template <typename T, int N>
__device__ __forceinline__ void store_part(T* __restrict__ p, int left, const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < left) p[i] = from_f32<T>(v[i]);
}
