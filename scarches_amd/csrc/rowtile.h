// Rows held in registers (gfx950): TPR threads share a row, each holds V vectors of 16 bytes of it, so that a row is read
// once whatever is computed of it.  Used by the layer norm and the row quantization.
#pragma once
#include "common.h"
#include "dtypes.h"

// Elements of a 16-byte vector.
template <typename T>
constexpr int vec_of() { return 16 / (int)sizeof(T); }

// How the width n of a row meets the vectors.
enum {
    ROW_FULL,       // n is a whole number of vectors: a vector is there or not
    ROW_RAGGED,     // it is not: the last vector is moved back to end with the row.  Its first elements belong to the vector
                    // before as well; sums leave them out (`skip`), results are written twice with the same values
    ROW_TINY        // the row is shorter than a vector: element by element
};
inline int row_mode(int n, int vec) { return n < vec ? ROW_TINY : n % vec ? ROW_RAGGED : ROW_FULL; }

// Vector j of thread t: its first column, how many of its elements are another vector's, and whether there is one at all.
template <typename T, int TPR, int MODE>
struct Cols {
    int c, skip;
    bool there;
    __device__ __forceinline__ Cols(int j, int t, int n) {
        constexpr int VEC = vec_of<T>();
        c = (j * TPR + t) * VEC;
        there = c < n;
        skip = 0;
        if (MODE == ROW_RAGGED && c > n - VEC) {
            skip = c - (n - VEC);
            c = n - VEC;
        }
    }
    __device__ __forceinline__ bool own(int i, int n) const {
        return MODE == ROW_FULL || (MODE == ROW_RAGGED ? i >= skip : i < n);
    }
};
// Vectors are loaded as the 16 bytes that they are and unpacked where they are used: a conversion next to its load would
// wait for each load in turn.
typedef uint32_t raw_t __attribute__((ext_vector_type(4)));
template <int MODE, typename T>
__device__ __forceinline__ void load_cols(const T* __restrict__ row, int c, int n, raw_t& v) {
    if (MODE == ROW_TINY) {
        T t[vec_of<T>()] = {};
#pragma unroll
        for (int i = 0; i < vec_of<T>(); ++i)
            if (i < n) t[i] = row[i];
        __builtin_memcpy(&v, t, 16);
    } else {
        __builtin_memcpy(&v, row + c, 16);
    }
}
template <typename T>
__device__ __forceinline__ void unpack(const raw_t& raw, float (&v)[vec_of<T>()]);
template <>
__device__ __forceinline__ void unpack<float>(const raw_t& raw, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(raw[i]);
}
template <>
__device__ __forceinline__ void unpack<sca_bf16>(const raw_t& raw, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(raw[i] << 16);
        v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
    }
}
template <>
__device__ __forceinline__ void unpack<sca_f16>(const raw_t& raw, float (&v)[8]) {
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    const half8 h = __builtin_bit_cast(half8, raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
}
// The same for a later pass over the row: the compiler must not keep the values of the pass before, which take twice the
// registers of 16-bit rows.
template <typename T>
__device__ __forceinline__ void unpack_again(raw_t& raw, float (&v)[vec_of<T>()]) {
    if (sizeof(T) == 2) asm volatile("" : "+v"(raw));
    unpack<T>(raw, v);
}
template <int MODE, typename T, int VEC>
__device__ __forceinline__ void store_cols(T* __restrict__ row, int c, int n, const float (&v)[VEC], bool stream) {
    if (MODE == ROW_TINY) store_part<T, VEC>(row, n, v);
    else if (stream) stream_vec<T, VEC>(row + c, v);
    else store_vec<T, VEC>(row + c, v);
}

// Sum / integer maximum over the TPR threads of a row, in every one of them.  TPR > 64: all threads of the workgroup call it
// together, and `scratch` (one entry per wave) is LDS that nothing else uses until the next barrier.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    if constexpr (TPR >= 64) v = wave_sum(v);
    else if constexpr (TPR == 4) {
        v += dpp_f32<0xB1>(v);      // quad_perm [1,0,3,2]
        v += dpp_f32<0x4E>(v);      // quad_perm [2,3,0,1]
    } else {
        v = row16_sum(v);
        if constexpr (TPR == 32) v += __shfl_xor(v, 16, 64);
        static_assert(TPR >= 16, "rows of 4, 16, 32, 64 or more lanes");
    }
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += scratch[threadIdx.x / TPR * (TPR / 64) + i];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_umax(uint32_t v, uint32_t* scratch) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) {
        const uint32_t b = __shfl_xor(v, o, 64);
        v = b > v ? b : v;
    }
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) {
            const uint32_t b = scratch[threadIdx.x / TPR * (TPR / 64) + i];
            v = b > v ? b : v;
        }
    }
    return v;
}
