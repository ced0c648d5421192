// Matrix product in 8-bit integers with a scale per row and per output channel (gfx950).
//
//   rows:    s_m = max_k |x_mk| / 127 (fp32),  q_mk = round(x_mk / s_m), ties to even     (sca_quant_rows_i8)
//   product: y_mn = (sum_k q_mk w_nk) * s_m * s_n + bias_n                                (sca_gemm_i8)
//
// The sum is exact in int32 (k < 2^31 / 128^2), so its order does not matter; the product is v_mfma_i32_*_i8.
#include "common.h"
#include "dtypes.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));

namespace {

// q = round(x / s) with the exact quotient: the estimate x * (1 / s) may fall on the other side of a middle, so its
// distance from x is taken without rounding (one fma: q s has at most 32 bits and the difference at most 24).
__device__ __forceinline__ float nearest(float x, float s, float inv) {
    float q = rintf(x * inv);
    const float d = fmaf(-q, s, x), h = 0.5f * s;
    if (d > h || (d == h && ((int)q & 1))) q += 1.f;
    else if (d < -h || (d == -h && ((int)q & 1))) q -= 1.f;
    return fminf(fmaxf(q, -127.f), 127.f);
}

// One wave per row, two passes over it.
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, long long ldx, long long rows, int k,
                                                         int8_t* __restrict__ q, long long ldq, float* __restrict__ scale) {
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    uint32_t amax = 0;
    for (int c = lane; c < k; c += 64) {
        const uint32_t b = __float_as_uint(to_f32(x[r * ldx + c])) & 0x7fffffffu;
        amax = b > amax ? b : amax;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t b = __shfl_xor(amax, o, 64);
        amax = b > amax ? b : amax;
    }
    const bool finite = amax < 0x7f800000u;
    const float s = finite ? __uint_as_float(amax) / 127.f : __uint_as_float(0x7fc00000u);
    const bool tiny = !(s >= 1e-37f);            // 1 / s is not a number of this type: the quotient in 64 bits
    const float inv = 1.f / s;
    for (long long c = lane; c < ldq; c += 64) {
        float v = 0.f;
        if (c < k && finite && s > 0.f) {
            const float xv = to_f32(x[r * ldx + c]);
            v = tiny ? fminf(fmaxf((float)rint((double)xv / (double)s), -127.f), 127.f) : nearest(xv, s, inv);
        }
        q[r * ldq + c] = (int8_t)(int)v;
    }
    if (lane == 0) scale[r] = s;
}

__device__ __forceinline__ i32x4 load16(const int8_t* p, int left) {
    i32x4 v = {0, 0, 0, 0};
    if (left >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else {
        int8_t b[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = i < left ? p[i] : 0;
        __builtin_memcpy(&v, b, 16);
    }
    return v;
}

// One wave per 16 x 16 tile of the result.
template <typename B, typename Y>
__global__ __launch_bounds__(64) void gemm_i8_kernel(const int8_t* __restrict__ xq, long long ldx,
                                                     const float* __restrict__ sx, const int8_t* __restrict__ wq,
                                                     long long ldw, const float* __restrict__ sw,
                                                     const B* __restrict__ bias, long long M, int N, int K,
                                                     Y* __restrict__ y, long long ldy) {
    const int lane = threadIdx.x;
    const long long m0 = (long long)blockIdx.x * 16;
    const int n0 = blockIdx.y * 16;
    const long long m = m0 + (lane & 15);
    const int n = n0 + (lane & 15), ko = (lane >> 4) * 16;
    i32x4 acc = {0, 0, 0, 0};
    for (int k = 0; k < K; k += 64) {
        const int left = K - k - ko;
        const i32x4 a = load16(xq + (m < M ? m : M - 1) * ldx + k + ko, left);
        const i32x4 b = load16(wq + (long long)(n < N ? n : N - 1) * ldw + k + ko, left);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0);
    }
    if (n >= N) return;
    const float s = sw[n], add = bias ? to_f32(bias[n]) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long r = m0 + (lane >> 4) * 4 + i;
        if (r < M) y[r * ldy + n] = from_f32<Y>(fmaf((float)acc[i] * sx[r], s, add));
    }
}

template <typename T>
int quant_rows(const void* x, long long ldx, long long rows, int k, int8_t* q, long long ldq, float* scale,
               hipStream_t st) {
    hipLaunchKernelGGL((quant_rows_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, (const T*)x, ldx, rows,
                       k, q, ldq, scale);
    SCA_CHECK_LAUNCH();
    return 0;
}

template <typename B, typename Y>
int gemm_i8(const int8_t* xq, long long ldx, const float* sx, const int8_t* wq, long long ldw, const float* sw,
            const void* bias, long long M, int N, int K, void* y, long long ldy, hipStream_t st) {
    hipLaunchKernelGGL((gemm_i8_kernel<B, Y>), dim3((unsigned)((M + 15) / 16), (N + 15) / 16), dim3(64), 0, st, xq, ldx,
                       sx, wq, ldw, sw, (const B*)bias, M, N, K, (Y*)y, ldy);
    SCA_CHECK_LAUNCH();
    return 0;
}

constexpr int I8_MAX_K = (1 << 17) - 1;         // 2^17 products of -128 * -128 would pass int32

}  // namespace

extern "C" int sca_gemm_i8_max_k(void) { return I8_MAX_K; }

extern "C" int sca_quant_rows_i8(const void* x, long long ldx, int dtype, long long rows, int k, int8_t* q,
                                 long long ldq, float* scale, void* stream) {
    if (dtype < SCA_F32 || dtype > SCA_F16 || rows < 0 || k <= 0 || ldx < 0 || ldq < k) return -1;
    if (rows == 0) return 0;
    if (!x || !q || !scale) return -1;
    hipStream_t st = (hipStream_t)stream;
    return dtype == SCA_F32    ? quant_rows<float>(x, ldx, rows, k, q, ldq, scale, st)
           : dtype == SCA_BF16 ? quant_rows<sca_bf16>(x, ldx, rows, k, q, ldq, scale, st)
                               : quant_rows<sca_f16>(x, ldx, rows, k, q, ldq, scale, st);
}

extern "C" int sca_gemm_i8(const int8_t* xq, long long ldx, const float* sx, const int8_t* wq, long long ldw,
                           const float* sw, const void* bias, int btype, long long M, int N, int K, void* y, int ytype,
                           long long ldy, void* stream) {
    if (ytype < SCA_F32 || ytype > SCA_F16 || (btype != SCA_F32 && btype != ytype)) return -1;
    if (M < 0 || N < 0 || K <= 0 || K > I8_MAX_K || ldx < 0 || ldw < K || ldy < N) return -1;
    if (M == 0 || N == 0) return 0;
    if (!xq || !sx || !wq || !sw || !y) return -1;
    hipStream_t st = (hipStream_t)stream;
#define I8_CALL(B, Y) gemm_i8<B, Y>(xq, ldx, sx, wq, ldw, sw, bias, M, N, K, y, ldy, st)
    if (ytype == SCA_F32) return I8_CALL(float, float);
    if (ytype == SCA_BF16) return btype == SCA_F32 ? I8_CALL(float, sca_bf16) : I8_CALL(sca_bf16, sca_bf16);
    return btype == SCA_F32 ? I8_CALL(float, sca_f16) : I8_CALL(sca_f16, sca_f16);
#undef I8_CALL
}
