// Layer norm over the last dimension with weight and bias, forward and backward (gfx950).
//
//   h = (x - mean(x)) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = h * w + b
//   a = dy * w:  dx = rstd * (a - mean(a) - h * mean(a * h));  dw = sum over rows of dy * h;  db = sum over rows of dy
//
// fp32 / bf16 / fp16 rows of any width and pitch; statistics, sums and gradients are held in fp32 and rounded once when
// they are stored.  (sca_layer_fwd / sca_layer_bwd normalise without weight and bias inside the conditional layers.)
#include "common.h"
#include "dtypes.h"

namespace {

// One wave per row, three passes over the row.
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const T* __restrict__ x, long long ldx, long long rows, int n,
                                                     const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                     T* __restrict__ y, long long ldy, float* __restrict__ stats) {
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const T* xr = x + r * ldx;
    float s = 0.f;
    for (int c = lane; c < n; c += 64) s += to_f32(xr[c]);
    const float mean = wave_sum(s) / (float)n;
    float q = 0.f;
    for (int c = lane; c < n; c += 64) {
        const float d = to_f32(xr[c]) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(wave_sum(q) / (float)n + eps);
    for (int c = lane; c < n; c += 64) {
        float v = (to_f32(xr[c]) - mean) * rstd;
        if (w) v *= to_f32(w[c]);
        if (b) v += to_f32(b[c]);
        y[r * ldy + c] = from_f32<T>(v);
    }
    if (lane == 0 && stats) {
        stats[r] = mean;
        stats[rows + r] = rstd;
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_dx_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x,
                                                    long long ldx, long long rows, int n, const W* __restrict__ w,
                                                    const float* __restrict__ stats, T* __restrict__ dx, long long lddx) {
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const float mean = stats[r], rstd = stats[rows + r];
    float s1 = 0.f, s2 = 0.f;
    for (int c = lane; c < n; c += 64) {
        const float a = to_f32(dy[r * lddy + c]) * (w ? to_f32(w[c]) : 1.f);
        s1 += a;
        s2 = fmaf(a, (to_f32(x[r * ldx + c]) - mean) * rstd, s2);
    }
    const float m1 = wave_sum(s1) / (float)n, m2 = wave_sum(s2) / (float)n;
    for (int c = lane; c < n; c += 64) {
        const float a = to_f32(dy[r * lddy + c]) * (w ? to_f32(w[c]) : 1.f);
        const float h = (to_f32(x[r * ldx + c]) - mean) * rstd;
        dx[r * lddx + c] = from_f32<T>(rstd * (a - m1 - h * m2));
    }
}

constexpr int LN_SLABS = 256;       // row ranges of the weight gradients, summed in a fixed order

template <typename T>
__global__ __launch_bounds__(256) void ln_dw_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x,
                                                    long long ldx, long long rows, int n,
                                                    const float* __restrict__ stats, float* __restrict__ part) {
    const int c = blockIdx.y * 256 + threadIdx.x;
    if (c >= n) return;
    const long long per = (rows + gridDim.x - 1) / gridDim.x;
    const long long r0 = blockIdx.x * per, r1 = r0 + per < rows ? r0 + per : rows;
    float sw = 0.f, sb = 0.f;
    for (long long r = r0; r < r1; ++r) {
        const float d = to_f32(dy[r * lddy + c]);
        sw = fmaf(d, (to_f32(x[r * ldx + c]) - stats[r]) * stats[rows + r], sw);
        sb += d;
    }
    part[(long long)blockIdx.x * 2 * n + c] = sw;
    part[(long long)blockIdx.x * 2 * n + n + c] = sb;
}

template <typename W>
__global__ __launch_bounds__(256) void ln_dw_finish_kernel(const float* __restrict__ part, int slabs, int n,
                                                           W* __restrict__ dw, W* __restrict__ db) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float sw = 0.f, sb = 0.f;
    for (int s = 0; s < slabs; ++s) {
        sw += part[(long long)s * 2 * n + c];
        sb += part[(long long)s * 2 * n + n + c];
    }
    if (dw) dw[c] = from_f32<W>(sw);
    if (db) db[c] = from_f32<W>(sb);
}

int ln_slabs(long long rows) { return rows < LN_SLABS ? (int)(rows > 0 ? rows : 1) : LN_SLABS; }

template <typename T, typename W>
int ln_fwd(const void* x, long long ldx, long long rows, int n, const void* w, const void* b, float eps, void* y,
           long long ldy, float* stats, hipStream_t st) {
    hipLaunchKernelGGL((ln_fwd_kernel<T, W>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, (const T*)x, ldx, rows,
                       n, (const W*)w, (const W*)b, eps, (T*)y, ldy, stats);
    SCA_CHECK_LAUNCH();
    return 0;
}

template <typename T, typename W>
int ln_bwd(const void* dy, long long lddy, const void* x, long long ldx, long long rows, int n, const void* w,
           const float* stats, void* dx, long long lddx, void* dw, void* db, float* ws, hipStream_t st) {
    if (rows > 0 && dx)
        hipLaunchKernelGGL((ln_dx_kernel<T, W>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, (const T*)dy, lddy,
                           (const T*)x, ldx, rows, n, (const W*)w, stats, (T*)dx, lddx);
    if (dw || db) {
        const int slabs = ln_slabs(rows);
        hipLaunchKernelGGL((ln_dw_kernel<T>), dim3(slabs, (n + 255) / 256), dim3(256), 0, st, (const T*)dy, lddy,
                           (const T*)x, ldx, rows, n, stats, ws);
        hipLaunchKernelGGL((ln_dw_finish_kernel<W>), dim3((n + 255) / 256), dim3(256), 0, st, ws, slabs, n, (W*)dw,
                           (W*)db);
    }
    SCA_CHECK_LAUNCH();
    return 0;
}

bool ln_types_ok(int dtype, int wtype) {
    return dtype >= SCA_F32 && dtype <= SCA_F16 && (wtype == SCA_F32 || wtype == dtype);
}

}  // namespace

#define LN_DISPATCH(FN, ...)                                                                   \
    (dtype == SCA_F32    ? FN<float, float>(__VA_ARGS__)                                       \
     : dtype == SCA_BF16 ? (wtype == SCA_F32 ? FN<sca_bf16, float>(__VA_ARGS__)                \
                                             : FN<sca_bf16, sca_bf16>(__VA_ARGS__))            \
                         : (wtype == SCA_F32 ? FN<sca_f16, float>(__VA_ARGS__)                 \
                                             : FN<sca_f16, sca_f16>(__VA_ARGS__)))

extern "C" int sca_layernorm_fwd(const void* x, long long ldx, int dtype, long long rows, int n, const void* w,
                                 const void* b, int wtype, float eps, void* y, long long ldy, float* stats,
                                 void* stream) {
    if (!ln_types_ok(dtype, wtype) || rows < 0 || n <= 0 || ldx < 0 || ldy < n || !(eps >= 0.f)) return -1;
    if (rows == 0) return 0;
    if (!x || !y) return -1;
    return LN_DISPATCH(ln_fwd, x, ldx, rows, n, w, b, eps, y, ldy, stats, (hipStream_t)stream);
}

extern "C" long long sca_layernorm_bwd_workspace_floats(long long rows, int n) {
    return rows < 0 || n <= 0 ? -1 : 2LL * n * ln_slabs(rows);
}

extern "C" int sca_layernorm_bwd(const void* dy, long long lddy, const void* x, long long ldx, int dtype,
                                 long long rows, int n, const void* w, int wtype, const float* stats, void* dx,
                                 long long lddx, void* dw, void* db, float* ws, void* stream) {
    if (!ln_types_ok(dtype, wtype) || rows < 0 || n <= 0 || lddy < 0 || ldx < 0 || (dx && lddx < n)) return -1;
    if (rows > 0 && (!dy || !x || !stats)) return -1;
    if ((dw || db) && !ws) return -1;
    return LN_DISPATCH(ln_bwd, dy, lddy, x, ldx, rows, n, w, stats, dx, lddx, dw, db, ws, (hipStream_t)stream);
}
