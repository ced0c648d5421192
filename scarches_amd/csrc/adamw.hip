// AdamW over a list of tensors in one launch, with 32-bit or 8-bit states (gfx950).
//
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)        (decoupled decay)
//
// A launch walks a table of tensors that lies in device memory (one entry per tensor, one per chunk of 2048 elements), so
// the number of tensors costs no launches.  The step number lives in device memory as well: the last workgroup to finish
// advances it, so a captured step counts on when it is replayed.
//
// 8-bit states: every 256 elements of a tensor share a power-of-two scale per moment, with m / scale held as e4m3 and
// v / scale as e5m2 floats (v spans twice the exponents of m).  Rounding to that grid is stochastic: at b2 = 0.999 a step
// moves v by 0.1 %, far below the grid's 12.5 - 25 %, and rounding to the nearest would never let it move at all; the
// random bits are Philox words of (element, tensor, step) under the caller's seed, so a run repeats bit for bit.  A
// positive v is never rounded to 0 (its m would then be divided by eps alone).  The moments are evaluated in 64 bits and
// rounded once to 32 before they go to the grid: which of two codes is taken does not depend on the order of the
// arithmetic.  (The update itself uses the moments before they are rounded to 8 bits.)
#include "common.h"
#include "dtypes.h"
#include "adamw_table.h"

namespace {

constexpr int CHUNK = 2048;         // elements per table chunk: 8 per thread, loads of a chunk in flight together
constexpr int QBLOCK = 256;         // elements per 8-bit scale: one wave, four consecutive elements per lane

struct AdamWArgs {
    const sca_adamw_tensor* tensors;
    const sca_adamw_chunk* chunks;
    int n_chunks, n_tensors;
    const float* hyper;             // sca_begin_step's block, or null: the scalars below and the tensors' own steps
    float lr, eps;
    double beta1, beta2, log_beta1, log_beta2;
    float b1, b2, one_minus_b1, one_minus_b2;       // 1 - beta taken in 64 bits: 1.0f - 0.999f is off by 1.3e-5
    uint64_t seed;
    unsigned* done;                 // 0 before and after every launch
};

struct Coef {
    float decay, step_size, inv_bc2, eps, clip;
    uint32_t t;
};

__device__ __forceinline__ Coef coefficients(const AdamWArgs& a, const sca_adamw_tensor& q) {
    Coef c;
    float lr, bc1, bc2s;
    if (a.hyper) {
        lr = a.hyper[1]; bc1 = a.hyper[2]; bc2s = a.hyper[3]; c.eps = a.hyper[4]; c.clip = a.hyper[5]; c.t = 0;
    } else {
        const double t = (double)(*q.step + 1);
        lr = a.lr;
        bc1 = (float)-expm1(t * a.log_beta1);           // 1 - beta^t without the cancellation
        bc2s = (float)sqrt(-expm1(t * a.log_beta2));
        c.eps = a.eps; c.clip = 0.f; c.t = (uint32_t)(*q.step + 1);
    }
    c.decay = 1.0f - lr * q.weight_decay;
    c.step_size = lr / bc1;
    c.inv_bc2 = 1.0f / bc2s;
    return c;
}

__device__ __forceinline__ float updated(float p, float m, float v, const Coef& c) {
    return fmaf(-c.step_size, m / fmaf(sqrtf(v), c.inv_bc2, c.eps), p * c.decay);
}

// The 256 values x[lane][4] of a wave on the grid of an 8-bit float with MANT fraction bits and exponent bias BIAS,
// behind a power of two: the four codes of a lane, and the scale.  rnd: 16 random bits per element; of the two grid
// neighbours the upper one is taken where the way from the lower one exceeds 1 - rnd / 65536.
template <int MANT, int BIAS, bool LEAST>
__device__ __forceinline__ uint32_t to_grid(const float (&x)[4], const uint32_t (&rnd)[4], float& scale) {
    constexpr int TOP = MANT == 3 ? 8 : 15;             // the largest value is 1.75 * 2^TOP
    constexpr int DROP = 23 - MANT;
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
        amax = b > amax ? b : amax;                     // as integers: a NaN is above every number
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t b = __shfl_xor(amax, o, 64);
        amax = b > amax ? b : amax;
    }
    if (amax == 0u || amax >= 0x7f800000u) {            // nothing, or not finite (then all 256 are NaN from now on)
        scale = amax == 0u ? 0.f : __uint_as_float(0x7fc00000u);
        return 0u;
    }
    int e = (int)(amax >> 23) - 127 - TOP + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < -126 ? -126 : e;
    scale = __uint_as_float((uint32_t)(e + 127) << 23);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float t = fabsf(x[i]) * inv;
        uint32_t code;
        if (t < __uint_as_float((uint32_t)(128 - BIAS) << 23)) {        // below 2^(1 - BIAS): steps of equal size
            const float f = t * __uint_as_float((uint32_t)(127 + BIAS - 1 + MANT + 16) << 23);
            code = ((uint32_t)(int)f + rnd[i]) >> 16;
        } else {
            code = ((__float_as_uint(t) + (rnd[i] << (DROP - 16))) >> DROP) - ((127 - BIAS) << MANT);
        }
        if (LEAST && code == 0u && x[i] > 0.f) code = 1u;
        if (!LEAST && code != 0u && x[i] < 0.f) code |= 0x80u;
        out |= code << (8 * i);
    }
    return out;
}

template <typename T>
__device__ __forceinline__ void step32(const sca_adamw_tensor& q, long long i, int left, const Coef& c,
                                       const AdamWArgs& a) {
    T* p = (T*)q.p + i;
    const T* g = (const T*)q.g + i;
    float *m = (float*)q.m + i, *v = (float*)q.v + i;
    float pv[4], gv[4], mv[4], vv[4];
    const bool whole = q.vec && left >= 4;
    if (whole) {
        load_vec<T, 4>(p, pv); load_vec<T, 4>(g, gv); load_vec<float, 4>(m, mv); load_vec<float, 4>(v, vv);
    } else {
        load_part<T, 4>(p, left, pv); load_part<T, 4>(g, left, gv); load_part<float, 4>(m, left, mv);
        load_part<float, 4>(v, left, vv);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float gk = gv[k];
        if (c.clip > 0.f) gk = fminf(fmaxf(gk, -c.clip), c.clip);
        mv[k] = fmaf(a.b1, mv[k], a.one_minus_b1 * gk);
        vv[k] = fmaf(a.b2, vv[k], a.one_minus_b2 * gk * gk);
        pv[k] = updated(pv[k], mv[k], vv[k], c);
    }
    if (whole) {
        store_vec<T, 4>(p, pv); store_vec<float, 4>(m, mv); store_vec<float, 4>(v, vv);
    } else {
        store_part<T, 4>(p, left, pv); store_part<float, 4>(m, left, mv); store_part<float, 4>(v, left, vv);
    }
}

template <typename T>
__device__ __forceinline__ void step8(const sca_adamw_tensor& q, long long i, int left, const Coef& c, const AdamWArgs& a) {
    T* p = (T*)q.p + i;
    const T* g = (const T*)q.g + i;
    uint8_t *m = (uint8_t*)q.m + i, *v = (uint8_t*)q.v + i;
    const long long blk = i / QBLOCK;
    float pv[4], gv[4], mn[4], vn[4];
    uint32_t mq = 0, vq = 0;
    const bool whole = q.vec && left >= 4;
    if (whole) {
        load_vec<T, 4>(p, pv); load_vec<T, 4>(g, gv);
        mq = *(const uint32_t*)m; vq = *(const uint32_t*)v;
    } else {
        load_part<T, 4>(p, left, pv); load_part<T, 4>(g, left, gv);
        for (int k = 0; k < 4; ++k)
            if (k < left) {
                mq |= (uint32_t)m[k] << (8 * k);
                vq |= (uint32_t)v[k] << (8 * k);
            }
    }
    // (a wave whose block lies behind the tensor's end has nothing to do; the scale of its block does not exist)
    const bool any = (i & ~(long long)(QBLOCK - 1)) < q.n;
    const double ms = any ? (double)q.m_scale[blk] : 0.0, vs = any ? (double)q.v_scale[blk] : 0.0;
    const float md[4] = {__builtin_amdgcn_cvt_f32_fp8((int)mq, 0), __builtin_amdgcn_cvt_f32_fp8((int)mq, 1),
                         __builtin_amdgcn_cvt_f32_fp8((int)mq, 2), __builtin_amdgcn_cvt_f32_fp8((int)mq, 3)};
    const float vd[4] = {__builtin_amdgcn_cvt_f32_bf8((int)vq, 0), __builtin_amdgcn_cvt_f32_bf8((int)vq, 1),
                         __builtin_amdgcn_cvt_f32_bf8((int)vq, 2), __builtin_amdgcn_cvt_f32_bf8((int)vq, 3)};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const double gd = (double)gv[k];
        mn[k] = k < left ? (float)fma(a.beta1, (double)md[k] * ms, (1.0 - a.beta1) * gd) : 0.f;
        vn[k] = k < left ? (float)fma(a.beta2, (double)vd[k] * vs, (1.0 - a.beta2) * gd * gd) : 0.f;
        pv[k] = updated(pv[k], mn[k], vn[k], c);
    }
    const Philox4 w = philox4x32_10((uint32_t)(i >> 2), (uint32_t)((unsigned long long)i >> 34), (uint32_t)q.id, c.t,
                                    (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
    const uint32_t wm[4] = {w.x & 0xffffu, w.y & 0xffffu, w.z & 0xffffu, w.w & 0xffffu};
    const uint32_t wv[4] = {w.x >> 16, w.y >> 16, w.z >> 16, w.w >> 16};
    float msn, vsn;
    mq = to_grid<3, 7, false>(mn, wm, msn);
    vq = to_grid<2, 15, true>(vn, wv, vsn);
    if (!any) return;
    if (whole) {
        store_vec<T, 4>(p, pv);
        *(uint32_t*)m = mq; *(uint32_t*)v = vq;
    } else {
        store_part<T, 4>(p, left, pv);
        for (int k = 0; k < 4; ++k)
            if (k < left) {
                m[k] = (uint8_t)(mq >> (8 * k));
                v[k] = (uint8_t)(vq >> (8 * k));
            }
    }
    if ((threadIdx.x & 63) == 0) {
        q.m_scale[blk] = msn;
        q.v_scale[blk] = vsn;
    }
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamWArgs a) {
    for (int k = blockIdx.x; k < a.n_chunks; k += gridDim.x) {
        const sca_adamw_chunk ch = a.chunks[k];
        const sca_adamw_tensor q = a.tensors[ch.tensor];
        const Coef c = coefficients(a, q);
        for (int h = 0; h < CHUNK; h += 1024) {
            const long long i = (long long)ch.index * CHUNK + h + 4 * threadIdx.x;
            const long long l = q.n - i;
            const int left = l >= 4 ? 4 : l > 0 ? (int)l : 0;
            if (BITS == 32) {
                if (left <= 0) continue;
                if (q.dtype == SCA_F32) step32<float>(q, i, left, c, a);
                else if (q.dtype == SCA_BF16) step32<sca_bf16>(q, i, left, c, a);
                else step32<sca_f16>(q, i, left, c, a);
            } else {
                if (q.dtype == SCA_F32) step8<float>(q, i, left, c, a);
                else if (q.dtype == SCA_BF16) step8<sca_bf16>(q, i, left, c, a);
                else step8<sca_f16>(q, i, left, c, a);
            }
        }
    }
    if (a.hyper) return;
    // every workgroup has read the steps it needs before it counts itself done; the last one advances them
    __shared__ unsigned last;
    __syncthreads();
    if (threadIdx.x == 0) last = __hip_atomic_fetch_add(a.done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (last != gridDim.x - 1) return;
    for (int j = threadIdx.x; j < a.n_tensors; j += 256) *a.tensors[j].step += 1;
    if (threadIdx.x == 0) *a.done = 0u;
}

}  // namespace

extern "C" int sca_adamw_chunk_elements(void) { return CHUNK; }
extern "C" int sca_adamw_block_elements(void) { return QBLOCK; }

extern "C" int sca_adamw_step(const sca_adamw_tensor* tensors, int n_tensors, const sca_adamw_chunk* chunks,
                              int n_chunks, int state_bits, const float* hyper, float lr, double beta1, double beta2,
                              float eps, uint64_t seed, uint32_t* done, void* stream) {
    if (n_tensors < 0 || n_chunks < 0 || (state_bits != 32 && state_bits != 8)) return -1;
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return -1;
    if (!hyper && !(eps >= 0.f && done)) return -1;
    if (hyper && state_bits != 32) return -1;
    if (n_tensors == 0) return 0;
    if (!tensors || (n_chunks > 0 && !chunks)) return -1;
    AdamWArgs a{tensors, chunks, n_chunks, n_tensors, hyper, lr, eps, beta1, beta2, log(beta1), log(beta2),
                (float)beta1, (float)beta2, (float)(1.0 - beta1), (float)(1.0 - beta2), seed, (unsigned*)done};
    int grid = n_chunks < 2048 ? n_chunks : 2048;
    if (grid < 1) grid = 1;
    if (state_bits == 32) hipLaunchKernelGGL((adamw_kernel<32>), dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((adamw_kernel<8>), dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    SCA_CHECK_LAUNCH();
    return 0;
}
