// AdamW over a list of tensors in one launch, with 32-bit or 8-bit states (gfx950).
//
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)        (decoupled decay)
//
// A step walks a table of tensors that lies in device memory (one entry per tensor, one per chunk of 2048 elements), so
// the number of tensors costs no launches.  The step numbers live in device memory as well, so that a captured step counts
// on when it is replayed: a small launch in front advances them and derives every tensor's coefficients (in 64 bits, once,
// instead of in every workgroup).  A caller that knows the step number gives it and does without that launch (3 us of 15
// for a small network); the numbers in memory are kept up all the same.
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

struct Coef {                       // what a step needs to know of a tensor
    float lr, step_size, inv_bc2, eps, clip;
    uint32_t t;
    uint32_t pad[2];
};
static_assert(sizeof(Coef) == 32, "sca_adamw_scratch_bytes");

// Of step t: lr / (1 - beta1^t) and 1 / sqrt(1 - beta2^t), without the cancellation.
__host__ __device__ inline Coef coef_of(int64_t t, float lr, float eps, double log_beta1, double log_beta2) {
    Coef c = {};
    c.lr = lr;
    c.step_size = lr / (float)-expm1((double)t * log_beta1);
    c.inv_bc2 = 1.0f / (float)sqrt(-expm1((double)t * log_beta2));
    c.eps = eps;
    c.t = (uint32_t)t;
    return c;
}

struct AdamWArgs {
    const sca_adamw_tensor* tensors;
    const sca_adamw_chunk* chunks;
    Coef* coef;                     // [n_tensors], or null: `given` for all
    Coef given;
    int64_t t;                      // with `given`: what the tensors' steps become
    int n_chunks, n_tensors;
    const float* hyper;             // sca_begin_step's block, or null: the scalars below and the tensors' own steps
    float lr, eps;
    double beta1, beta2, log_beta1, log_beta2;
    float b1, b2, one_minus_b1, one_minus_b2;       // 1 - beta taken in 64 bits: 1.0f - 0.999f is off by 1.3e-5
    uint64_t seed;
};

__global__ __launch_bounds__(256) void adamw_begin_kernel(const AdamWArgs a) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= a.n_tensors) return;
    const sca_adamw_tensor q = a.tensors[j];
    Coef c = {};
    if (a.hyper) {
        c.lr = a.hyper[1];
        c.step_size = a.hyper[1] / a.hyper[2];
        c.inv_bc2 = 1.0f / a.hyper[3];
        c.eps = a.hyper[4];
        c.clip = a.hyper[5];
    } else {
        const int64_t t = *q.step + 1;
        *q.step = t;
        c = coef_of(t, a.lr, a.eps, a.log_beta1, a.log_beta2);
    }
    a.coef[j] = c;
}

// New gradients for the tensors of a table: the addresses travel as the launch's arguments, so that nothing on the host has to
// outlive the call.  (zero_grad() drops the gradients and the next backward pass finds other storage for them, at every step
// of an ordinary loop; a new table costs 60 us there, this 4.)
constexpr int PER_LAUNCH = 384;
struct GradPointers { const void* g[PER_LAUNCH]; };
__global__ __launch_bounds__(PER_LAUNCH) void adamw_set_grads_kernel(sca_adamw_tensor* tensors, int n, const GradPointers p) {
    if ((int)threadIdx.x < n) tensors[threadIdx.x].g = p.g[threadIdx.x];
}

// p of four elements.  denom = sqrt(v) / sqrt(1 - b2^t) + eps; v_sqrt_f32 and v_rcp_f32 are good to one unit in the last
// place where their arguments are ordinary numbers, the exact sequences (some 25 instructions) are for what is near the
// denormal ones.
__device__ __forceinline__ void update(float (&p)[4], const float (&m)[4], const float (&v)[4], const Coef& c,
                                       float decay) {
    float denom[4], q[4], lo = 1e30f, hi = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        denom[k] = fmaf(__builtin_amdgcn_sqrtf(v[k]), c.inv_bc2, c.eps);
        q[k] = m[k] * __builtin_amdgcn_rcpf(denom[k]);
        lo = fminf(lo, denom[k]);
        hi = fmaxf(hi, denom[k]);
    }
    if (!(lo > 1e-17f && hi < 1e30f)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = m[k] / fmaf(sqrtf(v[k]), c.inv_bc2, c.eps);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = fmaf(-c.step_size, q[k], p[k] * decay);
}

// Addresses out of a table in memory are of no known kind to the compiler: told that they are device memory it takes the
// loads and stores for that, whose waits are counted in order.
template <typename T>
__device__ __forceinline__ T* global(const void* p) {
    return (T*)(__attribute__((address_space(1))) T*)(uintptr_t)p;
}

// What a launch reads only, and every lane alike: through the scalar cache.
template <typename T>
__device__ __forceinline__ const T* constant(const T* p) {
    return (const T*)(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// ---- 32-bit states ------------------------------------------------------------------------------------------------------
// 2 x 4 elements of a chunk: all loads first.  28 bytes and 22 instructions an element (fp32): bound by memory (173 M values
// 880 us, 5.5 TB/s).
template <typename T>
__device__ __forceinline__ void chunk32(const sca_adamw_tensor& q, long long i0, const Coef& c, const AdamWArgs& a) {
    float pv[2][4], gv[2][4], mv[2][4], vv[2][4];
    int left[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long i = i0 + h * 1024, l = q.n - i;
        left[h] = l >= 4 ? 4 : l > 0 ? (int)l : 0;
        const T *p = global<T>(q.p) + i, *g = global<T>(q.g) + i;
        const float *m = global<float>(q.m) + i, *v = global<float>(q.v) + i;
        if (q.vec && left[h] == 4) {
            load_vec<T, 4>(p, pv[h]); load_vec<T, 4>(g, gv[h]); load_vec<float, 4>(m, mv[h]); load_vec<float, 4>(v, vv[h]);
        } else {
            load_part<T, 4>(p, left[h], pv[h]); load_part<T, 4>(g, left[h], gv[h]);
            load_part<float, 4>(m, left[h], mv[h]); load_part<float, 4>(v, left[h], vv[h]);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long i = i0 + h * 1024;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float gk = gv[h][k];
            if (c.clip > 0.f) gk = fminf(fmaxf(gk, -c.clip), c.clip);
            mv[h][k] = fmaf(a.b1, mv[h][k], a.one_minus_b1 * gk);
            vv[h][k] = fmaf(a.b2, vv[h][k], a.one_minus_b2 * gk * gk);
        }
        update(pv[h], mv[h], vv[h], c, 1.0f - c.lr * q.weight_decay);
        T* p = global<T>(q.p) + i;
        float *m = global<float>(q.m) + i, *v = global<float>(q.v) + i;
        if (q.vec && left[h] == 4) {
            store_vec<T, 4>(p, pv[h]); store_vec<float, 4>(m, mv[h]); store_vec<float, 4>(v, vv[h]);
        } else {
            store_part<T, 4>(p, left[h], pv[h]); store_part<float, 4>(m, left[h], mv[h]);
            store_part<float, 4>(v, left[h], vv[h]);
        }
    }
}

// ---- 8-bit states -------------------------------------------------------------------------------------------------------
// Philox4x32-10 as in common.h, with one 32 x 32 -> 64 bit product per pair of halves.
__device__ __forceinline__ Philox4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(b >> 32), c1, k0, 0x96);       // a ^ b ^ c
        c1 = (uint32_t)b;
        c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(a >> 32), c3, k1, 0x96);
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    return Philox4{c0, c1, c2, c3};
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
    return o > v ? o : v;
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    v = dpp_umax<0xB1>(v);
    v = dpp_umax<0x4E>(v);
    v = dpp_umax<0x141>(v);
    v = dpp_umax<0x140>(v);
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 64; r += 16) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)v, r);
        m = o > m ? o : m;
    }
    return m;
}

// The 256 values x[lane][4] of a wave on the grid of an 8-bit float with MANT fraction bits and exponent bias BIAS, behind a
// power of two: the four codes of a lane, and the scale.  w: a random word per element, whose low (SIGNED: the first
// moment) or high half decides: of the two grid neighbours the upper one is taken where the way from the lower one is at
// least 1 - half / 65536.  For a normal number that is an integer addition to its bits in front of the cut; the numbers
// below 2^(1 - BIAS) scales, whose steps are of equal size, take a branch of their own.
template <int MANT, int BIAS, bool SIGNED>
__device__ __forceinline__ uint32_t to_grid(const float (&x)[4], const uint32_t (&w)[4], float& scale) {
    constexpr int TOP = MANT == 3 ? 8 : 15;             // the largest value is 1.75 * 2^TOP
    constexpr int DROP = 23 - MANT;
    uint32_t b[4], amax = 0, amin = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        b[i] = SIGNED ? __float_as_uint(x[i]) & 0x7fffffffu : __float_as_uint(x[i]);
        amax = b[i] > amax ? b[i] : amax;               // as integers: a NaN is above every number
        amin = b[i] < amin ? b[i] : amin;
    }
    amax = wave_umax(amax);
    if (amax == 0u || amax >= 0x7f800000u) {            // nothing, or not finite (then all 256 are NaN from now on)
        scale = amax == 0u ? 0.f : __uint_as_float(0x7fc00000u);
        return 0u;
    }
    int e = (int)(amax >> 23) - 127 - TOP + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < -126 ? -126 : e;
    scale = __uint_as_float((uint32_t)(e + 127) << 23);
    // code = ((bits of x / scale) + random bits) >> DROP, the exponent counted from the type's; dividing by 2^e is a
    // subtraction from the exponent
    const uint32_t shift = (uint32_t)(e + 127 - BIAS) << 23;
    uint32_t code[4], sign = 0;
    if (SIGNED) {                                       // the four sign bits as the codes' top bits
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x0c0c0703u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x07030c0cu);
        sign = (lo | hi) & 0x80808080u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t r = SIGNED ? (w[i] & 0xffffu) << (DROP - 16) : w[i] >> (32 - DROP) & ~((1u << (DROP - 16)) - 1u);
        code[i] = (b[i] - shift + r) >> DROP;
    }
    if (e + 128 - BIAS <= 0 || amin < (uint32_t)(e + 128 - BIAS) << 23) {
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t = __uint_as_float(b[i]) * inv;
            const uint32_t r = SIGNED ? w[i] & 0xffffu : w[i] >> 16;
            if (t < __uint_as_float((uint32_t)(128 - BIAS) << 23)) {
                const float f = t * __uint_as_float((uint32_t)(127 + BIAS - 1 + MANT + 16) << 23);
                code[i] = ((uint32_t)(int)f + r) >> 16;
                if (!SIGNED && code[i] == 0u && b[i] != 0u) code[i] = 1u;       // a positive moment stays positive
                if (SIGNED && code[i] == 0u) sign &= ~(0x80u << (8 * i));
            } else {
                code[i] = ((__float_as_uint(t) + (r << (DROP - 16))) >> DROP) - ((127 - BIAS) << MANT);
            }
        }
    }
    return (code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24) | sign;
}

// 2 x 4 elements of a chunk, a block of 256 per wave and half.  10 bytes (bf16) and 71 instructions an element, a
// third of them for the random bits and as many for the two roundings: bound by arithmetic (173 M bf16 values 430 us, 4.0
// TB/s; fp32 values 490 us, 5.7 TB/s; without the generator, or with the moments in 32 bits, the bf16 ones take 405).
template <typename T>
__device__ __forceinline__ void chunk8(const sca_adamw_tensor& q, long long i0, const Coef& c, const AdamWArgs& a) {
    float pv[2][4], gv[2][4], ms[2], vs[2];
    uint32_t mq[2], vq[2];
    int left[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long i = i0 + h * 1024, l = q.n - i;
        left[h] = l >= 4 ? 4 : l > 0 ? (int)l : 0;
        const T *p = global<T>(q.p) + i, *g = global<T>(q.g) + i;
        const uint8_t *m = global<uint8_t>(q.m) + i, *v = global<uint8_t>(q.v) + i;
        // (a wave whose block lies behind the tensor's end has nothing to do, and there is no scale of its block)
        const bool any = (i & ~(long long)(QBLOCK - 1)) < q.n;
        ms[h] = any ? global<float>(q.m_scale)[i / QBLOCK] : 0.f;
        vs[h] = any ? global<float>(q.v_scale)[i / QBLOCK] : 0.f;
        if (q.vec && left[h] == 4) {
            load_vec<T, 4>(p, pv[h]); load_vec<T, 4>(g, gv[h]);
            mq[h] = *(const uint32_t*)m; vq[h] = *(const uint32_t*)v;
        } else {
            load_part<T, 4>(p, left[h], pv[h]); load_part<T, 4>(g, left[h], gv[h]);
            mq[h] = vq[h] = 0u;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < left[h]) {
                    mq[h] |= (uint32_t)m[k] << (8 * k);
                    vq[h] |= (uint32_t)v[k] << (8 * k);
                }
        }
    }
    const double one_b1 = 1.0 - a.beta1, one_b2 = 1.0 - a.beta2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long i = i0 + h * 1024;
        if ((i & ~(long long)(QBLOCK - 1)) >= q.n) return;
        const double bm = a.beta1 * (double)ms[h], bv = a.beta2 * (double)vs[h];
        const float md[4] = {__builtin_amdgcn_cvt_f32_fp8((int)mq[h], 0), __builtin_amdgcn_cvt_f32_fp8((int)mq[h], 1),
                             __builtin_amdgcn_cvt_f32_fp8((int)mq[h], 2), __builtin_amdgcn_cvt_f32_fp8((int)mq[h], 3)};
        const float vd[4] = {__builtin_amdgcn_cvt_f32_bf8((int)vq[h], 0), __builtin_amdgcn_cvt_f32_bf8((int)vq[h], 1),
                             __builtin_amdgcn_cvt_f32_bf8((int)vq[h], 2), __builtin_amdgcn_cvt_f32_bf8((int)vq[h], 3)};
        float mn[4], vn[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double gd = (double)gv[h][k];
            mn[k] = (float)fma((double)md[k], bm, one_b1 * gd);
            vn[k] = (float)fma(one_b2 * gd, gd, (double)vd[k] * bv);
        }
        if (left[h] < 4) {                      // behind the end (a scale that is NaN must not get in)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                mn[k] = k < left[h] ? mn[k] : 0.f;
                vn[k] = k < left[h] ? vn[k] : 0.f;
            }
        }
        update(pv[h], mn, vn, c, 1.0f - c.lr * q.weight_decay);
        const Philox4 w = philox((uint32_t)(i >> 2), (uint32_t)((unsigned long long)i >> 34), (uint32_t)q.id, c.t,
                                 (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
        const uint32_t word[4] = {w.x, w.y, w.z, w.w};
        float msn, vsn;
        const uint32_t mc = to_grid<3, 7, true>(mn, word, msn), vc = to_grid<2, 15, false>(vn, word, vsn);
        T* p = global<T>(q.p) + i;
        uint8_t *m = global<uint8_t>(q.m) + i, *v = global<uint8_t>(q.v) + i;
        if (q.vec && left[h] == 4) {
            store_vec<T, 4>(p, pv[h]);
            *(uint32_t*)m = mc; *(uint32_t*)v = vc;
        } else {
            store_part<T, 4>(p, left[h], pv[h]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < left[h]) {
                    m[k] = (uint8_t)(mc >> (8 * k));
                    v[k] = (uint8_t)(vc >> (8 * k));
                }
        }
        if ((threadIdx.x & 63) == 0) {
            global<float>(q.m_scale)[i / QBLOCK] = msn;
            global<float>(q.v_scale)[i / QBLOCK] = vsn;
        }
    }
}

// One chunk per workgroup.  (As many workgroups as fit, each walking every so many chunks, take 20 % longer: they do not
// end together.)
template <int BITS>
__global__ __launch_bounds__(256, BITS == 8 ? 6 : 4) void adamw_kernel(const AdamWArgs a) {
    for (long long k = blockIdx.x; k < a.n_chunks; k += gridDim.x) {
        const sca_adamw_chunk ch = constant(a.chunks)[k];
        const sca_adamw_tensor q = constant(a.tensors)[ch.tensor];
        const Coef c = a.coef ? constant(a.coef)[ch.tensor] : a.given;
        const long long i = (long long)ch.index * CHUNK + 4 * threadIdx.x;
        if (BITS == 32) {
            if (q.dtype == SCA_F32) chunk32<float>(q, i, c, a);
            else if (q.dtype == SCA_BF16) chunk32<sca_bf16>(q, i, c, a);
            else chunk32<sca_f16>(q, i, c, a);
        } else {
            if (q.dtype == SCA_F32) chunk8<float>(q, i, c, a);
            else if (q.dtype == SCA_BF16) chunk8<sca_bf16>(q, i, c, a);
            else chunk8<sca_f16>(q, i, c, a);
        }
    }
    if (!a.coef && blockIdx.x == 0)             // (nothing in this launch reads the steps)
        for (int j = threadIdx.x; j < a.n_tensors; j += 256) *a.tensors[j].step = a.t;
}

}  // namespace

extern "C" int sca_adamw_chunk_elements(void) { return CHUNK; }
extern "C" int sca_adamw_block_elements(void) { return QBLOCK; }
extern "C" long long sca_adamw_scratch_bytes(int n_tensors) { return n_tensors < 0 ? -1 : (long long)n_tensors * sizeof(Coef); }

extern "C" int sca_adamw_set_grads(sca_adamw_tensor* tensors, int n_tensors, const void* const* grads, void* stream) {
    if (n_tensors < 0 || (n_tensors > 0 && (!tensors || !grads))) return -1;
    if (n_tensors == 0) return 0;
    for (int j = 0; j < n_tensors; j += PER_LAUNCH) {
        const int n = n_tensors - j < PER_LAUNCH ? n_tensors - j : PER_LAUNCH;
        GradPointers p = {};
        for (int i = 0; i < n; ++i) p.g[i] = grads[j + i];
        hipLaunchKernelGGL(adamw_set_grads_kernel, dim3(1), dim3(PER_LAUNCH), 0, (hipStream_t)stream, tensors + j, n, p);
    }
    SCA_CHECK_LAUNCH();
    return 0;
}

extern "C" int sca_adamw_step(const sca_adamw_tensor* tensors, int n_tensors, const sca_adamw_chunk* chunks,
                              int n_chunks, int state_bits, const float* hyper, long long t, float lr, double beta1,
                              double beta2, float eps, uint64_t seed, void* scratch, void* stream) {
    if (n_tensors < 0 || n_chunks < 0 || (state_bits != 32 && state_bits != 8) || t < 0) return -1;
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return -1;
    if (hyper ? state_bits != 32 || t != 0 : !(eps >= 0.f)) return -1;
    if (n_tensors == 0) return 0;
    if (!tensors || (n_chunks > 0 && !chunks)) return -1;
    if (t == 0 && (!scratch || ((uintptr_t)scratch & 15))) return -1;
    hipStream_t st = (hipStream_t)stream;
    AdamWArgs a{tensors, chunks, t ? nullptr : (Coef*)scratch, Coef{}, t, n_chunks, n_tensors, hyper, lr, eps, beta1, beta2,
                log(beta1), log(beta2), (float)beta1, (float)beta2, (float)(1.0 - beta1), (float)(1.0 - beta2), seed};
    if (t) a.given = coef_of(t, lr, eps, a.log_beta1, a.log_beta2);
    else hipLaunchKernelGGL(adamw_begin_kernel, dim3((n_tensors + 255) / 256), dim3(256), 0, st, a);
    int grid = n_chunks < (1 << 23) ? n_chunks : 1 << 23;               // fewer than 2^32 threads
    if (t && grid == 0) grid = 1;                                       // (the steps)
    if (grid > 0 && state_bits == 32) hipLaunchKernelGGL((adamw_kernel<32>), dim3(grid), dim3(256), 0, st, a);
    else if (grid > 0) hipLaunchKernelGGL((adamw_kernel<8>), dim3(grid), dim3(256), 0, st, a);
    SCA_CHECK_LAUNCH();
    return 0;
}
