// Matrix product in 8-bit integers with a scale per row and per output channel (gfx950).
//
//   rows:    s_m = max_k |x_mk| / 127 (fp32),  q_mk = round(x_mk / s_m), ties to even     (sca_quant_rows_i8)
//   product: y_mn = (sum_k q_mk w_nk) * s_m * s_n + bias_n                                (sca_gemm_i8)
//
// The sum is exact in int32 (k < 2^31 / 128^2), so its order does not matter; the product is v_mfma_i32_*_i8.
#include "common.h"
#include "dtypes.h"
#include "rowtile.h"
#include <type_traits>

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

namespace {

// What a row's largest magnitude (as bits: a NaN is above every number) makes of its values.
//
// inv: of the two fp32 numbers around 1 / s the one on the same side of 127 / amax as 1 / s itself.  Values of a short type
// lie half way between two steps of amax / 127 all the time; s, which is that rounded, puts them to one side by the rounding's
// 2^-24, and an estimate x * inv with that property to the same side.  (With the nearest inv nearly every vector of a bf16
// row holds a value that has to be corrected.)
struct RowScale {
    float s, inv, half;
    uint32_t keep;               // 0: a row of zeros, or with a value that is not finite
    bool tiny;                   // 1 / s is not a number of this type: the quotient in 64 bits
    __device__ __forceinline__ explicit RowScale(uint32_t bits) {
        const float amax = __uint_as_float(bits);
        s = bits < 0x7f800000u ? amax / 127.f : __uint_as_float(0x7fc00000u);
        keep = s > 0.f ? 0xffffffffu : 0u;
        tiny = s > 0.f && s < 1e-37f;
        inv = keep ? 1.f / s : 0.f;
        half = 0.5f * s;
        const float side = fmaf(-127.f, s, amax), got = fmaf(inv, amax, -127.f);       // (one rounding each: exact signs)
        if (keep && side > 0.f && !(got > 0.f)) inv = __uint_as_float(__float_as_uint(inv) + 1u);
        if (keep && side < 0.f && !(got < 0.f)) inv = __uint_as_float(__float_as_uint(inv) - 1u);
    }
};
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// q = round(x / s) of VEC values, ties to even, with the exact quotient, packed; not for a tiny scale.  x / s + 1.5 * 2^23 in
// one fma is an integer whose low byte is q in two's complement.  The estimate may fall on the other side of a middle, so its
// distance from x is taken without rounding (one fma: q s has at most 31 bits and the difference at most 24), and where one
// of the values is half a step or more away from its q, all are put right: a branch per vector, seldom taken.  (8192 rows
// of 4096 bf16 values: 18 us, the rate of a copy; a comparison and a choice for every value takes 55.)
template <int VEC>
__device__ __forceinline__ void quantized(const RowScale& sc, const float (&v)[VEC], uint32_t (&w)[VEC / 4]) {
    constexpr float MAGIC = 12582912.f;
    float t[VEC], far = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        t[i] = fmaf(v[i], sc.inv, MAGIC);
        far = fmaxf(far, fabsf(fmaf(-(t[i] - MAGIC), sc.s, v[i])));
    }
    if (far >= sc.half) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            // beyond half a step, or at it with an odd q: the neighbour.  (|d| + the last bit of q, as integers, > half)
            const float d = fmaf(-(t[i] - MAGIC), sc.s, v[i]);
            if (magnitude(d) + (__float_as_uint(t[i]) & 1u) > __float_as_uint(sc.half)) t[i] += copysignf(1.f, d);
        }
    }
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 1]), __float_as_uint(t[4 * i]), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 3]), __float_as_uint(t[4 * i + 2]), 0x04000c0cu);
        w[i] = (lo | hi) & sc.keep;
    }
}

// A row whose scale is below what fp32 can invert: element by element, the quotient in 64 bits.
template <typename T>
__device__ __noinline__ void quantize_tiny(const T* x, int k, int8_t* q, float s, int t, int step) {
    for (int c = t; c < k; c += step)
        q[c] = (int8_t)(int)fmin(fmax(rint((double)to_f32(x[c]) / (double)s), -127.0), 127.0);
}

// 16 bytes at p, of which `left` belong to the row of K bytes (what lies behind counts as 0).  The row's end is read as the 16
// bytes that end with it, moved down: a byte at a time takes sixteen loads (a row shorter than that has no other way).
__device__ __forceinline__ i32x4 load16(const int8_t* p, int left, int K) {
    i32x4 v = {0, 0, 0, 0};
    if (left >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else if (left > 0 && K >= 16) {
        uint64_t w[2];
        __builtin_memcpy(w, p - (16 - left), 16);
        const int shift = 8 * (16 - left);
        const uint64_t lo = shift < 64 ? w[0] >> shift | w[1] << 1 << (63 - shift) : w[1] >> (shift - 64);
        w[1] = shift < 64 ? w[1] >> shift : 0;
        w[0] = lo;
        __builtin_memcpy(&v, w, 16);
    } else if (left > 0) {
        int8_t b[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = i < left ? p[i] : 0;
        __builtin_memcpy(&v, b, 16);
    }
    return v;
}

// Rows of a weight to a pitch whose rows start 16-byte aligned, zeros behind them: workgroups `first` and up of the launch that
// quantizes x beside it.
struct AlignRows {
    const int8_t* w; long long ldw;
    int n, k;
    int8_t* to; long long pitch;
    unsigned first;
};
__device__ __forceinline__ unsigned blocks_left() { return gridDim.x; }
__device__ __forceinline__ unsigned blocks_left(const AlignRows& a) { return a.first; }
template <int NT>
__device__ __forceinline__ void align_rows(const AlignRows& a) {
    for (long long r = blockIdx.x - a.first; r < a.n; r += gridDim.x - a.first)
        for (long long c = threadIdx.x * 16; c < a.pitch; c += NT * 16)
            *(i32x4*)(a.to + r * a.pitch + c) = load16(a.w + r * a.ldw + c, a.k - (int)c, a.k);
}

// TPR threads per row, the row in registers: one read of 16 bytes a lane, one write.  Bound by memory.  Rows: nothing, or
// AlignRows (arguments and a branch that are of no use cost 3 % of small calls).
template <typename T, int TPR, int V, int MODE, typename... Rows>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void quant_rows_kernel(const T* __restrict__ x, long long ldx,
                                                                           long long rows, int k, int8_t* __restrict__ q,
                                                                           long long ldq, float* __restrict__ scale,
                                                                           const Rows... al) {
    constexpr int VEC = vec_of<T>(), NT = TPR > 256 ? TPR : 256;
    __shared__ uint32_t scratch[16];
    const int t = threadIdx.x % TPR;
    if constexpr (sizeof...(Rows) > 0) {
        if (blockIdx.x >= blocks_left(al...)) return align_rows<NT>(al...);
    }
    for (long long r = (long long)blockIdx.x * (NT / TPR) + threadIdx.x / TPR; r < rows;
         r += (long long)blocks_left(al...) * (NT / TPR)) {
        const T* xr = x + r * ldx;
        raw_t x16[V] = {};
        float v[VEC];
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Cols<T, TPR, MODE> at(j, t, k);
            if (at.there) load_cols<MODE>(xr, at.c, k, x16[j]);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            unpack<T>(x16[j], v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) amax = magnitude(v[i]) > amax ? magnitude(v[i]) : amax;
        }
        const RowScale sc(row_umax<TPR>(amax, scratch));
        int8_t* qr = q + r * ldq;
        if (sc.tiny) {
            quantize_tiny(xr, k, qr, sc.s, t, TPR);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const Cols<T, TPR, MODE> at(j, t, k);
                uint32_t w[VEC / 4];
                unpack_again<T>(x16[j], v);
                quantized<VEC>(sc, v, w);
                if (!at.there) continue;
                if (MODE == ROW_TINY)
                    for (int i = 0; i < k; ++i) qr[i] = (int8_t)(w[i / 4] >> (8 * (i & 3)));
                else __builtin_memcpy(qr + at.c, w, VEC);
            }
        }
        for (long long c = (long long)k + t; c < ldq; c += TPR) qr[c] = 0;
        if (t == 0) scale[r] = sc.s;
    }
}

// Rows beyond what a workgroup's registers hold: one workgroup per row, read twice (the second time from a cache).
template <typename T>
__global__ __launch_bounds__(1024) void quant_rows_long_kernel(const T* __restrict__ x, long long ldx, long long rows,
                                                               int k, int8_t* __restrict__ q, long long ldq,
                                                               float* __restrict__ scale) {
    constexpr int VEC = vec_of<T>();
    __shared__ uint32_t scratch[16];
    float v[VEC];
    const int vecs = (k + VEC - 1) / VEC;
    for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        int8_t* qr = q + r * ldq;
        uint32_t amax = 0;
        for (int j = threadIdx.x; j < vecs; j += 1024) {
            load_vec<T, VEC>(xr + (j * VEC < k - VEC ? j * VEC : k - VEC), v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) amax = magnitude(v[i]) > amax ? magnitude(v[i]) : amax;
        }
        const RowScale sc(row_umax<1024>(amax, scratch));
        if (sc.tiny) {
            quantize_tiny(xr, k, qr, sc.s, threadIdx.x, 1024);
        } else {
            for (int j = threadIdx.x; j < vecs; j += 1024) {
                const int c = j * VEC < k - VEC ? j * VEC : k - VEC;
                load_vec<T, VEC>(xr + c, v);
                uint32_t w[VEC / 4];
                quantized<VEC>(sc, v, w);
                __builtin_memcpy(qr + c, w, VEC);
            }
        }
        for (long long c = (long long)k + threadIdx.x; c < ldq; c += 1024) qr[c] = 0;
        if (threadIdx.x == 0) scale[r] = sc.s;
    }
}

// Rows of a CSR matrix (canonical: one entry per row and column), log(1 + x) on the way: what sca_csr_gather_rows and
// quant_rows_kernel give, without the dense fp32 rows between them, nearly all of which are zeros (8192 cells of 284 stored
// counts in 2000 genes: 14 us instead of 17 + 13.6).  One wave per row, which is put together in LDS; the first HELD stored
// values of a lane stay in registers between the maximum and the quotients, what is beyond them is read again.
constexpr int CSR_LDS = 65536;

__global__ __launch_bounds__(64) void csr_quant_rows_kernel(const int64_t* __restrict__ indptr,
                                                            const int32_t* __restrict__ indices,
                                                            const float* __restrict__ data,
                                                            const int64_t* __restrict__ row_ids, int log1p,
                                                            int8_t* __restrict__ q, int ldq, float* __restrict__ scale) {
    extern __shared__ __attribute__((aligned(16))) int8_t row[];
    constexpr int HELD = 8;
    const long long b = blockIdx.x, r = row_ids ? row_ids[b] : b;
    const int64_t first = indptr[r], s = first + threadIdx.x, e = indptr[r + 1];
    const int held = e - first >= HELD * 64 ? HELD : (int)((e - first + 63) / 64);      // (the logarithms are what it waits for)
    float v[HELD];
    int g[HELD];
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const bool there = s + j * 64 < e;
        v[j] = there ? data[s + j * 64] : 0.f;
        g[j] = there ? indices[s + j * 64] : -1;
    }
    for (int c = threadIdx.x * 16; c < ldq; c += 1024) *(i32x4*)(row + c) = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        if (j >= held) break;
        if (log1p) v[j] = log1pf(v[j]);
        amax = magnitude(v[j]) > amax ? magnitude(v[j]) : amax;
    }
    for (int64_t k = s + HELD * 64; k < e; k += 64) {
        const float x = log1p ? log1pf(data[k]) : data[k];
        amax = magnitude(x) > amax ? magnitude(x) : amax;
    }
    const RowScale sc(row_umax<64>(amax, nullptr));
    auto put = [&](const float (&x)[4], const int* at) {
        uint32_t w[1];
        quantized<4>(sc, x, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (sc.tiny) w[0] = (uint32_t)(int)fmin(fmax(rint((double)x[i] / (double)sc.s), -127.0), 127.0) << (8 * i);
            if (at[i] >= 0) row[at[i]] = (int8_t)(w[0] >> (8 * i));
        }
    };
    __syncthreads();
#pragma unroll
    for (int j = 0; j < HELD; j += 4) {
        if (j >= held) break;
        const float x[4] = {v[j], v[j + 1], v[j + 2], v[j + 3]};
        put(x, g + j);
    }
    for (int64_t k = s + HELD * 64; k < e; k += 64) {
        const float x[4] = {log1p ? log1pf(data[k]) : data[k], 0.f, 0.f, 0.f};
        const int at[4] = {indices[k], -1, -1, -1};
        put(x, at);
    }
    __syncthreads();
    for (int c = threadIdx.x * 16; c < ldq; c += 1024) *(i32x4*)(q + b * ldq + c) = *(const i32x4*)(row + c);
    if (threadIdx.x == 0) scale[b] = sc.s;
}

struct I8Args {
    const int8_t* x; long long ldx; const float* sx;
    const int8_t* w; long long ldw; const float* sw;
    const void* bias; int btype;
    void* y; int ytype; long long ldy;
    long long M; int N, K;
    int tiles_m, tiles_n;
};

// y[m][n] from the finished sum: three roundings in fp32, one to the result's type.
__device__ __forceinline__ float scaled(int acc, float sx, float sw, float add) { return fmaf((float)acc * sx, sw, add); }
__device__ __forceinline__ void put(const I8Args& a, long long o, float v) {
    if (a.ytype == SCA_F32) ((float*)a.y)[o] = v;
    else if (a.ytype == SCA_BF16) ((sca_bf16*)a.y)[o] = from_f32<sca_bf16>(v);
    else ((sca_f16*)a.y)[o] = from_f32<sca_f16>(v);
}
__device__ __forceinline__ float bias_at(const I8Args& a, int n) {
    if (!a.bias) return 0.f;
    return a.btype == SCA_F32    ? ((const float*)a.bias)[n]
           : a.btype == SCA_BF16 ? to_f32(((const sca_bf16*)a.bias)[n])
                                 : to_f32(((const sca_f16*)a.bias)[n]);
}

// ---- few rows or little work: fragments straight from memory --------------------------------------------------------
// A workgroup of 8 waves owns a 16 x 16 tile of the result; the waves take the k steps in turn and their sums meet in LDS.
// No staging, no barrier in the k loop: every wave has its whole share of both operands in flight.
// T = int8_t: x is quantized.  Else every workgroup quantizes the (at most QUANT_ROWS) rows itself, into LDS, while its
// weights are on their way: for single rows a launch of its own costs more than this repeated work (1 x 4096 x 4000:
// 5.9 us instead of 2.9 + 4.9; four rows took 11.2 instead of 9.2).
constexpr int QUANT_ROWS = 2, QUANT_K = 8192;

// Columns [c, c + VEC) of a row of n; what lies behind the end reads as 0.
template <typename T, int VEC>
__device__ __forceinline__ void load_end(const T* __restrict__ row, int c, int n, float (&v)[VEC]) {
    if (c + VEC <= n) load_vec<T, VEC>(row + c, v);
    else load_part<T, VEC>(row + c, n - c, v);
}

template <typename T>
__global__ __launch_bounds__(512) void gemm_i8_direct_kernel(const I8Args a) {
    constexpr bool FUSED = !std::is_same<T, int8_t>::value;
    __shared__ int part[7][256];
    __shared__ float xs[QUANT_ROWS];
    __shared__ uint32_t amax[QUANT_ROWS];
    __shared__ __attribute__((aligned(16))) int8_t xq[FUSED ? QUANT_ROWS * QUANT_K : 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long m0 = (long long)(blockIdx.x % a.tiles_m) * 16;
    const int n0 = (int)(blockIdx.x / a.tiles_m) * 16;
    const long long m = m0 + (lane & 15), last = a.M - 1;
    const int n = n0 + (lane & 15), nn = n < a.N ? n : a.N - 1, ko = (lane >> 4) * 16;
    const int8_t* wp = a.w + (long long)nn * a.ldw + ko;
    // scales and bias are asked for ahead of the k loop: behind it a wave would wait for each
    const long long r0 = m0 + (lane >> 4) * 4;
    float sx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sx[i] = FUSED || wave ? 0.f : a.sx[r0 + i < last ? r0 + i : last];
    const float s = a.sw[nn], add = bias_at(a, nn);
    constexpr int U = 4;                         // k steps of 64 bytes whose loads are issued together
    i32x4 av[U], bv[U];
    auto load = [&](const int8_t* p, int k0, i32x4 (&v)[U]) {
        if (k0 + 64 * U <= a.K) {
#pragma unroll
            for (int u = 0; u < U; ++u) __builtin_memcpy(&v[u], p + k0 + u * 64, 16);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = load16(p + k0 + u * 64, a.K - k0 - u * 64 - ko, a.K);
        }
    };
    const int k_first = wave * 64 * U;
    if (k_first < a.K) load(wp, k_first, bv);
    const int8_t* xp;
    if constexpr (FUSED) {
        constexpr int VEC = vec_of<typename std::conditional<FUSED, T, float>::type>();
        const int M = (int)a.M, kp = (a.K + 16 * VEC - 1) / (16 * VEC) * (16 * VEC);     // (a multiple of 64)
        if (threadIdx.x < QUANT_ROWS) amax[threadIdx.x] = 0u;
        __syncthreads();
        float v[VEC];
        for (int r = 0; r < M; ++r) {
            uint32_t big = 0;
            for (int c = threadIdx.x * VEC; c < a.K; c += 512 * VEC) {
                load_end((const T*)(const void*)a.x + r * a.ldx, c, a.K, v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) big = magnitude(v[i]) > big ? magnitude(v[i]) : big;
            }
            big = row_umax<64>(big, nullptr);
            if (lane == 0) atomicMax(&amax[r], big);
        }
        __syncthreads();
        for (int r = 0; r < M; ++r) {
            const RowScale sc(amax[r]);
            const T* xr = (const T*)(const void*)a.x + r * a.ldx;
            for (int c = threadIdx.x * VEC; c < kp; c += 512 * VEC) {
                uint32_t w[VEC / 4];
                load_end(xr, c, a.K, v);
                quantized<VEC>(sc, v, w);
                __builtin_memcpy(xq + r * kp + c, w, VEC);
            }
            if (sc.tiny) {
                __syncthreads();
                quantize_tiny(xr, a.K, xq + r * kp, sc.s, threadIdx.x, 512);
            }
            if (threadIdx.x == 0) xs[r] = sc.s;
        }
        __syncthreads();
        xp = xq + ((lane & 15) < M ? (lane & 15) : M - 1) * kp + ko;
#pragma unroll
        for (int i = 0; i < 4; ++i) sx[i] = xs[r0 + i < M ? r0 + i : M - 1];
    } else {
        xp = a.x + (m < last ? m : last) * a.ldx + ko;
    }
    i32x4 acc = {0, 0, 0, 0};
    for (int k0 = k_first; k0 < a.K; k0 += 8 * 64 * U) {
        if (k0 != k_first) load(wp, k0, bv);
        if constexpr (FUSED) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (k0 + u * 64 < a.K) av[u] = *(const i32x4*)(xp + k0 + u * 64);
                else av[u] = i32x4{0, 0, 0, 0};
        } else {
            load(xp, k0, av);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[u], bv[u], acc, 0, 0, 0);
    }
    if (wave) {
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave - 1][i * 64 + lane] = acc[i];
    }
    __syncthreads();
    if (wave || n >= a.N) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 7; ++q) acc[i] += part[q][i * 64 + lane];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r0 + i < a.M) put(a, (r0 + i) * a.ldy + n, scaled(acc[i], sx[i], s, add));
}

// ---- tiles through LDS ----------------------------------------------------------------------------------------------
// A BM x BN tile per workgroup in steps of KB bytes of k through a ring of NS stages in LDS.  A row of a stage is KB bytes =
// KB / 16 chunks; row r holds chunk c at place c ^ swap(r), such that the 16 lanes that read together (16 rows, one chunk)
// touch all 64 banks once.  WM x WN waves, each (BM / WM) x (BN / WN) of the tile in 32 x 32 MFMA blocks.  KS > 1: KS such
// groups of waves share the tile, each with its own stages and every KS-th k step, and add up through LDS.
template <int KB>
__device__ __forceinline__ int swap_of(int r) { return KB == 128 ? (r >> 1) & 7 : (r >> 2) & 3; }

// Rows [r0, r0 + ROWS) of an operand at byte k0 of every row to LDS without a register in between; NT threads, thread t.
// The loads write lane after lane, so the permutation is in which chunk a lane asks for.  Rows behind the last one repeat
// it (what comes of them is not stored).
template <int ROWS, int KB, int NT>
__device__ __forceinline__ void stage_sources(const int8_t* p, long long ld, long long r0, long long rows, int t,
                                              const int8_t* (&src)[ROWS * KB / 16 / NT]) {
    constexpr int C = KB / 16;
#pragma unroll
    for (int i = 0; i < ROWS * C / NT; ++i) {
        const int slot = i * NT + t;
        const int r = slot / C, c = (slot % C) ^ swap_of<KB>(r);
        src[i] = p + (r0 + r < rows ? r0 + r : rows - 1) * ld + c * 16;
    }
}
// Load i of a stage: 16 bytes per lane.
template <int NT>
__device__ __forceinline__ void stage_direct(const int8_t* src, int i, int8_t* lds, int t) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)(lds + (i * NT + (t & ~63)) * 16), 16, 0, 0);
}
// The same through registers: any alignment, and the end of the rows (what lies behind it counts as 0).
template <int ROWS, int KB, int NT>
__device__ __forceinline__ void stage_load(const int8_t* __restrict__ p, long long ld, long long r0, long long rows,
                                           int k0, int K, int t, i32x4 (&v)[ROWS * KB / 16 / NT]) {
    constexpr int C = KB / 16;
#pragma unroll
    for (int i = 0; i < ROWS * C / NT; ++i) {
        const int slot = i * NT + t;
        const int r = slot / C, c = (slot % C) ^ swap_of<KB>(r);
        const long long row = r0 + r < rows ? r0 + r : rows - 1;
        v[i] = load16(p + row * ld + k0 + c * 16, K - k0 - c * 16, K);
    }
}
template <int ROWS, int KB, int NT>
__device__ __forceinline__ void stage_store(const i32x4 (&v)[ROWS * KB / 16 / NT], int8_t* lds, int t) {
#pragma unroll
    for (int i = 0; i < ROWS * KB / 16 / NT; ++i) *(i32x4*)(lds + (i * NT + t) * 16) = v[i];
}

// The F fragments (32 rows x 32 bytes) of a wave for MFMA step s of a stage; rows points at the wave's first row + lane % 32.
template <int KB, int F>
__device__ __forceinline__ void fragments(const int8_t* rows, int s, int lane, i32x4 (&v)[F]) {
    const int o = ((2 * s + (lane >> 5)) ^ swap_of<KB>(lane & 31)) << 4;
#pragma unroll
    for (int i = 0; i < F; ++i) v[i] = *(const i32x4*)(rows + i * 32 * KB + o);
}
template <int FM, int FN>
__device__ __forceinline__ void multiply(const i32x4 (&av)[FM], const i32x4 (&bv)[FN], i32x16 (&acc)[FM][FN]) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[i], bv[j], acc[i][j], 0, 0, 0);
}

// A wave's part of the tile to memory: 32 rows at a time through `strip`, LDS of the wave's own.
template <int BM, int BN, int WM, int WN, typename Y>
__device__ __forceinline__ void store_strips(const I8Args& a, const i32x16 (&acc)[BM / WM / 32][BN / WN / 32], int8_t* strip,
                                             const float* SX, const float (&sw)[BN / WN / 32],
                                             const float (&add)[BN / WN / 32], long long m0, int n0, int lane) {
    constexpr int FM = BM / WM / 32, FN = BN / WN / 32, TN = BN / WN;
    constexpr int V = 16 / sizeof(Y), PER = TN / V, ROWS = 64 / PER;       // 16-byte pieces of a row, rows per store
    Y* s = (Y*)strip;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        __builtin_amdgcn_sched_barrier(0);       // one strip at a time: moved together, four strips' values spill
        asm volatile("" ::: "memory");
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int r = 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
            const float sx = SX[i * 32 + r];
#pragma unroll
            for (int j = 0; j < FN; ++j) s[r * TN + j * 32 + (lane & 31)] = from_f32<Y>(scaled(acc[i][j][e], sx, sw[j], add[j]));
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        const int c = (lane % PER) * V;
#pragma unroll
        for (int q = 0; q < 32 / ROWS; ++q) {
            const int r = q * ROWS + lane / PER;
            const long long m = m0 + i * 32 + r;
            if (m >= a.M || n0 + c >= a.N) continue;
            Y* out = (Y*)a.y + m * a.ldy + n0 + c;
            if (n0 + c + V <= a.N) {
                const i32x4 v = *(const i32x4*)(s + r * TN + c);
                __builtin_memcpy(out, &v, 16);
            } else {
                for (int k = 0; k < V && n0 + c + k < a.N; ++k) out[k] = s[r * TN + c + k];
            }
        }
    }
}

// Workgroup -> tile: workgroups go to the 8 XCDs in turn, so each XCD is given one contiguous range of tiles, walked in
// groups of 8 rows of tiles: what runs on it together shares operands through its L2.
__device__ __forceinline__ void tile_of(const I8Args& a, int& tm, int& tn) {
    const int n = a.tiles_m * a.tiles_n, b = blockIdx.x, per = n / 8, rest = n % 8, xcd = b % 8;
    const int id = xcd * per + (xcd < rest ? xcd : rest) + b / 8;
    const int g = id / (8 * a.tiles_n), first = g * 8, height = a.tiles_m - first < 8 ? a.tiles_m - first : 8;
    const int in = id - g * 8 * a.tiles_n;
    tm = first + in % height;
    tn = in / height;
}

// Waits until at most N of the wave's memory loads are in flight (they return in order) and its LDS reads have returned.
template <int N>
__device__ __forceinline__ void loads_left() {
    static_assert(N < 64, "vmcnt has 6 bits");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
}
// A barrier that does not wait for the loads in flight (__syncthreads does).  Nothing is moved across it.
__device__ __forceinline__ void bare_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <int BM, int BN, int WM, int WN, int KB, int NS, int KS, bool DIRECT, typename Y>
__global__ __launch_bounds__(WM* WN* KS * 64) void gemm_i8_tile_kernel(const I8Args a) {
    constexpr int NT = WM * WN * 64, FM = BM / WM / 32, FN = BN / WN / 32;
    constexpr int SA = BM * KB, SB = BN * KB;
    // (arrays of their own, so that the compiler sees that a stage being read is none being filled)
    constexpr int Z2 = NS > 2 ? KS : 0;
    __shared__ __attribute__((aligned(256))) int8_t A0[KS * SA], A1[KS * SA], A2[Z2 * SA + 16], A3[Z2 * SA + 16];
    __shared__ __attribute__((aligned(256))) int8_t B0[KS * SB], B1[KS * SB], B2[Z2 * SB + 16], B3[Z2 * SB + 16];
    __shared__ float SX[BM];
    const int group = KS > 1 ? threadIdx.x / NT : 0, t = threadIdx.x - group * NT;
    const int lane = t & 63, wave = t >> 6, wm = wave / WN, wn = wave % WN;
    int tm, tn;
    tile_of(a, tm, tn);
    const long long m0 = (long long)tm * BM;
    const int n0 = tn * BN;
    int8_t* const As[4] = {A0 + group * SA, A1 + group * SA, A2 + group * SA, A3 + group * SA};
    int8_t* const Bs[4] = {B0 + group * SB, B1 + group * SB, B2 + group * SB, B3 + group * SB};
    i32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    // scales and bias are asked for ahead of the k loop (behind it a wave would wait for each)
    if (threadIdx.x < BM) SX[threadIdx.x] = a.sx[m0 + threadIdx.x < a.M ? m0 + threadIdx.x : a.M - 1];
    float sw[FN], add[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + wn * (BN / WN) + j * 32 + (lane & 31);
        sw[j] = a.sw[n < a.N ? n : a.N - 1];
        add[j] = bias_at(a, n < a.N ? n : a.N - 1);
    }

    // Rounds in which every group has a whole step; what is left of the rows is one last round through registers.
    const int rounds = a.K / (KB * KS), k_rest = (rounds * KS + group) * KB;
    const bool rest = rounds * KS * KB < a.K;
    constexpr int LA = SA / 16 / NT, LB = SB / 16 / NT, L = LA + LB;         // 16-byte loads of a thread per stage
    constexpr int S = KB / 32;                                               // MFMA steps of a round
    i32x4 va[LA], vb[LB];
    constexpr bool EARLY = KS > 1;           // (few registers: its loads are in flight from the start)
    if (EARLY && DIRECT && rest) {
        stage_load<BM, KB, NT>(a.x, a.ldx, m0, a.M, k_rest, a.K, t, va);
        stage_load<BN, KB, NT>(a.w, a.ldw, n0, a.N, k_rest, a.K, t, vb);
    }
    const int8_t *ar[NS], *br[NS];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
        ar[u] = As[u] + (wm * (BM / WM) + (lane & 31)) * KB;
        br[u] = Bs[u] + (wn * (BN / WN) + (lane & 31)) * KB;
    }
    i32x4 av[2][FM], bv[2][FN];
    if constexpr (DIRECT) {
        // A ring of NS stages.  The barrier of a round stands in front of its last MFMA step: behind it the stage is free
        // (its fragments are in registers) and the next one has arrived, so the first fragments of the next round and the
        // loads NS rounds ahead are asked for while that step still multiplies.
        if (rounds > 0) {
            const int8_t *pa[LA], *pb[LB];
            stage_sources<BM, KB, NT>(a.x, a.ldx, m0, a.M, t, pa);
            stage_sources<BN, KB, NT>(a.w, a.ldw, n0, a.N, t, pb);
            // loads [first, last) of the L that fill a stage for a round
            auto fill = [&](int round, int8_t* Ad, int8_t* Bd, int first, int last) {
                const int k0 = (round * KS + group) * KB;
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (i >= first && i < last) {
                        if (i < LA) stage_direct<NT>(pa[i < LA ? i : 0] + k0, i, Ad, t);
                        else stage_direct<NT>(pb[i < LA ? 0 : i - LA] + k0, i - LA, Bd, t);
                    }
            };
            // waits until a stage has arrived behind which `behind` more are on their way
            auto arrived = [&](int behind) {
                if (NS > 3 && behind >= 3) loads_left<(NS > 3 ? 3 : 0) * L>();
                else if (NS > 2 && behind == 2) loads_left<(NS > 2 ? 2 : 0) * L>();
                else if (behind == 1) loads_left<L>();
                else loads_left<0>();
            };
            // One round: S MFMA steps, row by row of the wave's fragments.  STEADY: NS more rounds follow (straight code,
            // whose waits are constants).  sched_barrier: the order is meant; left to itself the compiler puts the
            // reads of the next fragments behind the products they should run beside (0.75 instead of 0.55 us a round).
            auto turn = [&](auto steady, int r, int u) {
                constexpr bool STEADY = decltype(steady)::value;
                const int next = (u + 1) % NS;
#pragma unroll
                for (int q = 0; q < S; ++q) {
                    if (q == S - 1 && (STEADY || r + 1 < rounds)) {
                        if (STEADY) loads_left<(NS - 2) * L>();
                        else arrived(rounds - 2 - r < NS - 2 ? rounds - 2 - r : NS - 2);
                        bare_barrier();
                        fragments<KB>(ar[next], 0, lane, av[S & 1]);
                        fragments<KB>(br[next], 0, lane, bv[S & 1]);
                    }
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int j = 0; j < FN; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[q & 1][i], bv[q & 1][j], acc[i][j], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        if (q < S - 1) {
                            if (i == 0) {
                                fragments<KB>(ar[u], q + 1, lane, av[(q + 1) & 1]);
                                fragments<KB>(br[u], q + 1, lane, bv[(q + 1) & 1]);
                            }
                        } else if (STEADY || r + NS < rounds) {
                            fill(r + NS, As[u], Bs[u], i * L / FM, (i + 1) * L / FM);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            static_assert(S % 2 == 0, "the fragments of step 0 are in the first of the two sets");
#pragma unroll
            for (int u = 0; u < NS; ++u)
                if (u < rounds) fill(u, As[u], Bs[u], 0, L);
            arrived(rounds - 1 < NS - 1 ? rounds - 1 : NS - 1);
            bare_barrier();
            fragments<KB>(ar[0], 0, lane, av[0]);
            fragments<KB>(br[0], 0, lane, bv[0]);
            int r = 0;
            for (; r + 2 * NS <= rounds; r += NS) {
#pragma unroll
                for (int u = 0; u < NS; ++u) turn(std::true_type{}, r + u, u);
            }
#pragma unroll
            for (int u = 0; u < 2 * NS - 1; ++u)
                if (r + u < rounds) turn(std::false_type{}, r + u, u % NS);
        }
    } else {
        // Through registers: the next step's loads are in flight while the present one is multiplied; two stages.
        auto load = [&](int round) {
            const int k0 = (round * KS + group) * KB;
            stage_load<BM, KB, NT>(a.x, a.ldx, m0, a.M, k0, a.K, t, va);
            stage_load<BN, KB, NT>(a.w, a.ldw, n0, a.N, k0, a.K, t, vb);
        };
        if (rounds > 0) load(0);
        for (int r0 = 0; r0 < rounds; r0 += 2) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = r0 + u;
                if (r < rounds) {
                    stage_store<BM, KB, NT>(va, As[u], t);
                    stage_store<BN, KB, NT>(vb, Bs[u], t);
                    __syncthreads();
                    if (r + 1 < rounds) load(r + 1);
#pragma unroll
                    for (int q = 0; q < S; ++q) {
                        fragments<KB>(ar[u], q, lane, av[0]);
                        fragments<KB>(br[u], q, lane, bv[0]);
                        multiply(av[0], bv[0], acc);
                    }
                }
            }
        }
    }
    __syncthreads();                                         // no load to LDS is in flight, no stage is being read
    if (rest) {
        if (!(EARLY && DIRECT)) {
            stage_load<BM, KB, NT>(a.x, a.ldx, m0, a.M, k_rest, a.K, t, va);
            stage_load<BN, KB, NT>(a.w, a.ldw, n0, a.N, k_rest, a.K, t, vb);
        }
        stage_store<BM, KB, NT>(va, As[0], t);
        stage_store<BN, KB, NT>(vb, Bs[0], t);
        __syncthreads();
#pragma unroll
        for (int q = 0; q < S; ++q) {
            fragments<KB>(ar[0], q, lane, av[0]);
            fragments<KB>(br[0], q, lane, bv[0]);
            multiply(av[0], bv[0], acc);
        }
        __syncthreads();
    }
    if constexpr (KS > 1) {
        // The groups' sums meet in LDS (the stages are free behind the barrier), two tiles per array; each group finishes
        // its share of them.
        static_assert(FM == 1 && FN == 1 && KS == 4 && KS * SA >= 2 * BM * BN * 4, "a group finishes four results of a lane");
        int* const sums[4] = {(int*)A0, (int*)A0 + BM * BN, (int*)A1, (int*)A1 + BM * BN};
#pragma unroll
        for (int g = 0; g < KS; ++g)
            if (g == group)
#pragma unroll
                for (int e = 0; e < 16; ++e) sums[g][e * NT + t] = acc[0][0][e];
        __syncthreads();
        const int n = n0 + wn * (BN / WN) + (lane & 31);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int e = group * 4 + q, r = wm * (BM / WM) + 8 * group + 4 * (lane >> 5) + q;
            int v = 0;
#pragma unroll
            for (int g = 0; g < KS; ++g) v += sums[g][e * NT + t];
            if (n < a.N && m0 + r < a.M) ((Y*)a.y)[(m0 + r) * a.ldy + n] = from_f32<Y>(scaled(v, SX[r], sw[0], add[0]));
        }
    } else {
        // Strips of 32 rows through a part of LDS that is the wave's own, so that rows leave in 16-byte pieces.
        constexpr int STRIP = 32 * (BN / WN) * sizeof(Y), FIT = SA / STRIP;
        static_assert(FIT >= 1 && 4 * FIT >= WM * WN, "a strip per wave has to fit the stages of one operand");
        int8_t* const strips[4] = {A0, A1, A2, A3};
        int8_t* strip = strips[0];
#pragma unroll
        for (int q = 1; q < 4; ++q) strip = wave / FIT == q ? strips[q] : strip;
        store_strips<BM, BN, WM, WN, Y>(a, acc, strip + wave % FIT * STRIP, SX + wm * (BM / WM), sw, add,
                                        m0 + wm * (BM / WM), n0 + wn * (BN / WN), lane);
    }
}

constexpr long long MAX_BLOCKS = 1 << 20;        // a launch holds fewer than 2^32 threads; rows beyond it are looped over

template <typename T, int TPR, int V>
void launch_quant(const void* x, long long ldx, long long rows, int k, int8_t* q, long long ldq, float* scale,
                  AlignRows al, hipStream_t st) {
    constexpr int NT = TPR > 256 ? TPR : 256, PER = NT / TPR;
    const long long blocks = (rows + PER - 1) / PER;
    al.first = (unsigned)(blocks < MAX_BLOCKS ? blocks : MAX_BLOCKS);
    const dim3 grid(al.first + (al.n < 2048 ? al.n : 2048)), block(NT);
    const int mode = row_mode(k, vec_of<T>());
#define QUANT_ROWS_OF(x) (const T*)x, ldx, rows, k, q, ldq, scale
#define QUANT_MODE(MODE) \
    hipLaunchKernelGGL((quant_rows_kernel<T, TPR, V, MODE>), grid, block, 0, st, QUANT_ROWS_OF(x))
#define QUANT_ALIGN(MODE) \
    hipLaunchKernelGGL((quant_rows_kernel<T, TPR, V, MODE, AlignRows>), grid, block, 0, st, QUANT_ROWS_OF(x), al)
    if (TPR >= 64 && al.n) {
        if constexpr (TPR >= 64) {
            if (mode == ROW_FULL) QUANT_ALIGN(ROW_FULL);
            else QUANT_ALIGN(ROW_RAGGED);
        }
    } else if (mode == ROW_FULL) QUANT_MODE(ROW_FULL);
    else if (mode == ROW_RAGGED) QUANT_MODE(ROW_RAGGED);
    else if constexpr (TPR == 16) QUANT_MODE(ROW_TINY);
#undef QUANT_ROWS_OF
#undef QUANT_ALIGN
#undef QUANT_MODE
}

template <typename T>
void quant_rows(const void* x, long long ldx, long long rows, int k, int8_t* q, long long ldq, float* scale,
                const AlignRows& al, hipStream_t st) {
    const int vecs = (k + vec_of<T>() - 1) / vec_of<T>();
#define QUANT(TPR, V) return launch_quant<T, TPR, V>(x, ldx, rows, k, q, ldq, scale, al, st)
    // Few rows: a thread takes one or two vectors, so that the row is there after one trip to memory; many: a wave holds a row by
    // itself and meets no barrier.  us of many / few threads a row, launches on the same rows (fp32; bf16 rows of twice the values
    // alike):
    //            64 rows     1000       2000       4000       8000       16000
    //   n 1000   2.5 / 2.7   3.1 / 2.8  4.1 / 3.0  6.2 / 3.8  10.0 / 6.7  17.5 / 12.9
    //   n 2000   2.6 / 3.0   3.2 / 3.4  4.3 / 3.9  7.0 / 6.8  13.5 / 13.2 23.7 / 24.5
    //   n 4000   3.0 / 2.9   6.3 / 4.0  11.0 / 6.7 20.5 / 13.1 37.8 / 24.1 83.2 / 50.5
    // (The two meet at some 700, 1500 and 100 rows there; bf16 rows of 4000 values near 4000 rows.  The bounds lie above that.)
    if (vecs <= 16) QUANT(16, 1);
    if (vecs <= 64) QUANT(64, 1);
    if (vecs <= 128) QUANT(64, 2);
    if (vecs <= 256 && rows < 4096) QUANT(256, 1);
    if (vecs <= 256) QUANT(64, 4);
    if (vecs <= 512 && rows < 4096) QUANT(256, 2);
    if (vecs <= 512) QUANT(64, 8);
    if (vecs <= 1024 && rows < 1024) QUANT(1024, 1);
    if (vecs <= 1024) QUANT(256, 4);
    if (vecs <= 2048) QUANT(1024, 2);
    if (vecs <= 4096) QUANT(1024, 4);
    if (vecs <= 5120) QUANT(1024, 5);
    if (vecs <= 8192) QUANT(1024, 8);
#undef QUANT
    hipLaunchKernelGGL((quant_rows_long_kernel<T>), dim3((unsigned)(rows < MAX_BLOCKS ? rows : MAX_BLOCKS)), dim3(1024), 0,
                       st, (const T*)x, ldx, rows, k, q, ldq, scale);
}

template <int BM, int BN, int WM, int WN, int KB, int NS, int KS, bool DIRECT>
void launch_tile(I8Args a, hipStream_t st) {
    a.tiles_m = (int)((a.M + BM - 1) / BM);
    a.tiles_n = (a.N + BN - 1) / BN;
    const dim3 grid((unsigned)((long long)a.tiles_m * a.tiles_n)), block(WM * WN * KS * 64);
    if (a.ytype == SCA_F32)
        hipLaunchKernelGGL((gemm_i8_tile_kernel<BM, BN, WM, WN, KB, NS, KS, DIRECT, float>), grid, block, 0, st, a);
    else if (a.ytype == SCA_BF16)
        hipLaunchKernelGGL((gemm_i8_tile_kernel<BM, BN, WM, WN, KB, NS, KS, DIRECT, sca_bf16>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((gemm_i8_tile_kernel<BM, BN, WM, WN, KB, NS, KS, DIRECT, sca_f16>), grid, block, 0, st, a);
}

template <typename T>
void launch_direct(I8Args a, hipStream_t st) {
    a.tiles_m = (int)((a.M + 15) / 16);
    a.tiles_n = (a.N + 15) / 16;
    hipLaunchKernelGGL((gemm_i8_direct_kernel<T>), dim3((unsigned)((long long)a.tiles_m * a.tiles_n)), dim3(512), 0, st, a);
}

// Which kernel: us of direct with x in whole cache lines, as int8_matmul gets it from quantize_int8 (with x as sca_linear_i8 lays
// it out, pitch_of) / 64 x 64 by four groups / 128 x 128 / 256 x 256 tiles, results in bf16 (M x N x K):
//   1 x 4096 x 4000      4.9 (4.9) / 9.0 / 17 / 42          512 x 512 x 2048       9.9 (7.4) / 6.4 / 10.6 / 25
//   16 x 8192 x 4000    10.1 (8.0) / 10.9 / 18 / 43         300 x 300 x 4096       9.6 (7.2) / 8.7 / 18 / 46
//   128 x 128 x 2000     4.4 (3.9) / 6.7 / 11.4 / 26        8192 x 128 x 2000     36 (27) / 7.6 / 11.8 / 27
//   256 x 256 x 8000     9.8 (7.8) / 14.1 / 27 / 75         1024 x 1024 x 4096    58 (40) / 10.4 / 20 / 43
//   320 x 400 x 2000     6.4 (5.3) / 6.9 / 11.5 / 26        64 x 20000 x 128      15.4 (15.3) / 8.6 / 5.3 / 7.5
//   400 x 450 x 1500     7.2 (6.0) / 7.1 / 11.3 / 24        2048 x 2048 x 2048   116 (76) / 24 / 13.7 / 28
//   1000 x 250 x 300     6.0 (5.9) / 5.4 / 8.0 / 14         16384 x 256 x 4000   225 (160) / 44 / 25 / 46
//   4096 x 4096 x 4096   - / 153 / 83 / 67                  65536 x 64 x 512      39 (36) / 17 / 11.1 / 16.1
// Direct: one workgroup per CU at most, or a few with short rows (or single cells, whose x is read from the caches).  640 tiles
// and tiles * K = 1.2 million: over 264 sizes drawn with 257 to 1400 tiles and tiles * K from 0.15 to 6 million, x in whole lines,
// that takes 1.2 % longer than the better of the two kernels, and no other bound of tiles * K is better (1 million: 1.3 %, 1.5
// million: 1.4 %; direct / tile at up to 640 tiles: 0.75 up to 0.4 million, 0.88 to 1, 0.97 to 1.2, 1.06 to 2, 1.17 to 3).  x as
// sca_linear_i8 lays it out suits the direct kernel further up (0.70, 0.74, 0.78, 0.83, 0.92): the same bound takes 6 % longer there.
// 64: no more tiles than CUs.  Larger tiles read less; they need about one tile per CU, little of it lost behind the edges, and
// no last run over the chip with few of them (21986 x 543 x 608, 258 tiles of 256: 37 us, 24.5 in tiles of 128).  Over 60 sizes
// drawn between 2e9 and 1.3e11 products the rule takes 1 % longer than the best of the three.
constexpr int CUS = 256;
bool takes_direct(long long M, int N, int K) {
    const long long tiles = ((M + 15) / 16) * ((N + 15LL) / 16);
    if (tiles >= 1 << 23) return false;                                         // (fewer than 2^32 threads)
    return M <= 16 || tiles <= CUS || (tiles <= 5 * CUS / 2 && tiles * K <= 1200000);
}
void gemm_i8_rows(const I8Args& a, hipStream_t st) {
    const bool aligned = !(((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.ldx | (uintptr_t)a.ldw) & 15);
    auto tiles = [&](int b) { return ((a.M + b - 1) / b) * ((a.N + b - 1) / b); };
    auto runs = [&](int b, int per_cu) { return (tiles(b) + per_cu * CUS - 1) / (per_cu * CUS); };
    if (takes_direct(a.M, a.N, a.K)) {
        launch_direct<int8_t>(a, st);
    } else if (aligned && tiles(256) >= 192 && 16 * tiles(256) <= 5 * tiles(128) && 11 * runs(256, 1) * CUS <= 15 * tiles(256)) {
        launch_tile<256, 256, 2, 4, 64, 4, 1, true>(a, st);
    } else if (aligned) {
        if (tiles(64) > CUS) launch_tile<128, 128, 2, 2, 64, 4, 1, true>(a, st);
        else launch_tile<64, 64, 2, 2, 128, 2, 4, true>(a, st);
    } else {
        // (what a run of tiles over the chip takes, two of the larger ones per CU, fitted to 60 sizes: within 1 % of the better)
        if (runs(128, 2) * (4 + 0.0104 * a.K) < runs(64, 1) * (3.25 + 0.0028 * a.K))
            launch_tile<128, 128, 2, 2, 64, 4, 1, false>(a, st);
        else launch_tile<64, 64, 2, 2, 128, 2, 4, false>(a, st);
    }
}
// Fewer than 2^32 threads a launch: rows beyond 2^23 tiles of 128 x 128 (256 threads; of the other tiles the rule above takes
// fewer) in slices.
void gemm_i8(const I8Args& a, hipStream_t st) {
    const long long wide = (a.N + 127LL) / 128, most = (wide < 1 << 23 ? (1 << 23) / wide : 1) * 128;
    const int size = a.ytype == SCA_F32 ? 4 : 2;
    I8Args s = a;
    for (long long m = 0; m < a.M; m += most) {
        s.x = a.x + m * a.ldx;
        s.sx = a.sx + m;
        s.y = (char*)a.y + m * a.ldy * size;
        s.M = a.M - m < most ? a.M - m : most;
        gemm_i8_rows(s, st);
    }
}

constexpr int MAX_N = 0x7ffff000;               // (columns are counted in 32 bits, a step of all threads ahead)
constexpr int I8_MAX_K = (1 << 17) - 1;         // 2^17 products of -128 * -128 would pass int32

void quantize(const void* x, long long ldx, int dtype, long long rows, int k, int8_t* q, long long ldq, float* scale,
              hipStream_t st, const AlignRows& al = AlignRows{}) {
    if (dtype == SCA_F32) quant_rows<float>(x, ldx, rows, k, q, ldq, scale, al, st);
    else if (dtype == SCA_BF16) quant_rows<sca_bf16>(x, ldx, rows, k, q, ldq, scale, al, st);
    else quant_rows<sca_f16>(x, ldx, rows, k, q, ldq, scale, al, st);
}
// (N: the direct kernel takes 32 threads an output, and a launch fewer than 2^32)
bool one_launch(long long M, int N, int K) { return M <= QUANT_ROWS && K <= QUANT_K - 128 && (N + 15LL) / 16 < 1 << 23; }
// Pitch of the rows that sca_linear_i8 quantizes for itself.  Tiles want whole cache lines (128 x 128 tiles, 16384 x 256 x
// 4000: 25.0 us, 28.8 with 16 bytes more); the direct kernel, whose 16 lanes read 16 rows, wants them to start in different
// banks (16 x 4096 x 4000: 6.6 us on whole lines, 5.5 with an odd number of 16-byte pieces; 320 x 400 x 2000: 6.4, 5.2).
long long pitch_of(int K, bool direct) {
    return direct ? (((long long)K + 15) / 16 | 1) * 16 : ((long long)K + 127) & ~127LL;
}
// A weight whose rows are not 16-byte aligned is copied to rows that are, in the launch that quantizes x, where that is
// little work beside the product (us of the product with rows as they are / aligned: 1071 x 1338 x 2217 23 / 14, 20030 x 1294 x
// 1636 90 / 67, 665 x 1621 x 6263 43 / 28; but 22267 x 1920 x 68 27.5 / 29.2, and 213 x 2051 x 7874 24 / 19 with 6 for the copy).
bool worth_aligning(long long M, int N, int K) { return M >= 512 && K >= 512 && K <= 32768 && !takes_direct(M, N, K); }

}  // namespace

extern "C" int sca_gemm_i8_max_k(void) { return I8_MAX_K; }

extern "C" int sca_quant_rows_i8(const void* x, long long ldx, int dtype, long long rows, int k, int8_t* q,
                                 long long ldq, float* scale, void* stream) {
    if (dtype < SCA_F32 || dtype > SCA_F16 || rows < 0 || k <= 0 || k > MAX_N || ldx < 0 || ldq < k) return -1;
    if (rows == 0) return 0;
    if (!x || !q || !scale) return -1;
    quantize(x, ldx, dtype, rows, k, q, ldq, scale, (hipStream_t)stream);
    SCA_CHECK_LAUNCH();
    return 0;
}

extern "C" int sca_csr_quant_rows_i8(const int64_t* indptr, const int32_t* indices, const float* data,
                                     const int64_t* row_ids, int B, int G, int apply_log1p, int8_t* q, int ldq,
                                     float* scale, void* stream) {
    if (B < 0 || G <= 0 || ldq < G || (ldq & 15) || ((uintptr_t)q & 15)) return -1;
    if (ldq > CSR_LDS) return -2;
    if (B == 0) return 0;
    if (!indptr || !indices || !data || !q || !scale) return -1;
    constexpr int MOST = 1 << 25;                // (fewer than 2^32 threads a launch)
    for (long long b = 0; b < B; b += MOST)
        hipLaunchKernelGGL(csr_quant_rows_kernel, dim3((unsigned)(B - b < MOST ? B - b : MOST)), dim3(64), ldq,
                           (hipStream_t)stream, row_ids ? indptr : indptr + b, indices, data, row_ids ? row_ids + b : nullptr,
                           apply_log1p, q + b * ldq, ldq, scale + b);
    SCA_CHECK_LAUNCH();
    return 0;
}

extern "C" int sca_gemm_i8(const int8_t* xq, long long ldx, const float* sx, const int8_t* wq, long long ldw,
                           const float* sw, const void* bias, int btype, long long M, int N, int K, void* y, int ytype,
                           long long ldy, void* stream) {
    if (ytype < SCA_F32 || ytype > SCA_F16 || (btype != SCA_F32 && btype != ytype)) return -1;
    if (M < 0 || N < 0 || N > MAX_N || K <= 0 || K > I8_MAX_K || ldx < 0 || ldw < K || ldy < N) return -1;
    if (M == 0 || N == 0) return 0;
    if (!xq || !sx || !wq || !sw || !y) return -1;
    gemm_i8(I8Args{xq, ldx, sx, wq, ldw, sw, bias, btype, y, ytype, ldy, M, N, K, 0, 0}, (hipStream_t)stream);
    SCA_CHECK_LAUNCH();
    return 0;
}

extern "C" long long sca_linear_i8_workspace_bytes(long long M, int N, int K) {
    if (M < 0 || N < 0 || N > MAX_N || K <= 0 || K > I8_MAX_K) return -1;
    if (one_launch(M, N, K)) return 0;
    return M * (pitch_of(K, takes_direct(M, N, K)) + 4) + (worth_aligning(M, N, K) ? N * pitch_of(K, false) : 0);
}

extern "C" int sca_linear_i8(const void* x, long long ldx, int dtype, const int8_t* wq, long long ldw, const float* sw,
                             const void* bias, int btype, long long M, int N, int K, void* y, int ytype, long long ldy,
                             void* ws, void* stream) {
    if (dtype < SCA_F32 || dtype > SCA_F16 || ytype < SCA_F32 || ytype > SCA_F16) return -1;
    if (btype != SCA_F32 && btype != ytype) return -1;
    if (M < 0 || N < 0 || N > MAX_N || K <= 0 || K > I8_MAX_K || ldx < 0 || ldw < K || ldy < N) return -1;
    if (M == 0 || N == 0) return 0;
    if (!x || !wq || !sw || !y) return -1;
    hipStream_t st = (hipStream_t)stream;
    I8Args a{(const int8_t*)x, ldx, nullptr, wq, ldw, sw, bias, btype, y, ytype, ldy, M, N, K, 0, 0};
    if (one_launch(M, N, K)) {
        if (dtype == SCA_F32) launch_direct<float>(a, st);
        else if (dtype == SCA_BF16) launch_direct<sca_bf16>(a, st);
        else launch_direct<sca_f16>(a, st);
    } else {
        if (!ws || ((uintptr_t)ws & 15)) return -1;
        const long long pitch = pitch_of(K, takes_direct(M, N, K));
        int8_t* q = (int8_t*)ws;
        float* scale = (float*)(q + M * pitch);
        AlignRows al = {};
        if (worth_aligning(M, N, K)) {
            scale = (float*)(q + M * pitch + N * pitch_of(K, false));
            if (((uintptr_t)wq | (uintptr_t)ldw) & 15) {
                al = AlignRows{wq, ldw, N, K, q + M * pitch, pitch_of(K, false), 0};
                a.w = al.to; a.ldw = al.pitch;
            }
        }
        quantize(x, ldx, dtype, M, K, q, pitch, scale, st, al);
        a.x = q; a.ldx = pitch; a.sx = scale;
        gemm_i8(a, st);
    }
    SCA_CHECK_LAUNCH();
    return 0;
}
