// Layer norm over the last dimension with weight and bias, forward and backward (gfx950).
//
//   h = (x - mean(x)) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = h * w + b
//   a = dy * w:  dx = rstd * (a - mean(a) - h * mean(a * h));  dw = sum over rows of dy * h;  db = sum over rows of dy
//
// fp32 / bf16 / fp16 rows of any width and pitch; statistics, sums and gradients are held in fp32 and rounded once when
// they are stored.  (sca_layer_fwd / sca_layer_bwd normalise without weight and bias inside the conditional layers.)
//
// All passes are bound by memory, so a row is read once: TPR threads (16 ... 1024, as wide as the row needs) hold it in
// registers, the mean and then the squared distances from it are summed from there.  The backward pass keeps the column
// sums of dw and db in registers over all rows that a thread walks and leaves one slab of partial sums per workgroup, so
// that they cost no second pass over x and dy; a second launch adds the slabs in a fixed order (no atomics).
#include "common.h"
#include "dtypes.h"
#include "rowtile.h"

namespace {

constexpr int MAX_N = 0x7ffff000;                // (columns are counted in 32 bits, a step of all threads ahead)
constexpr long long MAX_BLOCKS = 1 << 20;        // a launch holds fewer than 2^32 threads; rows beyond it are looped over

// Weight elements [c, c + VEC) of n (type W, so up to 32 bytes), `other` where there is no weight.
template <int MODE, typename W, int VEC>
__device__ __forceinline__ void load_weight(const W* __restrict__ w, int c, int n, float other, float (&v)[VEC]) {
    if (w) {
        if (MODE == ROW_TINY) load_part<W, VEC>(w, n, v);
        else load_vec<W, VEC>(w + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = other;
    }
}

template <typename T, typename W, int TPR, int V, int MODE>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_fwd_kernel(const T* __restrict__ x, long long ldx,
                                                                       long long rows, int n, const W* __restrict__ w,
                                                                       const W* __restrict__ b, float eps,
                                                                       T* __restrict__ y, long long ldy, bool stream,
                                                                       float* __restrict__ stats) {
    constexpr int VEC = vec_of<T>(), NT = TPR > 256 ? TPR : 256;
    __shared__ float scratch[16];
    const int t = threadIdx.x % TPR;
    for (long long r = (long long)blockIdx.x * (NT / TPR) + threadIdx.x / TPR; r < rows;
         r += (long long)gridDim.x * (NT / TPR)) {
        const T* xr = x + r * ldx;
        raw_t raw[V] = {};
        float v[VEC];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Cols<T, TPR, MODE> at(j, t, n);
            if (at.there) load_cols<MODE>(xr, at.c, n, raw[j]);
        }
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Cols<T, TPR, MODE> at(j, t, n);
            unpack<T>(raw[j], v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += at.own(i, n) ? v[i] : 0.f;        // (a vector that is not there is 0)
        }
        const float mean = row_sum<TPR>(s, scratch) / (float)n;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Cols<T, TPR, MODE> at(j, t, n);
            unpack_again<T>(raw[j], v);
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = at.own(i, n) ? v[i] - mean : 0.f;
                p = fmaf(d, d, p);
            }
            q += at.there ? p : 0.f;
        }
        const float rstd = 1.0f / sqrtf(row_sum<TPR>(q, scratch) / (float)n + eps);
        T* yr = y + r * ldy;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Cols<T, TPR, MODE> at(j, t, n);
            if (!at.there) continue;
            float g[VEC], o[VEC];
            load_weight<MODE>(w, at.c, n, 1.f, g);
            load_weight<MODE>(b, at.c, n, 0.f, o);
            unpack_again<T>(raw[j], v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = fmaf((v[i] - mean) * rstd, g[i], o[i]);
            store_cols<MODE>(yr, at.c, n, v, stream);
        }
        if (t == 0 && stats) {
            stats[r] = mean;
            stats[rows + r] = rstd;
        }
    }
}

// Rows beyond what a workgroup's registers hold: one workgroup per row, three passes (the later ones from a cache).
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* __restrict__ x, long long ldx, long long rows, int n,
                                                           const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                           T* __restrict__ y, long long ldy, bool stream,
                                                           float* __restrict__ stats) {
    constexpr int VEC = vec_of<T>();
    __shared__ float scratch[16];
    const int vecs = (n + VEC - 1) / VEC;
    float v[VEC];
    auto col = [&](int j) { return j * VEC < n - VEC ? j * VEC : n - VEC; };
    for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        float s = 0.f, q = 0.f;
        for (int j = threadIdx.x; j < vecs; j += 1024) {
            const int skip = j * VEC - col(j);
            load_vec<T, VEC>(xr + col(j), v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += i >= skip ? v[i] : 0.f;
        }
        const float mean = row_sum<1024>(s, scratch) / (float)n;
        for (int j = threadIdx.x; j < vecs; j += 1024) {
            const int skip = j * VEC - col(j);
            load_vec<T, VEC>(xr + col(j), v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = i >= skip ? v[i] - mean : 0.f;
                q = fmaf(d, d, q);
            }
        }
        const float rstd = 1.0f / sqrtf(row_sum<1024>(q, scratch) / (float)n + eps);
        for (int j = threadIdx.x; j < vecs; j += 1024) {
            float g[VEC], o[VEC];
            load_weight<ROW_RAGGED>(w, col(j), n, 1.f, g);
            load_weight<ROW_RAGGED>(b, col(j), n, 0.f, o);
            load_vec<T, VEC>(xr + col(j), v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = fmaf((v[i] - mean) * rstd, g[i], o[i]);
            store_cols<ROW_RAGGED>(y + r * ldy, col(j), n, v, stream);
        }
        if (threadIdx.x == 0 && stats) {
            stats[r] = mean;
            stats[rows + r] = rstd;
        }
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------------
struct LnBwd {
    const void* dy; long long lddy;
    const void* x; long long ldx;
    long long rows; int n;
    const void* w;
    const float* stats;
    void* dx; long long lddx; bool stream;
    float* part;                 // [slab][2][n] partial sums of (dw, db), or null
    float* means;                // rows beyond the registers: [2][rows]
};

// NT threads, TPR of them a row.  HOLD: the weight stays in registers; the longest rows read it again (from a cache).
template <typename T, typename W, int TPR, int V, int MODE, int NT, bool HOLD = true>
__global__ __launch_bounds__(NT) void ln_bwd_kernel(const LnBwd a) {
    constexpr int VEC = vec_of<T>(), PER = NT / TPR, COLS = TPR * V * VEC;
    __shared__ float scratch[16];
    __shared__ __attribute__((aligned(16))) float sums[PER > 1 ? PER * COLS : 4];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, n = a.n;
    const float inv_n = 1.f / (float)n;
    float held[HOLD ? V : 1][VEC], dw[V][VEC], db[V][VEC];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const Cols<T, TPR, MODE> at(j, t, n);
        if (HOLD && at.there) load_weight<MODE>((const W*)a.w, at.c, n, 1.f, held[HOLD ? j : 0]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) dw[j][i] = db[j][i] = 0.f;
    }
    auto weight = [&](int j, int c, float (&g)[VEC]) {
        if (!HOLD) load_weight<MODE>((const W*)a.w, c, n, 1.f, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (HOLD) g[i] = held[HOLD ? j : 0][i];
    };
    const long long step = (long long)gridDim.x * PER;
    raw_t xq[V] = {}, dq[V] = {};
    float mean = 0.f, rstd = 0.f;
    auto load = [&](long long r) {
        const T *xr = (const T*)a.x + r * a.ldx, *dr = (const T*)a.dy + r * a.lddy;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Cols<T, TPR, MODE> at(j, t, n);
            if (at.there) {
                load_cols<MODE>(xr, at.c, n, xq[j]);
                load_cols<MODE>(dr, at.c, n, dq[j]);
            }
        }
        mean = a.stats[r];
        rstd = a.stats[a.rows + r];
    };
    // 16-bit rows, whose arithmetic takes half as long as their loads: the next row is on its way meanwhile (16384 x 4000
    // bf16: 81 instead of 100 us, with results through the caches).  fp32 rows have no registers for it and run at the rate
    // of a copy without.
    constexpr bool AHEAD = sizeof(T) == 2 && HOLD;
    // (where rows meet at barriers, a wave without a row of its own goes along with zeros)
    constexpr bool TOGETHER = PER > 1 && TPR > 64;
    long long r = (long long)blockIdx.x * PER + sub;
    if (AHEAD && r < a.rows) load(r);
    for (; (TOGETHER ? r - sub : r) < a.rows; r += step) {
        const bool mine = !TOGETHER || r < a.rows;
        if (!AHEAD && mine) load(r);
        raw_t x0[V], d0[V];
        const float mean0 = mine ? mean : 0.f, rstd0 = mine ? rstd : 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            x0[j] = mine ? xq[j] : raw_t{0, 0, 0, 0};
            d0[j] = mine ? dq[j] : raw_t{0, 0, 0, 0};
        }
        if (AHEAD && r + step < a.rows) load(r + step);
        float s1 = 0.f, s2 = 0.f, h[VEC], d[VEC], g[VEC];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Cols<T, TPR, MODE> at(j, t, n);
            if (!at.there) continue;
            weight(j, at.c, g);
            unpack<T>(x0[j], h);
            unpack<T>(d0[j], d);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                h[i] = (h[i] - mean0) * rstd0;
                dw[j][i] = fmaf(d[i], h[i], dw[j][i]);
                db[j][i] += d[i];
                const float p = at.own(i, n) ? d[i] * g[i] : 0.f;
                s1 += p;
                s2 = fmaf(p, h[i], s2);
            }
        }
        if (!a.dx) continue;
        const float m1 = row_sum<TPR>(s1, scratch) * inv_n, m2 = row_sum<TPR>(s2, scratch) * inv_n;
        T* out = (T*)a.dx + r * a.lddx;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Cols<T, TPR, MODE> at(j, t, n);
            if (!at.there || !mine) continue;
            weight(j, at.c, g);
            unpack_again<T>(x0[j], h);
            unpack_again<T>(d0[j], d);
#pragma unroll
            for (int i = 0; i < VEC; ++i) d[i] = rstd0 * (fmaf(d[i], g[i], -m1) - (h[i] - mean0) * rstd0 * m2);
            store_cols<MODE>(out, at.c, n, d, a.stream);
        }
    }
    if (!a.part) return;
    float* slab = a.part + (long long)blockIdx.x * 2 * n;
    auto put = [&](const float (&v)[V][VEC], float* out) {
        if constexpr (PER == 1) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const Cols<T, TPR, MODE> at(j, t, n);
                if (at.there) store_vec<float, VEC>(out + at.c, v[j]);
            }
        } else {
            // the rows' sums side by side in LDS, each column added up by one thread
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) store_vec<float, VEC>(sums + sub * COLS + (j * TPR + t) * VEC, v[j]);
            __syncthreads();
            for (int o = threadIdx.x; o < COLS; o += NT) {
                const int first = o / VEC * VEC, i = o % VEC;
                if (first >= n || (MODE == ROW_TINY && i >= n)) continue;
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < PER; ++k) s += sums[k * COLS + o];
                out[(MODE == ROW_RAGGED && first > n - VEC ? n - VEC : first) + i] = s;
            }
        }
    };
    put(dw, slab);
    put(db, slab + n);
}

// Rows beyond the registers.  Both operands are read twice: once row by row for the two means, one
// workgroup per row, and once by columns, for dx and the sums of dw and db together.  (500 x 40000 fp32:
// 71 us, 3.4 TB/s by the three arrays.)
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_means_long_kernel(const LnBwd a) {
    constexpr int VEC = vec_of<T>();
    __shared__ float scratch[16];
    const int n = a.n, vecs = (n + VEC - 1) / VEC;
    float h[VEC], d[VEC], g[VEC];
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *xr = (const T*)a.x + r * a.ldx, *dr = (const T*)a.dy + r * a.lddy;
        const float mean = a.stats[r], rstd = a.stats[a.rows + r];
        float s1 = 0.f, s2 = 0.f;
        for (int j = threadIdx.x; j < vecs; j += 1024) {
            const int c = j * VEC < n - VEC ? j * VEC : n - VEC, skip = j * VEC - c;
            load_vec<T, VEC>(xr + c, h);
            load_vec<T, VEC>(dr + c, d);
            load_weight<ROW_RAGGED>((const W*)a.w, c, n, 1.f, g);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float p = i >= skip ? d[i] * g[i] : 0.f;
                s1 += p;
                s2 = fmaf(p, (h[i] - mean) * rstd, s2);
            }
        }
        s1 = row_sum<1024>(s1, scratch);
        s2 = row_sum<1024>(s2, scratch);
        if (threadIdx.x == 0) {
            a.means[r] = s1 / (float)n;
            a.means[a.rows + r] = s2 / (float)n;
        }
    }
}
// A thread owns the columns of one vector over a slab of rows, four of them in flight.
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_bwd_long_kernel(const LnBwd a) {
    constexpr int VEC = vec_of<T>(), U = 4;
    const int n = a.n, slab = blockIdx.y, slabs = gridDim.y;
    const long long first = ((long long)blockIdx.x * 256 + threadIdx.x) * VEC;
    if (first >= n) return;
    const int c = first < n - VEC ? (int)first : n - VEC;
    const long long r0 = a.rows * slab / slabs, r1 = a.rows * (slab + 1) / slabs;
    float g[VEC], dw[VEC] = {}, db[VEC] = {};
    load_weight<ROW_RAGGED>((const W*)a.w, c, n, 1.f, g);
    for (long long r = r0; r < r1; r += U) {
        raw_t x[U], dy[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long at = r + u < r1 ? r + u : r1 - 1;
            load_cols<ROW_RAGGED>((const T*)a.x + at * a.ldx, c, n, x[u]);
            load_cols<ROW_RAGGED>((const T*)a.dy + at * a.lddy, c, n, dy[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r + u >= r1) break;
            const float mean = a.stats[r + u], rstd = a.stats[a.rows + r + u];
            float h[VEC], d[VEC];
            unpack<T>(x[u], h);
            unpack<T>(dy[u], d);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                h[i] = (h[i] - mean) * rstd;
                dw[i] = fmaf(d[i], h[i], dw[i]);
                db[i] += d[i];
            }
            if (!a.dx) continue;
            const float m1 = a.means[r + u], m2 = a.means[a.rows + r + u];
#pragma unroll
            for (int i = 0; i < VEC; ++i) d[i] = rstd * (fmaf(d[i], g[i], -m1) - h[i] * m2);
            store_cols<ROW_RAGGED>((T*)a.dx + (r + u) * a.lddx, c, n, d, a.stream);
        }
    }
    if (!a.part) return;
    float* out = a.part + (long long)slab * 2 * n + c;
    store_vec<float, VEC>(out, dw);
    store_vec<float, VEC>(out + n, db);
}

// dw and db from the slabs: 32 columns per workgroup, 32 threads a column, added in a fixed order.
template <typename W>
__global__ __launch_bounds__(1024) void ln_dw_finish_kernel(const float* __restrict__ part, int slabs, int n,
                                                            W* __restrict__ dw, W* __restrict__ db, long long first) {
    __shared__ float sum[32][33];
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const long long c = first + (long long)blockIdx.x * 32 + lane, width = 2LL * n;      // column of [dw | db]
    float v = 0.f;
    if (c < width) {
#pragma unroll 8
        for (int s = k; s < slabs; s += 32) v += part[s * width + c];
    }
    sum[k][lane] = v;
    __syncthreads();
    if (k || c >= width) return;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += sum[i][lane];
    W* out = c < n ? dw : db;
    if (out) out[c < n ? c : c - n] = from_f32<W>(v);
}

// ---- launches ---------------------------------------------------------------------------------------------------------
constexpr int CUS = 256;
// Longest row of the backward pass in registers: four (fp32) or two (16 bits) vectors of 1024 threads, and one more where
// there are rows enough that the partial sums, two rows of every workgroup, weigh little (us of reading twice / this, fp32
// rows of 20000: 64 rows 14.6 / 17.1, 1000 68 / 66, 4000 284 / 211).
constexpr int max_held(int vec, long long rows) { return rows < 512 ? 16384 : vec == 4 ? 20480 : 24576; }

// Results of 100 MB and more are stored past the caches (us without / with, GPU busy with this alone: forward of 16384 x
// 4000 fp32 97 / 77, bf16 44.4 / 43.1, and 59 / 53 on inputs that are in no cache; backward of the bf16 rows 82 / 68).  Of
// less, the caches keep a part for the operator that reads them next, and 8192 x 2000 fp32 (66 MB) gains nothing: 22.2 / 21.5
// and 35.7 / 37.7.
bool past_the_caches(long long rows, int n, size_t size) { return (double)rows * n * size >= 1e8; }

// How the backward pass holds a row of `vecs` vectors: TPR threads, at most 32 elements each (five values are kept per
// element); 0: not at all.  nt: threads of a workgroup - half as many where there are not enough rows to give every CU
// eight waves.  Four waves a row and four rows a workgroup (us of one wave a row / this; 1000, 2000, 8000 rows): fp32 of 493
// vectors 15.0 / 12.4, 18.5 / 15.1, 38.3 / 35.1; of 251 vectors 10.4 / 9.6, 11.7 / 9.7, 21.9 / 22.8; fp16 of 126 vectors
// 10.1 / 10.6, 9.6 / 11.0, 15.3 / 22.2.
// slabs: one slab of partial sums per workgroup, which walks the rows: one workgroup per CU.  Rows that are not held: four
// workgroups per CU over columns and slabs, and eight rows or more a slab, so that the partial sums stay a small part of
// what is read.
struct BwdShape { int tpr, nt, slabs; };
BwdShape bwd_shape(long long rows, int n, int vec) {
    const int vecs = (n + vec - 1) / vec, v = 32 / vec;
    BwdShape s;
    const bool four = vecs > 128 && vecs <= 512 && (vecs > 256 || rows <= 8 * CUS);
    s.tpr = vecs <= 4 ? 4 : vecs <= 16 ? 16 : vecs <= 32 ? 32 : vecs <= 256 && !four ? 64 : vecs <= 256 * v ? 256
            : n <= max_held(vec, rows) ? 1024 : 0;
    s.nt = four ? 1024 : s.tpr > 64 ? s.tpr : rows * s.tpr <= 512 * CUS ? 256 : 512;
    if (s.tpr == 0) {
        const long long wide = (n + 256LL * vec - 1) / (256LL * vec), want = 4 * CUS / wide, most = (rows + 7) / 8;
        s.slabs = (int)(want < 1 || most < 1 ? 1 : want < most ? want : most);
        return s;
    }
    const int per = s.nt / s.tpr;
    const long long blocks = (rows + per - 1) / per;
    const int most = s.nt == 256 && s.tpr == 256 ? 2 * CUS : CUS;
    s.slabs = (int)(blocks < 1 ? 1 : blocks < most ? blocks : most);
    return s;
}

template <typename T, typename W>
int ln_fwd(const void* x, long long ldx, long long rows, int n, const void* w, const void* b, float eps, void* y,
           long long ldy, float* stats, hipStream_t st) {
    constexpr int VEC = vec_of<T>();
    const int vecs = (n + VEC - 1) / VEC, mode = row_mode(n, VEC);
    const bool stream = past_the_caches(rows, n, sizeof(T));
#define FWD_MODE(TPR, V, MODE)                                                                                           \
    hipLaunchKernelGGL((ln_fwd_kernel<T, W, TPR, V, MODE>), dim3((unsigned)(blocks < MAX_BLOCKS ? blocks : MAX_BLOCKS)), \
                       dim3(NT), 0, st, (const T*)x, ldx, rows, n, (const W*)w, (const W*)b, eps, (T*)y, ldy, stream, stats)
#define FWD(TPR, V)                                                             \
    do {                                                                        \
        constexpr int NT = TPR > 256 ? TPR : 256;                               \
        const long long blocks = (rows + NT / TPR - 1) / (NT / TPR);            \
        if (mode == ROW_FULL) FWD_MODE(TPR, V, ROW_FULL);                       \
        else FWD_MODE(TPR, V, ROW_RAGGED);                                      \
    } while (0)
    if (mode == ROW_TINY) {
        constexpr int NT = 256;
        const long long blocks = (rows + 63) / 64;
        FWD_MODE(4, 1, ROW_TINY);
    }
    // Few rows: a thread takes one or two vectors, so that the row is there after one trip to memory; many: a wave holds a row by
    // itself and meets no barrier.  us of many / few threads a row, launches on the same rows:
    //                 64 rows     1000       2000        4000        8000        16000
    //   fp32 n 1000   2.6 / 2.9   3.5 / 3.5  4.6 / 4.3   7.3 / 6.2   12.3 / 10.7 21.9 / 20.8
    //   fp32 n 2000   2.9 / 4.0   4.4 / 5.1  6.6 / 6.9   12.1 / 10.8 21.4 / 21.7 38.2 / 39.4
    //   bf16 n 4000   3.3 / 5.4   5.3 / 6.6  7.9 / 8.9   13.3 / 13.1 22.5 / 24.9 41.0 / 41.9
    //   fp32 n 4000   3.4 / 3.5   8.4 / 6.5  14.7 / 10.6 25.7 / 20.6 46.6 / 37.9 89.2 / 73.2
    // (The two meet at some 1000, 3000, 4000 and 256 rows there; the bounds, 4096 and 1024, lie above that.)
    else if (vecs <= 4) FWD(4, 1);
    else if (vecs <= 16) FWD(16, 1);
    else if (vecs <= 32) FWD(32, 1);
    else if (vecs <= 64) FWD(64, 1);
    else if (vecs <= 128) FWD(64, 2);
    else if (vecs <= 256 && rows < 4096) FWD(256, 1);
    else if (vecs <= 256) FWD(64, 4);
    else if (vecs <= 512 && rows < 4096) FWD(256, 2);
    else if (vecs <= 512) FWD(64, 8);
    else if (vecs <= 1024 && rows < 1024) FWD(1024, 1);
    else if (vecs <= 1024) FWD(256, 4);
    else if (vecs <= 2048) FWD(1024, 2);
    else if (vecs <= 4096) FWD(1024, 4);
    else if (vecs <= 5120) FWD(1024, 5);
    else if (VEC == 4 && vecs <= 8192) FWD(1024, (VEC == 4 ? 8 : 5));
    else
        hipLaunchKernelGGL((ln_fwd_long_kernel<T, W>), dim3((unsigned)(rows < MAX_BLOCKS ? rows : MAX_BLOCKS)),
                           dim3(1024), 0, st, (const T*)x, ldx, rows, n, (const W*)w, (const W*)b, eps, (T*)y, ldy, stream,
                           stats);
#undef FWD
#undef FWD_MODE
    SCA_CHECK_LAUNCH();
    return 0;
}

template <typename T, typename W>
int ln_bwd(LnBwd a, void* dw, void* db, hipStream_t st) {
    constexpr int VEC = vec_of<T>(), V = 32 / VEC;
    const int n = a.n, vecs = (n + VEC - 1) / VEC, mode = row_mode(n, VEC);
    const BwdShape sh = bwd_shape(a.rows, n, VEC);
    a.stream = past_the_caches(a.rows, n, sizeof(T));
    if (a.rows > 0 && sh.tpr) {
#define BWD_MODE(TPR, V, MODE, ...)                                                                                       \
    hipLaunchKernelGGL((ln_bwd_kernel<T, W, TPR, V, MODE, __VA_ARGS__>), dim3((unsigned)sh.slabs), dim3(sh.nt), 0, st, a)
#define BWD(TPR, V, NT)                                         \
    do {                                                        \
        if (mode == ROW_FULL) BWD_MODE(TPR, V, ROW_FULL, NT);   \
        else BWD_MODE(TPR, V, ROW_RAGGED, NT);                  \
    } while (0)
#define BWD2(TPR, V)                        \
    do {                                    \
        if (sh.nt == 256) BWD(TPR, V, 256); \
        else BWD(TPR, V, 512);              \
    } while (0)
        if (sh.nt > sh.tpr && sh.tpr == 256 && vecs <= 256) BWD(256, 1, 1024);
        else if (sh.nt > sh.tpr && sh.tpr == 256) BWD(256, 2, 1024);
        else if (mode == ROW_TINY && sh.nt == 256) BWD_MODE(4, 1, ROW_TINY, 256);
        else if (mode == ROW_TINY) BWD_MODE(4, 1, ROW_TINY, 512);
        else if (vecs <= 4) BWD2(4, 1);
        else if (vecs <= 16) BWD2(16, 1);
        else if (vecs <= 32) BWD2(32, 1);
        else if (vecs <= 64) BWD2(64, 1);
        else if (vecs <= 64 * 2) BWD2(64, 2);
        else if (vecs <= 64 * 4) BWD2(64, 4);
        else if (vecs <= 256 * V) BWD(256, V, 256);
        else if (vecs <= 1024 * (V / 2)) BWD(1024, V / 2, 1024);
        else if (mode == ROW_FULL) BWD_MODE(1024, V / 2 + 1, ROW_FULL, 1024, false);
        else BWD_MODE(1024, V / 2 + 1, ROW_RAGGED, 1024, false);
#undef BWD2
#undef BWD
#undef BWD_MODE
    } else if (a.rows > 0) {
        if (a.dx)
            hipLaunchKernelGGL((ln_means_long_kernel<T, W>), dim3((unsigned)(a.rows < MAX_BLOCKS ? a.rows : MAX_BLOCKS)),
                               dim3(1024), 0, st, a);
        hipLaunchKernelGGL((ln_bwd_long_kernel<T, W>), dim3((unsigned)((n + 256LL * VEC - 1) / (256LL * VEC)), sh.slabs),
                           dim3(256), 0, st, a);
    }
    const long long columns = dw || db ? 2LL * n : 0;
    for (long long c = 0; c < columns; c += 32 * MAX_BLOCKS) {           // (more than one launch from n = 2^24 on)
        const long long left = (columns - c + 31) / 32;
        hipLaunchKernelGGL((ln_dw_finish_kernel<W>), dim3((unsigned)(left < MAX_BLOCKS ? left : MAX_BLOCKS)), dim3(1024), 0, st,
                           a.part, a.rows > 0 ? sh.slabs : 0, n, (W*)dw, (W*)db, c);
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
    if (!ln_types_ok(dtype, wtype) || rows < 0 || n <= 0 || n > MAX_N || ldx < 0 || ldy < n || !(eps >= 0.f)) return -1;
    if (rows == 0) return 0;
    if (!x || !y) return -1;
    return LN_DISPATCH(ln_fwd, x, ldx, rows, n, w, b, eps, y, ldy, stats, (hipStream_t)stream);
}

extern "C" long long sca_layernorm_bwd_workspace_floats(long long rows, int n) {
    if (rows < 0 || n <= 0 || n > MAX_N) return -1;
    const BwdShape a = bwd_shape(rows, n, 4), b = bwd_shape(rows, n, 8);             // whatever the type
    return 2LL * n * (a.slabs > b.slabs ? a.slabs : b.slabs) + (a.tpr && b.tpr ? 0 : 2 * rows);
}

extern "C" int sca_layernorm_bwd(const void* dy, long long lddy, const void* x, long long ldx, int dtype,
                                 long long rows, int n, const void* w, int wtype, const float* stats, void* dx,
                                 long long lddx, void* dw, void* db, float* ws, void* stream) {
    if (!ln_types_ok(dtype, wtype) || rows < 0 || n <= 0 || n > MAX_N || lddy < 0 || ldx < 0 || (dx && lddx < n)) return -1;
    if (rows > 0 && (!dy || !x || !stats)) return -1;
    if (!dx && !dw && !db) return 0;
    const int vec = dtype == SCA_F32 ? 4 : 8;
    if (!ws && (dw || db || n > max_held(vec, rows))) return -1;
    LnBwd a{dy, lddy, x, ldx, rows, n, w, stats, dx, lddx, false, dw || db ? ws : nullptr, nullptr};
    if (n > max_held(vec, rows)) a.means = ws + 2LL * n * bwd_shape(rows, n, vec).slabs;
    return LN_DISPATCH(ln_bwd, a, dw, db, (hipStream_t)stream);
}
