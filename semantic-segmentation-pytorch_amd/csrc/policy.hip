// Log probability of chosen labels and the clipped policy loss with a KL term over per-row categoricals (gfx950): what a segmentation
// network (one categorical of 150 classes per pixel) needs to be tuned on a reward instead of labels.  Stands beside log_softmax / NLL
// (head.hip); unlike those it never writes a [P, C] map of probabilities.
//
//   lp = z[a] - max z - log sum_c exp(z[c] - max z)
//   d = lp - old;  ratio = exp d;  s = min(ratio A, clip(ratio, 1 - lo, 1 + hi) A);  k = exp(ref - lp) - (ref - lp) - 1
//   loss = sum over valid rows of (-s + w k) / (number of valid rows)
//   dz[c] = g (1[c = a] - exp(z[c] - max z - log sum)),  g = upstream * (-(not clipped) ratio A + w (1 - exp(ref - lp))) / valid rows
//
// Rows are valid where the label is not ignore_index and inside [0, C); the others add nothing and get a zero gradient, whatever their
// logits hold.  A row belongs to G lanes (G = 1, 4, 16, 64 or a block of 256): a running maximum and a running sum, one pass over the
// logits.  The maximum and the logarithm of the sum are kept apart for the gradient (their sum loses the logarithm's bits once the
// logits are large), which is a second pass over the logits and one write.  Bound: HBM.
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <class T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <class T>
struct Vec<T, 1> {
    typedef T type;
};
template <class T, int V>
__device__ __forceinline__ void unpack(const typename Vec<T, V>::type& v, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = (float)v;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = (float)v[j];
    }
}
template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[V]) {
    unpack<T, V>(*reinterpret_cast<const typename Vec<T, V>::type*>(p), x);
}
// H vectors of a row, a group of G lanes' apart; what lies behind the row is -infinity
template <class T, int G, int V, int H>
__device__ __forceinline__ void load_part(const T* __restrict__ zr, int c0, int C, typename Vec<T, V>::type (&raw)[H]) {
#pragma unroll
    for (int u = 0; u < H; ++u) {
        const int c = c0 + u * (G * V);
        if (c + V <= C) {
            raw[u] = *reinterpret_cast<const typename Vec<T, V>::type*>(zr + c);
        } else if constexpr (V == 1) {
            raw[u] = (T)-INFINITY;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) raw[u][j] = c + j < C ? zr[c + j] : (T)-INFINITY;
        }
    }
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
    typename Vec<T, V>::type v;
    if constexpr (V == 1) {
        v = (T)x[0];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (T)x[j];
    }
    *reinterpret_cast<typename Vec<T, V>::type*>(p) = v;
}

constexpr int LP_HELD = 8;              // vectors of a row that a lane holds at once
constexpr int LP_MAX_BLOCKS = 2048;     // partial sums of the loss

struct PolicyArgs {
    const float* advantage;             // [images]
    const float* old_logp;              // [P]
    const float* ref_logp;              // [P] or NULL
    int64_t rows_per_advantage;
    int small_rows;                     // row numbers fit 32 bits (a 64-bit division costs more than a row of 150 classes)
    float clip_low, clip_high, kl_weight;
    float* coef;                        // [P] d(loss * valid rows) / d lp
    double* partial;                    // [blocks][4]: loss, kl, clipped, valid
};

template <int G>
__device__ __forceinline__ float group_max(float v, float* lds) {
    if constexpr (G > 1) {
#pragma unroll
        for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    }
    if constexpr (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
    }
    return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v, float* lds) {
    if constexpr (G > 1) {
#pragma unroll
        for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    }
    if constexpr (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[4 + (threadIdx.x >> 6)] = v;
        __syncthreads();
        v = (lds[4] + lds[5]) + (lds[6] + lds[7]);
    }
    return v;
}

template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
template <int L, class V>
__device__ __forceinline__ V lanes_sum(V v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

struct RowSums {
    double loss = 0.0, kl = 0.0;
    int clipped = 0, count = 0;
};
// one row's answer, by one lane; returns d(loss * rows that count) / d lp
template <bool POLICY>
__device__ __forceinline__ float finish_row(int64_t row, float za, bool valid, float top, float logs, float* __restrict__ lp_out,
                                           float2* __restrict__ stats, const PolicyArgs& pa, RowSums& acc) {
    const float lp = valid ? (za - top) - logs : 0.f;
    if (stats) stats[row] = make_float2(top, logs);
    float coef = 0.f;
    if constexpr (!POLICY) {
        lp_out[row] = lp;
    } else {
        if (valid) {
            const float A = pa.advantage[pa.small_rows ? (int64_t)((uint32_t)row / (uint32_t)pa.rows_per_advantage) : row / pa.rows_per_advantage];
            const float ratio = expf(lp - pa.old_logp[row]);
            const float whole = ratio * A;
            const float cut = fminf(fmaxf(ratio, 1.f - pa.clip_low), 1.f + pa.clip_high) * A;
            const bool clip = cut < whole;
            float l = clip ? -cut : -whole;
            coef = clip ? 0.f : -whole;
            if (pa.ref_logp) {
                const float d = pa.ref_logp[row] - lp;
                const float e = expm1f(d);                           // exp(d) - 1 - d cancels for small d
                const float k = e - d;
                l = fmaf(pa.kl_weight, k, l);
                coef = fmaf(-pa.kl_weight, e, coef);
                acc.kl += (double)k;
            }
            acc.loss += (double)l;
            acc.clipped += clip ? 1 : 0;
            acc.count += 1;
        }
        pa.coef[row] = coef;
    }
    return coef;
}
__device__ __forceinline__ void block_partial(const RowSums& acc, double* __restrict__ partial) {
    __shared__ double sum[4][4];
    const double loss = wave_sum_d(acc.loss), kl = wave_sum_d(acc.kl);
    const double clipped = wave_sum_d((double)acc.clipped), count = wave_sum_d((double)acc.count);
    const int w = threadIdx.x >> 6, j = threadIdx.x;
    if ((threadIdx.x & 63) == 0) { sum[w][0] = loss; sum[w][1] = kl; sum[w][2] = clipped; sum[w][3] = count; }
    __syncthreads();
    if (j < 4) partial[(int64_t)blockIdx.x * 4 + j] = (sum[0][j] + sum[1][j]) + (sum[2][j] + sum[3][j]);
}

// POLICY: the loss (lp is not written); otherwise lp of every row.  stats[row] = {max, log sum} (may be NULL)
template <class T, int G, int V, bool POLICY>
__global__ __launch_bounds__(256) void label_logp_kernel(const T* __restrict__ z, int64_t ld, const int64_t* __restrict__ label,
                                                         int64_t ignore, int64_t P, int C, float* __restrict__ lp_out,
                                                         float2* __restrict__ stats, const PolicyArgs pa) {
    __shared__ float lds[8];
    constexpr int ROWS = 256 / G;
    const int sub = threadIdx.x % G;
    RowSums acc;
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < P; row0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = row0 + threadIdx.x / G;
        const bool live = row < P;
        const T* zr = z + (live ? row : 0) * ld;
        const int64_t a = live ? label[row] : -1;
        const bool valid = live && a != ignore && a >= 0 && a < C;
        const float za = valid ? (float)zr[a] : 0.f;
        float m = -INFINITY, s = 0.f;
        if (live) {
            // a long row (a block's) has the next part on its way while one is summed
            constexpr int HELD = G == 256 ? LP_HELD / 2 : LP_HELD;
            typename Vec<T, V>::type raw[HELD], next[HELD];
            load_part<T, G, V, HELD>(zr, sub * V, C, raw);
            for (int c0 = sub * V; c0 < C; c0 += G * V * HELD) {
                if (G == 256 && c0 + G * V * HELD < C) load_part<T, G, V, HELD>(zr, c0 + G * V * HELD, C, next);
                __builtin_amdgcn_sched_barrier(0);
                float x[HELD][V];
                float top = -INFINITY;
#pragma unroll
                for (int u = 0; u < HELD; ++u) {
                    unpack<T, V>(raw[u], x[u]);
#pragma unroll
                    for (int j = 0; j < V; ++j) top = fmaxf(top, x[u][j]);
                }
                const float mn = fmaxf(m, top);
                const float ref = mn == -INFINITY ? 0.f : mn;            // nothing but -infinity so far: exp(-inf) = 0, not NaN
                s *= m == -INFINITY ? 0.f : __expf(m - ref);
#pragma unroll
                for (int u = 0; u < HELD; ++u)
#pragma unroll
                    for (int j = 0; j < V; ++j) s += __expf(x[u][j] - ref);
                m = mn;
                if (G < 256) break;                                      // rows of a group fit its lanes' registers (group_of)
#pragma unroll
                for (int u = 0; u < HELD; ++u) raw[u] = next[u];
            }
        }
        const float top = group_max<G>(m, lds);
        const float ref = top == -INFINITY ? 0.f : top;
        s = group_sum<G>(m == -INFINITY && s == 0.f ? 0.f : s * __expf(m - ref), lds);
        const float logs = logf(s);
        if (sub == 0 && live) finish_row<POLICY>(row, za, valid, ref, logs, lp_out, stats, pa, acc);
    }
    if constexpr (POLICY) block_partial(acc, pa.partial);
}

// Dense rows of few classes: a block takes 256 / L rows, one stretch of memory, in 16-byte loads that no row's start or end interrupts,
// through LDS; then L lanes read a row each.  A row alone is 300 to 600 bytes at 150 classes: loads of its own are 4 or 8 bytes wide.
constexpr int TILE_BYTES = 20480;       // 8 blocks of a compute unit at once
//
// GRAD: the rows are in registers when the loss of a row is known, so their gradient for an upstream gradient of 1 is written at once,
// through the same tile: the logits are read once and not again by a backward pass.  It needs 1 / (rows that count) beforehand
// (count_rows_kernel, 8 bytes a row).
constexpr int COUNT_BLOCKS = 256;
template <class T, int L, int W, bool POLICY, bool GRAD>
__global__ __launch_bounds__(256) void label_logp_tile_kernel(const T* __restrict__ z, const int64_t* __restrict__ label, int64_t ignore,
                                                              int64_t P, int C, float* __restrict__ lp_out, float2* __restrict__ stats,
                                                              const PolicyArgs pa, const int* __restrict__ counts, T* __restrict__ dz) {
    constexpr int ROWS = 256 / L, PER = 16 / (int)sizeof(T);
    constexpr int HELD = TILE_BYTES / 256 / ((int)sizeof(T) * W);      // W: elements of a read from LDS (2 where C is even)
    __shared__ u32x4 tile[TILE_BYTES / 16];
    const int sub = threadIdx.x % L;
    const int64_t tiles = (P + ROWS - 1) / ROWS;
    RowSums acc;
    float share = 0.f;                                                 // 1 / rows that count
    if constexpr (GRAD) {
        __shared__ int part[4];
        const int s = lanes_sum<64>(counts[threadIdx.x]);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        const int n = (part[0] + part[1]) + (part[2] + part[3]);
        share = n > 0 ? 1.f / (float)n : 0.f;
    }
    for (int64_t b = blockIdx.x; b < tiles; b += gridDim.x) {
        const int64_t row0 = b * ROWS, row = row0 + threadIdx.x / L;
        const int count = (int)min(P - row0, (int64_t)ROWS) * C;       // elements of this tile
        const T* src = z + row0 * C;                                   // ROWS * C elements are whole 16-byte pieces: L <= 16
        const int vecs = count / PER;
        const bool live = row < P;
        const int64_t a = live ? label[row] : -1;
        u32x4 v[TILE_BYTES / 4096];
#pragma unroll
        for (int u = 0; u < TILE_BYTES / 4096; ++u)
            v[u] = vecs ? reinterpret_cast<const u32x4*>(src)[min((int)threadIdx.x + u * 256, vecs - 1)] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int u = 0; u < TILE_BYTES / 4096; ++u)
            if ((int)threadIdx.x + u * 256 < vecs) tile[threadIdx.x + u * 256] = v[u];
        T* t = reinterpret_cast<T*>(tile);
        for (int i = vecs * PER + threadIdx.x; i < count; i += 256) t[i] = src[i];         // the end of the last tile
        __syncthreads();
        const bool valid = live && a != ignore && a >= 0 && a < C;
        const T* tr = t + (live ? threadIdx.x / L : 0) * C;
        float x[HELD][W];
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            const int c = (sub + k * L) * W;
            if (c < C) {
                load_vec<T, W>(tr + c, x[k]);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) x[k][j] = -INFINITY;
            }
        }
#pragma unroll
        for (int k = 0; k < HELD; ++k)
#pragma unroll
            for (int j = 0; j < W; ++j) m = fmaxf(m, x[k][j]);
        m = lanes_max<L>(m);
        const float top = m == -INFINITY ? 0.f : m;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < HELD; ++k)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                x[k][j] = __expf(x[k][j] - top);
                s += x[k][j];
            }
        s = lanes_sum<L>(s);
        float coef = 0.f;
        if (sub == 0 && live) coef = finish_row<POLICY>(row, valid ? (float)tr[a] : 0.f, valid, top, logf(s), lp_out, stats, pa, acc);
        if constexpr (GRAD) {
            const float g = __shfl(coef, (threadIdx.x & 63) / L * L, 64) * share, over = 1.f / s;
            T* tw = t + threadIdx.x / L * C;
            if (live) {
#pragma unroll
                for (int k = 0; k < HELD; ++k) {
                    const int c = (sub + k * L) * W;
#pragma unroll
                    for (int j = 0; j < W; ++j) x[k][j] = valid ? g * ((c + j == (int)a ? 1.f : 0.f) - x[k][j] * over) : 0.f;
                    if (c < C) store_vec<T, W>(tw + c, x[k]);
                }
            }
            __syncthreads();
            T* dst = dz + row0 * C;
#pragma unroll
            for (int u = 0; u < TILE_BYTES / 4096; ++u)
                if ((int)threadIdx.x + u * 256 < vecs) reinterpret_cast<u32x4*>(dst)[threadIdx.x + u * 256] = tile[threadIdx.x + u * 256];
            for (int i = vecs * PER + threadIdx.x; i < count; i += 256) dst[i] = t[i];
        }
        __syncthreads();
    }
    if constexpr (POLICY) block_partial(acc, pa.partial);
}

// rows that count, per block
__global__ __launch_bounds__(256) void count_rows_kernel(const int64_t* __restrict__ label, int64_t ignore, int64_t P, int C,
                                                         int* __restrict__ counts) {
    __shared__ int part[4];
    int n = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < P; i += (int64_t)COUNT_BLOCKS * 256) {
        const int64_t a = label[i];
        n += a != ignore && a >= 0 && a < C ? 1 : 0;
    }
    n = lanes_sum<64>(n);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// x *= g[0]; nothing to do, and nothing read, where it is 1 (a loss that backward() is called on)
__global__ __launch_bounds__(256) void scale_by_kernel(float* __restrict__ x, int64_t n, const float* __restrict__ g) {
    const float f = g[0];
    if (f == 1.f) return;
    f32x4* x4 = reinterpret_cast<f32x4*>(x);
    const int64_t stride = (int64_t)gridDim.x * 256, quads = n >> 2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += stride) x4[i] = x4[i] * f;
    const int64_t i = quads * 4 + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) x[i] *= f;
}

struct PolicyOut {
    float* v[4];                        // loss, kl, clipped share, 1 / valid rows; all 0 where no row is valid
};
__global__ __launch_bounds__(256) void policy_finish_kernel(const double* __restrict__ partial, int blocks, const PolicyOut out) {
    __shared__ double sum[4][4];
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    for (int b = threadIdx.x; b < blocks; b += 256)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += partial[(int64_t)b * 4 + j];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double s = wave_sum_d(v[j]);
        if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6][j] = s;
    }
    __syncthreads();
    if (threadIdx.x < 4) {
        const int j = threadIdx.x;
        const double n = (sum[0][3] + sum[1][3]) + (sum[2][3] + sum[3][3]);
        const double x = (sum[0][j] + sum[1][j]) + (sum[2][j] + sum[3][j]);
        out.v[j][0] = n > 0.0 ? (float)((j < 3 ? x : 1.0) / n) : 0.f;
    }
}

// dz = g * scale * (1[c = a] - p); scale = gloss[0] * inv_count[0] where given, else 1
template <class T, int G, int V>
__global__ __launch_bounds__(256) void label_logp_bwd_kernel(const T* __restrict__ z, int64_t ld, const int64_t* __restrict__ label,
                                                             int64_t ignore, const float2* __restrict__ stats,
                                                             const float* __restrict__ g, const float* __restrict__ gloss,
                                                             const float* __restrict__ inv_count, T* __restrict__ dz, int64_t P, int C) {
    constexpr int ROWS = 256 / G;
    const int sub = threadIdx.x % G;
    const float scale = gloss ? gloss[0] * inv_count[0] : 1.f;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; row < P; row += (int64_t)gridDim.x * ROWS) {
        const T* zr = z + row * ld;
        T* dr = dz + row * C;
        const int64_t a = label[row];
        const bool valid = a != ignore && a >= 0 && a < C;
        const float2 st = stats[row];
        const float gr = valid ? g[row] * scale : 0.f;
        for (int c0 = sub * V; c0 < C; c0 += G * V * LP_HELD) {
            float x[LP_HELD][V];
#pragma unroll
            for (int u = 0; u < LP_HELD; ++u) {
                const int c = c0 + u * (G * V);
                if (c + V <= C) {
                    load_vec<T, V>(zr + c, x[u]);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) x[u][j] = c + j < C ? (float)zr[c + j] : 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < LP_HELD; ++u) {
                const int c = c0 + u * (G * V);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float p = __expf((x[u][j] - st.x) - st.y);
                    x[u][j] = valid ? gr * ((c + j == (int)a ? 1.f : 0.f) - p) : 0.f;
                }
                if (c + V <= C) {
                    store_vec<T, V>(dr + c, x[u]);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (c + j < C) dr[c + j] = (T)x[u][j];
                }
            }
        }
    }
}

// ---------------------------------------------------------------- host ---------------------------------------------------------
// lanes of a row: the fewest of 1, 4, 16, 64, 256 that hold it in LP_HELD vectors each; a longer row is walked by a block
static int group_of(int C, int V) {
    for (int g = 1; g < 256; g *= 4)
        if ((int64_t)g * V * LP_HELD >= C) return g;
    return 256;
}
// elements of a load: the widest that every row start (and, for the gradient, every row of dz) is aligned to
static int vec_of(int bytes, const void* z, int64_t ld, const void* dz, int C) {
    for (int v = 16 / bytes; v > 1; v >>= (bytes == 2 && v == 8 ? 2 : 1)) {
        const int64_t a = (int64_t)v * bytes;
        if (((uintptr_t)z % a) == 0 && (ld * bytes) % a == 0 && (!dz || (((uintptr_t)dz % a) == 0 && ((int64_t)C * bytes) % a == 0))) return v;
    }
    return 1;
}
static int lp_blocks(int64_t P, int G, int cap) {
    const int64_t b = (P + 256 / G - 1) / (256 / G);
    return (int)(b < cap ? b : cap);
}

struct LpCall {
    const void* z; int64_t ld; const int64_t* label; int64_t ignore; int64_t P; int C; float2* stats; hipStream_t st;
    // forward
    float* lp; const PolicyArgs* pa; void* grad; const int* counts;
    // backward
    const float* g; const float* gloss; const float* inv_count; void* dz;
};

template <class T, int G, int V>
static int lp_launch(const LpCall& c) {
    if (c.dz) {
        auto k = label_logp_bwd_kernel<T, G, V>;
        hipLaunchKernelGGL(k, dim3(lp_blocks(c.P, G, 1 << 20)), dim3(256), 0, c.st, (const T*)c.z, c.ld, c.label, c.ignore,
                           (const float2*)c.stats, c.g, c.gloss, c.inv_count, (T*)c.dz, c.P, c.C);
    } else if (c.pa) {
        auto k = label_logp_kernel<T, G, V, true>;
        hipLaunchKernelGGL(k, dim3(lp_blocks(c.P, G, LP_MAX_BLOCKS)), dim3(256), 0, c.st, (const T*)c.z, c.ld, c.label, c.ignore, c.P, c.C,
                           (float*)nullptr, c.stats, *c.pa);
    } else {
        auto k = label_logp_kernel<T, G, V, false>;
        hipLaunchKernelGGL(k, dim3(lp_blocks(c.P, G, 1 << 20)), dim3(256), 0, c.st, (const T*)c.z, c.ld, c.label, c.ignore, c.P, c.C, c.lp,
                           c.stats, PolicyArgs{});
    }
    SEMSEG_LAUNCH_CHECK();
    return 0;
}
template <class T, int V>
static int lp_group(const LpCall& c, int G) {
    switch (G) {
        case 1: return lp_launch<T, 1, V>(c);
        case 4: return lp_launch<T, 4, V>(c);
        case 16: return lp_launch<T, 16, V>(c);
        case 64: return lp_launch<T, 64, V>(c);
        default: return lp_launch<T, 256, V>(c);
    }
}
// lanes of a row in the tile kernel: the fewest whose rows fit the tile; 0: rows too long, not dense or not aligned
static int tile_lanes(int bytes, const void* z, int64_t ld, int64_t P, int C) {
    if ((ld != C && P > 1) || !aligned16(z)) return 0;
    for (int l = 1; l <= 16; l *= 2)
        if ((int64_t)(256 / l) * C * bytes <= TILE_BYTES) return l;
    return 0;
}
template <class T, int L, int W>
static int tile_launch(const LpCall& c) {
    const int64_t tiles = (c.P + 256 / L - 1) / (256 / L);
    const dim3 grid((unsigned)(tiles < LP_MAX_BLOCKS ? tiles : LP_MAX_BLOCKS)), block(256);
    const T* z = (const T*)c.z;
    if (c.grad) {
        if constexpr (sizeof(T) == 4) {
            auto k = label_logp_tile_kernel<T, L, W, true, true>;
            hipLaunchKernelGGL(k, grid, block, 0, c.st, z, c.label, c.ignore, c.P, c.C, (float*)nullptr, c.stats, *c.pa, c.counts, (T*)c.grad);
        }
    } else if (c.pa) {
        auto k = label_logp_tile_kernel<T, L, W, true, false>;
        hipLaunchKernelGGL(k, grid, block, 0, c.st, z, c.label, c.ignore, c.P, c.C, (float*)nullptr, c.stats, *c.pa, (const int*)nullptr,
                           (T*)nullptr);
    } else {
        auto k = label_logp_tile_kernel<T, L, W, false, false>;
        hipLaunchKernelGGL(k, grid, block, 0, c.st, z, c.label, c.ignore, c.P, c.C, c.lp, c.stats, PolicyArgs{}, (const int*)nullptr,
                           (T*)nullptr);
    }
    SEMSEG_LAUNCH_CHECK();
    return 0;
}
template <class T>
static int lp_typed(const LpCall& c) {
    if (!c.dz) {
        switch (tile_lanes((int)sizeof(T), c.z, c.ld, c.P, c.C)) {
            case 1: return c.C % 2 ? tile_launch<T, 1, 1>(c) : tile_launch<T, 1, 2>(c);
            case 2: return c.C % 2 ? tile_launch<T, 2, 1>(c) : tile_launch<T, 2, 2>(c);
            case 4: return c.C % 2 ? tile_launch<T, 4, 1>(c) : tile_launch<T, 4, 2>(c);
            case 8: return c.C % 2 ? tile_launch<T, 8, 1>(c) : tile_launch<T, 8, 2>(c);
            case 16: return c.C % 2 ? tile_launch<T, 16, 1>(c) : tile_launch<T, 16, 2>(c);
            default: break;
        }
    }
    const int V = vec_of((int)sizeof(T), c.z, c.ld, c.dz, c.C);
    const int G = group_of(c.C, V);
    if constexpr (sizeof(T) == 4) {
        return V == 4 ? lp_group<T, 4>(c, G) : V == 2 ? lp_group<T, 2>(c, G) : lp_group<T, 1>(c, G);
    } else {
        return V == 8 ? lp_group<T, 8>(c, G) : V == 2 ? lp_group<T, 2>(c, G) : lp_group<T, 1>(c, G);
    }
}
static int lp_dispatch(const LpCall& c, int type) {
    if (type == SEMSEG_TYPE_F32) return lp_typed<float>(c);
    if (type == SEMSEG_TYPE_BF16) return lp_typed<bf16_t>(c);
    if (type == SEMSEG_TYPE_F16) return lp_typed<f16_t>(c);
    return SEMSEG_EINVAL;
}
static bool lp_ok(const void* z, int64_t ld, const int64_t* label, int64_t P, int C) {
    return z && label && P > 0 && P <= (int64_t)1 << 40 && C > 0 && C <= 1 << 30 && ld >= C && (P == 1 || ld <= INT64_MAX / 8 / P);
}

extern "C" int semseg_label_logp_fwd(const void* z, int type, int64_t ld, const int64_t* label, int64_t ignore_index, int64_t P, int C,
                                     float* lp, float* stats, void* stream) {
    if (!lp_ok(z, ld, label, P, C) || !lp) return SEMSEG_EINVAL;
    LpCall c{};
    c.z = z; c.ld = ld; c.label = label; c.ignore = ignore_index; c.P = P; c.C = C; c.stats = (float2*)stats; c.st = (hipStream_t)stream;
    c.lp = lp;
    return lp_dispatch(c, type);
}

extern "C" size_t semseg_policy_loss_workspace_bytes(void) { return (size_t)LP_MAX_BLOCKS * 4 * sizeof(double) + COUNT_BLOCKS * sizeof(int); }

// Whether a loss whose gradient is wanted writes it in its forward pass.  float32 only: an upstream gradient other than 1 multiplies the
// written values, and 16-bit ones would be rounded twice.  From 8 classes on: counting the rows first costs 8 bytes a row, reading the
// logits again 4 C.  GPU time of loss and gradient, two passes against one: 262144 x 150 108 against 77 us, 65536 x 150 35.7 against 32.5,
// 400000 x 19 37.4 against 34.2, 1024 x 150 13.8 against 14.2 (its backward pass is cheaper to issue: 127 against 119 us of wall time),
// 2000000 x 2 49.4 against 54.5.
constexpr int ONE_PASS_CLASSES = 8;
static bool one_pass_able(const void* z, int type, int64_t ld, int64_t P, int C) {
    return z && type == SEMSEG_TYPE_F32 && P > 0 && P <= 1 << 30 && C > 0 && tile_lanes(4, z, ld, P, C) > 0;
}
extern "C" int semseg_policy_loss_one_pass(const void* z, int type, int64_t ld, int64_t P, int C) {
    return one_pass_able(z, type, ld, P, C) && C >= ONE_PASS_CLASSES;
}

extern "C" int semseg_scale_by(float* x, int64_t n, const float* g, void* stream) {
    if (!x || !g || n <= 0 || !aligned16(x)) return SEMSEG_EINVAL;
    const int64_t b = (n / 4 + 1023) / 1024;
    hipLaunchKernelGGL(scale_by_kernel, dim3((unsigned)(b < 1 ? 1 : b > 2048 ? 2048 : b)), dim3(256), 0, (hipStream_t)stream, x, n, g);
    SEMSEG_LAUNCH_CHECK();
    return 0;
}

extern "C" int semseg_policy_loss_fwd(const void* z, int type, int64_t ld, const int64_t* label, int64_t ignore_index, int64_t P, int C,
                                      const float* advantage, int64_t rows_per_advantage, const float* old_logp, const float* ref_logp,
                                      float clip_low, float clip_high, float kl_weight, float* stats, float* coef, float* loss, float* kl,
                                      float* clipped, float* inv_count, void* dz, void* workspace, size_t workspace_bytes, void* stream) {
    if (!lp_ok(z, ld, label, P, C) || !advantage || rows_per_advantage <= 0 || !old_logp || !stats || !coef || !loss || !kl || !clipped || !inv_count ||
        !(clip_low >= 0.f && clip_low <= 1.f) || !(clip_high >= 0.f) || !(kl_weight >= 0.f) || (kl_weight > 0.f && !ref_logp))
        return SEMSEG_EINVAL;
    if (!workspace || workspace_bytes < semseg_policy_loss_workspace_bytes()) return SEMSEG_EWORKSPACE;
    PolicyArgs pa{};
    pa.advantage = advantage; pa.old_logp = old_logp; pa.ref_logp = ref_logp; pa.rows_per_advantage = rows_per_advantage;
    pa.small_rows = P <= (int64_t)1 << 31 && rows_per_advantage <= (int64_t)1 << 31;
    pa.clip_low = clip_low; pa.clip_high = clip_high; pa.kl_weight = kl_weight; pa.coef = coef; pa.partial = (double*)workspace;
    LpCall c{};
    c.z = z; c.ld = ld; c.label = label; c.ignore = ignore_index; c.P = P; c.C = C; c.stats = (float2*)stats; c.st = (hipStream_t)stream;
    c.pa = &pa;
    if (dz) {
        if (!one_pass_able(z, type, ld, P, C) || !aligned16(dz)) return SEMSEG_EINVAL;
        int* counts = (int*)((char*)workspace + (size_t)LP_MAX_BLOCKS * 4 * sizeof(double));
        hipLaunchKernelGGL(count_rows_kernel, dim3(COUNT_BLOCKS), dim3(256), 0, c.st, label, ignore_index, P, C, counts);
        SEMSEG_LAUNCH_CHECK();
        c.grad = dz;
        c.counts = counts;
    }
    if (int rc = lp_dispatch(c, type)) return rc;
    const int bytes = type == SEMSEG_TYPE_F32 ? 4 : 2;
    const int l = tile_lanes(bytes, z, ld, P, C);
    const int blocks = lp_blocks(P, l ? l : group_of(C, vec_of(bytes, z, ld, nullptr, C)), LP_MAX_BLOCKS);
    hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(256), 0, c.st, (const double*)workspace, blocks,
                       PolicyOut{{loss, kl, clipped, inv_count}});
    SEMSEG_LAUNCH_CHECK();
    return 0;
}

extern "C" int semseg_label_logp_bwd(const void* z, int type, int64_t ld, const int64_t* label, int64_t ignore_index, const float* stats,
                                     const float* g, const float* gloss, const float* inv_count, int64_t P, int C, void* dz, void* stream) {
    if (!lp_ok(z, ld, label, P, C) || !stats || !g || !dz || (gloss && !inv_count)) return SEMSEG_EINVAL;
    LpCall c{};
    c.z = z; c.ld = ld; c.label = label; c.ignore = ignore_index; c.P = P; c.C = C; c.stats = (float2*)stats; c.st = (hipStream_t)stream;
    c.g = g; c.gloss = gloss; c.inv_count = inv_count; c.dz = dz;
    return lp_dispatch(c, type);
}
