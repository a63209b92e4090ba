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
// logits hold.  The maximum and the logarithm of the sum are kept apart for the gradient: their sum loses the logarithm's bits once the
// logits are large.
//
// Bound: HBM -- the logits read once, for a gradient read once more (or not, see GRAD) and the gradient written.  Three layouts:
//  * rows of few classes that lie close together (a map's pixels): a block takes 256 / L rows as one stretch of memory, through LDS;
//  * longer rows, or rows far apart: 16, 64 or 256 lanes a row, straight from memory, a running maximum and sum;
//  * few long rows (one token over a vocabulary): several blocks a row, joined by a second kernel.
// All memory accesses are 16 bytes wide wherever a row starts: the hardware takes them at any element's address, at full rate where that
// is a multiple of 4 (30100 x 2005 f32, every fourth row aligned: 5.0 TB/s read) and slower where it is not (1024 x 50257 bf16, every other
// row: 3.2 TB/s; 2048 x 32000, all rows aligned: 4.1).
// Exponentials are the hardware's exp2 of x log2 e: their relative error grows by 2^-24 for every unit below the row's maximum, where the
// terms are small.
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// N elements, aligned as one of them
template <class T, int N>
struct Vec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
    if constexpr (N == 1) {
        x[0] = (float)*p;
    } else {
        const typename Vec<T, N>::type v = *reinterpret_cast<const typename Vec<T, N>::type*>(p);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = (float)v[j];
    }
}
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
    if constexpr (N == 1) {
        *p = (T)x[0];
    } else {
        typename Vec<T, N>::type v;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (T)x[j];
        *reinterpret_cast<typename Vec<T, N>::type*>(p) = v;
    }
}

constexpr int LP_MAX_BLOCKS = 2048;     // partial sums of the loss
constexpr int COUNT_BLOCKS = 256;       // partial counts of the rows that count
constexpr int TILE_BYTES = 20480;       // 8 blocks of a compute unit at once, 7 with the 128 to 144 bytes more of the loss's partial sums
constexpr int MAX_SPLITS = 64;          // blocks of a long row

enum Mode { LOGP, LOSS, GRAD, BACK };   // GRAD: the loss and, for an upstream gradient of 1, the gradient of the logits

struct Rows {
    int64_t ld, ignore, P;
    const int64_t* label;
    int C;
};
struct ForwardArgs {
    float* lp;                          // LOGP: [P]
    float2* stats;                      // [P] {maximum, logarithm of the sum}, or NULL
    // the loss
    const float* advantage;
    const float* old_logp;
    const float* ref_logp;              // or NULL
    int64_t rows_per_advantage;
    int small_rows;                     // row numbers fit 32 bits (a 64-bit division costs more than a row of 150 classes)
    float clip_low, clip_high, kl_weight;
    float* coef;                        // [P] d(loss * rows that count) / d lp
    double* partial;                    // [blocks][4]: loss, kl, clipped, rows that count
    const int* counts;                  // GRAD: [COUNT_BLOCKS]
};
struct BackArgs {
    const float2* stats;
    const float* g;                     // [P]
    const float* gloss;                 // scalar, or NULL
    const float* inv_count;             // scalar, with gloss
};

// what belongs to a row beside its logits, requested before them
struct RowIn {
    int64_t a;
    bool valid;
    float A, old, ref;                  // LOSS, GRAD: the row's first lane alone
};
template <int MODE>
__device__ __forceinline__ RowIn row_in(const Rows& r, const ForwardArgs& f, int64_t row, bool live, bool lead) {
    RowIn in;
    in.A = in.old = in.ref = 0.f;
    in.a = live ? r.label[row] : -1;
    if (MODE != LOGP && lead && live) {
        const int64_t image = f.small_rows ? (int64_t)((uint32_t)row / (uint32_t)f.rows_per_advantage) : row / f.rows_per_advantage;
        in.A = f.advantage[image];
        in.old = f.old_logp[row];
        if (f.ref_logp) in.ref = f.ref_logp[row];
    }
    in.valid = live && in.a != r.ignore && in.a >= 0 && in.a < r.C;
    return in;
}

struct RowSums {
    double loss = 0.0, kl = 0.0;
    int clipped = 0, count = 0;
};
// one row's answer, by one lane; returns d(loss * rows that count) / d lp
template <int MODE>
__device__ __forceinline__ float finish_row(int64_t row, const RowIn& in, float za, float top, float logs, const ForwardArgs& f, RowSums& acc) {
    const float lp = in.valid ? (za - top) - logs : 0.f;
    if (f.stats) f.stats[row] = make_float2(top, logs);
    float coef = 0.f;
    if constexpr (MODE == LOGP) {
        f.lp[row] = lp;
    } else {
        if (in.valid) {
            const float ratio = expf(lp - in.old);
            const float whole = ratio * in.A;
            const float cut = fminf(fmaxf(ratio, 1.f - f.clip_low), 1.f + f.clip_high) * in.A;
            const bool clip = cut < whole;
            float l = clip ? -cut : -whole;
            coef = clip ? 0.f : -whole;
            if (f.ref_logp) {
                const float d = in.ref - lp;
                const float e = expm1f(d);                           // exp(d) - 1 - d cancels for small d
                const float k = d < INFINITY ? e - d : d;             // a chosen class of probability 0: infinite, not infinity - infinity
                if (f.kl_weight > 0.f) {                              // a term that is only watched may be infinite: 0 times it is not 0
                    l = fmaf(f.kl_weight, k, l);
                    coef = fmaf(-f.kl_weight, e, coef);
                }
                acc.kl += (double)k;
            }
            acc.loss += (double)l;
            acc.clipped += clip ? 1 : 0;
            acc.count += 1;
        }
        f.coef[row] = coef;
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
// the same over a group of G lanes, up to the block (lds: 8 floats; all threads of the block call)
template <int G>
__device__ __forceinline__ float group_max(float v, float* lds) {
    v = lanes_max<(G < 64 ? G : 64)>(v);
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
    v = lanes_sum<(G < 64 ? G : 64)>(v);
    if constexpr (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[4 + (threadIdx.x >> 6)] = v;
        __syncthreads();
        v = (lds[4] + lds[5]) + (lds[6] + lds[7]);
    }
    return v;
}

// ---------------------------------------------------------------- rows of few classes, close together --------------------------
// A block takes 256 / L rows, padding between them included, as one stretch of memory in 16-byte loads that no row's start or end
// interrupts, through LDS; then L lanes read a row each and hold it in registers.  A row alone is 300 to 600 bytes at 150 classes.
// Of 2 x 375 x 501 rows of 150 classes: f32 43 us, f16 27 us (5.2, 4.2 TB/s); a group of lanes per row straight from memory took 64 us in
// f16.  Rows of few classes are far from that rate: a tile has 256 / L rows however short they are, so 375750 rows of 19 classes take 9 to 11
// us in f32 and 7 in bf16 (2.6 to 3.2 and 2.1 TB/s of logits), 1048576 rows of 2 classes 8 us in both (1.1, 0.5).
// A gradient leaves the same way.  GRAD: the row is in registers when its loss is known, so its gradient is written at once and the logits
// are not read by a backward pass (2 x 512 x 512 x 150 f32: loss and gradient 139 us, with a second reading 219 us); it needs
// 1 / (rows that count) beforehand (count_rows_kernel, 8 bytes a row).
// W: elements of a read from LDS (2 where classes and pitch are even); HELD: reads of a lane, all unrolled (with a run-time bound the
// compiler puts the row into scratch memory and f16 rows take five times as long)
template <class T, int L, int W, int HELD, int MODE>
__global__ __launch_bounds__(256) void logp_tile_kernel(const T* __restrict__ z, const Rows r, const ForwardArgs f, const BackArgs k,
                                                        T* __restrict__ dz) {
    constexpr int ROWS = 256 / L, PER = 16 / (int)sizeof(T), LOADS = TILE_BYTES / 4096;
    __shared__ u32x4 tile[TILE_BYTES / 16];
    T* t = reinterpret_cast<T*>(tile);
    const int C = r.C, sub = threadIdx.x % L, mine = threadIdx.x / L;
    const int64_t tiles = (r.P + ROWS - 1) / ROWS;
    RowSums acc;
    float share = 1.f;
    if constexpr (MODE == GRAD) {                                      // 1 / rows that count
        __shared__ int part[4];
        const int s = lanes_sum<64>(f.counts[threadIdx.x]);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        const int n = (part[0] + part[1]) + (part[2] + part[3]);
        share = n > 0 ? 1.f / (float)n : 0.f;
    }
    if constexpr (MODE == BACK) {
        if (k.gloss) share = k.gloss[0] * k.inv_count[0];
    }
    for (int64_t b = blockIdx.x; b < tiles; b += gridDim.x) {
        const int64_t row0 = b * ROWS, row = row0 + mine;
        const int rows = (int)min(r.P - row0, (int64_t)ROWS);
        const bool live = mine < rows;
        const int count = (rows - 1) * (int)r.ld + C;                  // elements of the stretch
        const T* src = z + row0 * r.ld;
        const RowIn in = row_in<MODE == BACK ? LOGP : MODE>(r, f, row, live, sub == 0);
        float2 st = make_float2(0.f, 0.f);
        float g = 0.f;
        if (MODE == BACK && live) {
            st = k.stats[row];
            g = k.g[row];
        }
        const int vecs = count / PER;
        u32x4 v[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            typedef typename Vec<T, PER>::type piece;
            if (vecs) v[u] = __builtin_bit_cast(u32x4, *reinterpret_cast<const piece*>(src + (size_t)min((int)threadIdx.x + u * 256, vecs - 1) * PER));
        }
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
            if ((int)threadIdx.x + u * 256 < vecs) tile[threadIdx.x + u * 256] = v[u];
        for (int i = vecs * PER + threadIdx.x; i < count; i += 256) t[i] = src[i];         // what is no whole piece
        __syncthreads();
        const T* tr = t + (live ? mine : 0) * (int)r.ld;
        float x[HELD][W];
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int c = (sub + i * L) * W;
            if (c < C) {
                load_vec<T, W>(tr + c, x[i]);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) x[i][j] = -INFINITY;
            }
        }
        float over = 1.f;                                              // 1 / sum
        if constexpr (MODE != BACK) {
            const float za = in.valid && sub == 0 ? (float)tr[in.a] : 0.f;
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
#pragma unroll
                for (int j = 0; j < W; ++j) m = fmaxf(m, x[i][j]);
            }
            m = lanes_max<L>(m);
            const float top = m == -INFINITY ? 0.f : m;                // nothing but -infinity: exp(-inf) = 0, not NaN
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    x[i][j] = __expf(x[i][j] - top);
                    s += x[i][j];
                }
            }
            s = lanes_sum<L>(s);
            if (sub == 0 && live) g = finish_row<MODE>(row, in, za, top, logf(s), f, acc);
            if constexpr (MODE == GRAD) {
                g = __shfl(g, (threadIdx.x & 63) / L * L, 64);
                over = 1.f / s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
#pragma unroll
                for (int j = 0; j < W; ++j) x[i][j] = __expf((x[i][j] - st.x) - st.y);
            }
        }
        __syncthreads();                                               // every row has been read: the tile is free
        if constexpr (MODE == GRAD || MODE == BACK) {
            g *= share;
            T* tw = t + mine * C;
            if (live) {
#pragma unroll
                for (int i = 0; i < HELD; ++i) {
                    const int c = (sub + i * L) * W;
#pragma unroll
                    for (int j = 0; j < W; ++j) x[i][j] = in.valid ? g * ((c + j == (int)in.a ? 1.f : 0.f) - x[i][j] * over) : 0.f;
                    if (c < C) store_vec<T, W>(tw + c, x[i]);
                }
            }
            __syncthreads();
            T* dst = dz + row0 * C;                                    // 256 / L rows are whole 16-byte pieces: L <= 16
            const int total = rows * C, pieces = total / PER;
#pragma unroll
            for (int u = 0; u < LOADS; ++u)
                if ((int)threadIdx.x + u * 256 < pieces) reinterpret_cast<u32x4*>(dst)[threadIdx.x + u * 256] = tile[threadIdx.x + u * 256];
            for (int i = pieces * PER + threadIdx.x; i < total; i += 256) dst[i] = t[i];
            __syncthreads();
        }
    }
    if constexpr (MODE == LOSS || MODE == GRAD) block_partial(acc, f.partial);
}

// ---------------------------------------------------------------- longer rows, rows far apart, few rows ------------------------
// H vectors of a row, a group of G lanes' apart, from class c0 on; what lies at or behind `end` is -infinity
template <class T, int G, int V, int H>
__device__ __forceinline__ void load_part(const T* __restrict__ zr, int c0, int end, typename Vec<T, V>::type (&raw)[H]) {
#pragma unroll
    for (int u = 0; u < H; ++u) {
        const int c = c0 + u * (G * V);
        if (c + V <= end) {
            raw[u] = *reinterpret_cast<const typename Vec<T, V>::type*>(zr + c);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) raw[u][j] = c + j < end ? zr[c + j] : (T)-INFINITY;
        }
    }
}
// H: vectors that a lane has in flight, 4, or 8 for the longer rows of a wave (8 for all took 93 us for 120000 x 600 f32, 4 take 59)
// maximum (0 where there is nothing but -infinity) and sum of a lane's part of [begin, end)
template <class T, int G, int H>
__device__ __forceinline__ void lane_sum(const T* __restrict__ zr, int sub, int begin, int end, float& m, float& s) {
    constexpr int V = 16 / (int)sizeof(T), STEP = G * V * H;
    typename Vec<T, V>::type raw[H], next[H];
    m = -INFINITY;
    s = 0.f;
    load_part<T, G, V, H>(zr, begin + sub * V, end, raw);
    for (int c0 = begin + sub * V; c0 < end; c0 += STEP) {
        // a block's row has the next part on its way while one is summed
        if (G == 256 && c0 + STEP < end) load_part<T, G, V, H>(zr, c0 + STEP, end, next);
        __builtin_amdgcn_sched_barrier(0);
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) top = fmaxf(top, (float)raw[u][j]);
        const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
        s *= m == -INFINITY ? 0.f : __expf(m - ref);
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) s += __expf((float)raw[u][j] - ref);
        m = mn;
        if (G < 256) break;                                            // rows of a group fit its lanes' registers (group_of)
#pragma unroll
        for (int u = 0; u < H; ++u) raw[u] = next[u];
    }
}
// part of a sum, taken relative to the maximum `m` of its own, relative to `ref`
__device__ __forceinline__ float rescaled(float s, float m, float ref) { return m == -INFINITY && s == 0.f ? 0.f : s * __expf(m - ref); }

template <class T, int G, int H, int MODE>
__global__ __launch_bounds__(256) void logp_rows_kernel(const T* __restrict__ z, const Rows r, const ForwardArgs f) {
    __shared__ float lds[8];
    constexpr int ROWS = 256 / G;
    const int sub = threadIdx.x % G;
    RowSums acc;
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < r.P; row0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = row0 + threadIdx.x / G;
        const bool live = row < r.P;
        const T* zr = z + (live ? row : 0) * r.ld;
        const RowIn in = row_in<MODE>(r, f, row, live, sub == 0);
        float m = -INFINITY, s = 0.f;
        if (live) lane_sum<T, G, H>(zr, sub, 0, r.C, m, s);
        const float za = in.valid && sub == 0 ? (float)zr[in.a] : 0.f;
        const float top = group_max<G>(m, lds);
        const float ref = top == -INFINITY ? 0.f : top;
        s = group_sum<G>(rescaled(s, m, ref), lds);
        if (sub == 0 && live) finish_row<MODE>(row, in, za, ref, logf(s), f, acc);
    }
    if constexpr (MODE == LOSS) block_partial(acc, f.partial);
}

// few long rows: block (x, y) sums part y of row x, join_rows_kernel the parts.  One row of 131072 f32 classes: 18 us by one block, 5.5 us
// by 32; its gradient 23 and 3 us
template <class T>
__global__ __launch_bounds__(256) void logp_split_kernel(const T* __restrict__ z, const Rows r, int per, float2* __restrict__ parts) {
    __shared__ float lds[8];
    const int begin = (int)min((int64_t)blockIdx.y * per, (int64_t)r.C), end = (int)min((int64_t)begin + per, (int64_t)r.C);
    float m, s;
    lane_sum<T, 256, 4>(z + (int64_t)blockIdx.x * r.ld, threadIdx.x, begin, end, m, s);
    const float top = group_max<256>(m, lds);
    const float ref = top == -INFINITY ? 0.f : top;
    s = group_sum<256>(rescaled(s, m, ref), lds);
    if (threadIdx.x == 0) parts[(int64_t)blockIdx.x * gridDim.y + blockIdx.y] = make_float2(top, s);
}
template <class T, int MODE>
__global__ __launch_bounds__(256) void join_rows_kernel(const T* __restrict__ z, const Rows r, const ForwardArgs f, const float2* __restrict__ parts,
                                                        int splits) {
    RowSums acc;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);      // a wave a row, a lane a part
    const int lane = threadIdx.x & 63;
    const bool live = row < r.P;
    const RowIn in = row_in<MODE>(r, f, row, live, lane == 0);
    float2 p = make_float2(-INFINITY, 0.f);
    if (live && lane < splits) p = parts[row * splits + lane];
    const float za = in.valid && lane == 0 ? (float)z[row * r.ld + in.a] : 0.f;
    const float top = lanes_max<64>(p.x);
    const float ref = top == -INFINITY ? 0.f : top;
    // a part of nothing but -infinity was summed relative to 0
    const float s = lanes_sum<64>(p.x == -INFINITY ? (p.y == 0.f ? 0.f : p.y * __expf(0.f - ref)) : p.y * __expf(p.x - ref));
    if (lane == 0 && live) finish_row<MODE>(row, in, za, ref, logf(s), f, acc);
    if constexpr (MODE == LOSS) block_partial(acc, f.partial);
}

// dz of rows that are no tile; blockIdx.y: part of a long row
template <class T, int G, int H>
__global__ __launch_bounds__(256) void logp_rows_bwd_kernel(const T* __restrict__ z, const Rows r, const BackArgs k, int per, T* __restrict__ dz) {
    constexpr int ROWS = 256 / G, V = 16 / (int)sizeof(T);
    const int sub = threadIdx.x % G;
    const float scale = k.gloss ? k.gloss[0] * k.inv_count[0] : 1.f;
    const int begin = (int)min((int64_t)blockIdx.y * per, (int64_t)r.C), end = (int)min((int64_t)begin + per, (int64_t)r.C);
    for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; row < r.P; row += (int64_t)gridDim.x * ROWS) {
        const T* zr = z + row * r.ld;
        T* dr = dz + row * r.C;
        const int64_t a = r.label[row];
        const bool valid = a != r.ignore && a >= 0 && a < r.C;
        const float2 st = k.stats[row];
        const float g = valid ? k.g[row] * scale : 0.f;
        for (int c0 = begin + sub * V; c0 < end; c0 += G * V * H) {
            typename Vec<T, V>::type raw[H];
            load_part<T, G, V, H>(zr, c0, end, raw);
#pragma unroll
            for (int u = 0; u < H; ++u) {
                const int c = c0 + u * (G * V);
                float x[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float p = __expf(((float)raw[u][j] - st.x) - st.y);
                    x[j] = valid ? g * ((c + j == (int)a ? 1.f : 0.f) - p) : 0.f;
                }
                if (c + V <= end) {
                    store_vec<T, V>(dr + c, x);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (c + j < end) dr[c + j] = (T)x[j];
                }
            }
        }
    }
}

// ---------------------------------------------------------------- sums, counts, scaling ----------------------------------------
// rows that count, per block
__global__ __launch_bounds__(256) void count_rows_kernel(const Rows r, int* __restrict__ counts) {
    __shared__ int part[4];
    int n = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < r.P; i += (int64_t)COUNT_BLOCKS * 256) {
        const int64_t a = r.label[i];
        n += a != r.ignore && a >= 0 && a < r.C ? 1 : 0;
    }
    n = lanes_sum<64>(n);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// out = x g[0]; in place there is nothing to do, and nothing read, where it is 1 (a loss that backward() is called on).  A zero stays one under a factor that is not
// finite (an overflowed loss scale): most are the gradients of rows that do not count
__global__ __launch_bounds__(256) void scale_by_kernel(float* out, const float* x, int64_t n, const float* __restrict__ g) {
    const float s = g[0];
    if (s == 1.f && out == x) return;
    const bool plain = fabsf(s) < INFINITY;
    const f32x4* x4 = reinterpret_cast<const f32x4*>(x);
    f32x4* o4 = reinterpret_cast<f32x4*>(out);
    const int64_t stride = (int64_t)gridDim.x * 256, quads = n >> 2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += stride) {
        f32x4 v = x4[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = plain || v[j] != 0.f ? v[j] * s : v[j];
        o4[i] = v;
    }
    const int64_t i = quads * 4 + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = plain || x[i] != 0.f ? x[i] * s : x[i];
}

struct PolicyOut {
    float* v[4];                        // loss, kl, clipped share, 1 / rows that count; all 0 where no row counts
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

// ---------------------------------------------------------------- host ---------------------------------------------------------
static int bytes_of(int type) { return type == SEMSEG_TYPE_F32 ? 4 : 2; }

// how a call's rows are laid out over lanes and blocks; one rule for the kernels and for the scratch that they need
struct Plan {
    int lanes;          // of a row in the tile kernel; 0: not a tile
    int group;          // else lanes of a row: 16, 64, 256
    int splits, per;    // blocks of a row, and classes of each
    int64_t blocks;     // of the grid's first axis without a limit
};
static Plan plan_of(int bytes, int64_t ld, int64_t P, int C) {
    Plan p{0, 0, 1, C, 0};
    if (P == 1) ld = C;
    // a tile reads the padding between rows too: up to a quarter of a row
    for (int l = 1; l <= 16 && !p.lanes && ld <= C + C / 4; l *= 2)
        if ((256 / l) * ld * bytes <= TILE_BYTES) p.lanes = l;
    if (p.lanes) {
        p.blocks = (P + 256 / p.lanes - 1) / (256 / p.lanes);
        return p;
    }
    const int V = 16 / bytes;
    p.group = C <= 16 * V * 4 ? 16 : C <= 64 * V * 8 ? 64 : 256;
    p.blocks = (P + 256 / p.group - 1) / (256 / p.group);
    if (p.group == 256 && P < 512) {                         // fewer blocks than the 1024 that fill the chip: several of a row
        const int step = 256 * V * 4;
        const int64_t parts = ((int64_t)C + step - 1) / step;
        int64_t s = (1024 + P - 1) / P;
        if (s > MAX_SPLITS) s = MAX_SPLITS;
        if (s > parts) s = parts;
        p.per = (int)((parts + s - 1) / s) * step;
        p.splits = (int)(((int64_t)C + p.per - 1) / p.per);
        if (p.splits == 1) p.per = C;
    }
    return p;
}
static size_t split_bytes(const Plan& p, int64_t P) { return p.splits > 1 ? (size_t)P * p.splits * sizeof(float2) : 0; }

struct Call {
    const void* z;
    Rows r;
    Plan p;
    int mode;
    ForwardArgs f;
    BackArgs k;
    void* dz;
    float2* parts;
    int grid;           // blocks of the kernel that leaves the partial sums of the loss
    hipStream_t st;
};

template <class T, int L, int W, int HELD>
static void tile_launch(Call& c) {
    c.grid = (int)(c.p.blocks < LP_MAX_BLOCKS ? c.p.blocks : LP_MAX_BLOCKS);
    const T* z = (const T*)c.z;
    const dim3 grid(c.grid), block(256);
    if (c.mode == LOGP) {
        auto k = logp_tile_kernel<T, L, W, HELD, LOGP>;
        hipLaunchKernelGGL(k, grid, block, 0, c.st, z, c.r, c.f, c.k, (T*)nullptr);
    } else if (c.mode == LOSS) {
        auto k = logp_tile_kernel<T, L, W, HELD, LOSS>;
        hipLaunchKernelGGL(k, grid, block, 0, c.st, z, c.r, c.f, c.k, (T*)nullptr);
    } else if (c.mode == BACK) {
        auto k = logp_tile_kernel<T, L, W, HELD, BACK>;
        hipLaunchKernelGGL(k, grid, block, 0, c.st, z, c.r, c.f, c.k, (T*)c.dz);
    } else if constexpr (sizeof(T) == 4) {
        auto k = logp_tile_kernel<T, L, W, HELD, GRAD>;
        hipLaunchKernelGGL(k, grid, block, 0, c.st, z, c.r, c.f, c.k, (T*)c.dz);
    }
}
// elements that a lane holds: what the tile has for it (L doubles from there on, so more than half are used), fewer for few classes
template <class T, int L, int W>
static void tile_held(Call& c) {
    constexpr int MOST = TILE_BYTES / 256 / (int)sizeof(T);
    if constexpr (L == 1) {
        if (c.r.C <= 8) return tile_launch<T, L, W, 8 / W>(c);
        if constexpr (MOST > 20) {
            if (c.r.C <= 20) return tile_launch<T, L, W, 20 / W>(c);
        }
    }
    tile_launch<T, L, W, MOST / W>(c);
}
template <class T, int L>
static void tile_wide(Call& c) {
    if (c.r.C % 2 == 0 && c.r.ld % 2 == 0) tile_held<T, L, 2>(c);
    else tile_held<T, L, 1>(c);
}
template <class T, int G, int H>
static void rows_launch(Call& c) {
    const T* z = (const T*)c.z;
    const dim3 block(256);
    if (c.mode == BACK) {
        const int64_t most = 1 << 20;
        auto k = logp_rows_bwd_kernel<T, G, H>;
        hipLaunchKernelGGL(k, dim3((unsigned)(c.p.blocks < most ? c.p.blocks : most), c.p.splits), block, 0, c.st, z, c.r, c.k, c.p.per, (T*)c.dz);
        return;
    }
    if (c.p.splits > 1) {
        auto k = logp_split_kernel<T>;
        hipLaunchKernelGGL(k, dim3((unsigned)c.r.P, c.p.splits), block, 0, c.st, z, c.r, c.p.per, c.parts);
        c.grid = (int)((c.r.P + 3) / 4);
        if (c.mode == LOGP) {
            auto j = join_rows_kernel<T, LOGP>;
            hipLaunchKernelGGL(j, dim3(c.grid), block, 0, c.st, z, c.r, c.f, (const float2*)c.parts, c.p.splits);
        } else {
            auto j = join_rows_kernel<T, LOSS>;
            hipLaunchKernelGGL(j, dim3(c.grid), block, 0, c.st, z, c.r, c.f, (const float2*)c.parts, c.p.splits);
        }
        return;
    }
    if (c.mode == LOGP) {
        const int64_t most = 1 << 20;
        auto k = logp_rows_kernel<T, G, H, LOGP>;
        hipLaunchKernelGGL(k, dim3((unsigned)(c.p.blocks < most ? c.p.blocks : most)), block, 0, c.st, z, c.r, c.f);
    } else {
        c.grid = (int)(c.p.blocks < LP_MAX_BLOCKS ? c.p.blocks : LP_MAX_BLOCKS);
        auto k = logp_rows_kernel<T, G, H, LOSS>;
        hipLaunchKernelGGL(k, dim3(c.grid), block, 0, c.st, z, c.r, c.f);
    }
}
template <class T>
static int typed(Call& c) {
    switch (c.p.lanes) {
        case 1: tile_wide<T, 1>(c); break;
        case 2: tile_wide<T, 2>(c); break;
        case 4: tile_wide<T, 4>(c); break;
        case 8: tile_wide<T, 8>(c); break;
        case 16: tile_wide<T, 16>(c); break;
        default:
            if (c.p.group == 16) rows_launch<T, 16, 4>(c);
            else if (c.p.group == 64 && c.r.C <= 64 * 4 * (16 / (int)sizeof(T))) rows_launch<T, 64, 4>(c);
            else if (c.p.group == 64) rows_launch<T, 64, 8>(c);
            else rows_launch<T, 256, 4>(c);
    }
    SEMSEG_LAUNCH_CHECK();
    return 0;
}
static int dispatch(Call& c, int type) {
    if (type == SEMSEG_TYPE_F32) return typed<float>(c);
    if (type == SEMSEG_TYPE_BF16) return typed<bf16_t>(c);
    return typed<f16_t>(c);
}
static bool call_ok(const void* z, int type, int64_t ld, const int64_t* label, int64_t P, int C) {
    return z && label && (type == SEMSEG_TYPE_F32 || type == SEMSEG_TYPE_BF16 || type == SEMSEG_TYPE_F16) && P > 0 && P <= (int64_t)1 << 40 &&
           C > 0 && C <= 1 << 30 && ld >= C && (P == 1 || ld <= INT64_MAX / 8 / P);
}
static Call call_of(const void* z, int type, int64_t ld, const int64_t* label, int64_t ignore, int64_t P, int C, int mode, void* stream) {
    Call c{};
    c.z = z;
    c.r = Rows{P == 1 ? (int64_t)C : ld, ignore, P, label, C};
    c.p = plan_of(bytes_of(type), ld, P, C);
    c.mode = mode;
    c.st = (hipStream_t)stream;
    return c;
}

extern "C" size_t semseg_label_logp_workspace_bytes(int type, int64_t ld, int64_t P, int C) {
    return P > 0 && C > 0 ? split_bytes(plan_of(bytes_of(type), ld, P, C), P) : 0;
}

extern "C" int semseg_label_logp_fwd(const void* z, int type, int64_t ld, const int64_t* label, int64_t ignore_index, int64_t P, int C,
                                     float* lp, float* stats, void* workspace, size_t workspace_bytes, void* stream) {
    if (!call_ok(z, type, ld, label, P, C) || !lp) return SEMSEG_EINVAL;
    Call c = call_of(z, type, ld, label, ignore_index, P, C, LOGP, stream);
    const size_t need = split_bytes(c.p, P);
    if (need && (!workspace || workspace_bytes < need)) return SEMSEG_EWORKSPACE;
    c.parts = (float2*)workspace;
    c.f.lp = lp;
    c.f.stats = (float2*)stats;
    return dispatch(c, type);
}

// workspace: partial sums of the loss, counts of rows, parts of split rows
constexpr size_t PARTIAL_BYTES = (size_t)LP_MAX_BLOCKS * 4 * sizeof(double);
extern "C" size_t semseg_policy_loss_workspace_bytes(int type, int64_t ld, int64_t P, int C) {
    return PARTIAL_BYTES + COUNT_BLOCKS * sizeof(int) + semseg_label_logp_workspace_bytes(type, ld, P, C);
}

// Whether a loss whose gradient is wanted writes it in its forward pass.  float32 only: an upstream gradient other than 1 multiplies the
// written values, and 16-bit ones would be rounded twice.  From 8 classes on: counting the rows first costs 8 bytes a row, reading the
// logits again 4 C.  GPU time of loss and gradient of logits that are in no cache, two passes against one: 524288 x 150 219 against 139 us,
// 262144 x 150 113 against 75, 65536 x 150 34.6 against 33.3; maps that the cache holds lose by the two launches more: 400000 x 19 32.0 against 33.3,
// 375750 x 8 23.9 against 25.0, 8192 x 150 14.6 against 15.0, 1024 x 150 13.2 against 13.5 (and 5 us of wall time, of 50 to 75); below 8
// classes it is 1048576 x 2 29.7 against 35.9.
constexpr int ONE_PASS_CLASSES = 8;
static bool one_pass_able(const void* z, int type, int64_t ld, int64_t P, int C) {
    return z && type == SEMSEG_TYPE_F32 && P > 0 && P <= 1 << 30 && C > 0 && ld >= C && plan_of(4, ld, P, C).lanes > 0;
}
extern "C" int semseg_policy_loss_one_pass(const void* z, int type, int64_t ld, int64_t P, int C) {
    return one_pass_able(z, type, ld, P, C) && C >= ONE_PASS_CLASSES;
}

extern "C" int semseg_scale_by(float* out, const float* x, int64_t n, const float* g, void* stream) {
    if (!out || !x || !g || n <= 0 || !aligned16(out) || !aligned16(x)) return SEMSEG_EINVAL;
    const int64_t b = (n / 4 + 1023) / 1024;
    hipLaunchKernelGGL(scale_by_kernel, dim3((unsigned)(b < 1 ? 1 : b > 2048 ? 2048 : b)), dim3(256), 0, (hipStream_t)stream, out, x, n, g);
    SEMSEG_LAUNCH_CHECK();
    return 0;
}

extern "C" int semseg_policy_loss_fwd(const void* z, int type, int64_t ld, const int64_t* label, int64_t ignore_index, int64_t P, int C,
                                      const float* advantage, int64_t rows_per_advantage, const float* old_logp, const float* ref_logp,
                                      float clip_low, float clip_high, float kl_weight, float* stats, float* coef, float* loss, float* kl,
                                      float* clipped, float* inv_count, void* dz, void* workspace, size_t workspace_bytes, void* stream) {
    if (!call_ok(z, type, ld, label, P, C) || !advantage || rows_per_advantage <= 0 || !old_logp || !stats || !coef || !loss || !kl ||
        !clipped || !inv_count || !(clip_low >= 0.f && clip_low <= 1.f) || !(clip_high >= 0.f) || !(kl_weight >= 0.f) ||
        (kl_weight > 0.f && !ref_logp) || (dz && (!one_pass_able(z, type, ld, P, C) || !aligned16(dz))))
        return SEMSEG_EINVAL;
    if (!workspace || workspace_bytes < semseg_policy_loss_workspace_bytes(type, ld, P, C) || !aligned16(workspace)) return SEMSEG_EWORKSPACE;
    Call c = call_of(z, type, ld, label, ignore_index, P, C, dz ? GRAD : LOSS, stream);
    int* counts = (int*)((char*)workspace + PARTIAL_BYTES);
    c.parts = (float2*)((char*)workspace + PARTIAL_BYTES + COUNT_BLOCKS * sizeof(int));
    c.dz = dz;
    ForwardArgs& f = c.f;
    f.stats = (float2*)stats;
    f.advantage = advantage; f.old_logp = old_logp; f.ref_logp = ref_logp; f.rows_per_advantage = rows_per_advantage;
    f.small_rows = P <= (int64_t)1 << 31 && rows_per_advantage <= (int64_t)1 << 31;
    f.clip_low = clip_low; f.clip_high = clip_high; f.kl_weight = kl_weight;
    f.coef = coef;
    f.partial = (double*)workspace;
    f.counts = counts;
    if (dz) {
        hipLaunchKernelGGL(count_rows_kernel, dim3(COUNT_BLOCKS), dim3(256), 0, c.st, c.r, counts);
        SEMSEG_LAUNCH_CHECK();
    }
    if (int rc = dispatch(c, type)) return rc;
    hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(256), 0, c.st, (const double*)workspace, c.grid,
                       PolicyOut{{loss, kl, clipped, inv_count}});
    SEMSEG_LAUNCH_CHECK();
    return 0;
}

extern "C" int semseg_label_logp_bwd(const void* z, int type, int64_t ld, const int64_t* label, int64_t ignore_index, const float* stats,
                                     const float* g, const float* gloss, const float* inv_count, int64_t P, int C, void* dz, void* stream) {
    if (!call_ok(z, type, ld, label, P, C) || !stats || !g || !dz || !aligned16(dz) || (gloss && !inv_count)) return SEMSEG_EINVAL;
    Call c = call_of(z, type, ld, label, ignore_index, P, C, BACK, stream);
    c.k = BackArgs{(const float2*)stats, g, gloss, inv_count};
    c.dz = dz;
    return dispatch(c, type);
}
