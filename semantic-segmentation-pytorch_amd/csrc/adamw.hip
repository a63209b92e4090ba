// AdamW over many tensors at once, states in 32 bits or in 8 (adamw_math.h has the mathematics), and the global norm of many
// gradients (gfx950).  The framework's other optimiser is sgd_fused_kernel (head.hip).
//
// Bound: HBM.  A step with f32 gradients moves 28 bytes an element with states in 32 bits (p, m, v both ways, g once) and 16 with
// states in 8 bits; the norm moves the gradients once.  Layout of the work: every tensor is cut into chunks, a launch is the chunks of all
// tensors one after the other, and a block finds its tensor by comparing its number with the tensors' first chunks, 64 at a time, so no
// block is launched for nothing and no tensor needs a launch of its own.  The table of tensors of an AdamW step lies in the workspace: a
// small kernel before the step, which advances the step counts and forms the coefficients, copies it there from its arguments (a launch
// of the step per 48 tensors, with the table in its arguments, took 10 % longer for 168 tensors).  Step counts, learning rate and clip
// factor are device memory: a captured graph can be replayed.
#include "common.h"
#include "adamw_math.h"

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int ADAM_MAX_TENSORS = 1024;     // of one launch of a step
constexpr int ADAM_CHUNK = 4096;           // elements of a block: 4 quads a thread
constexpr int ADAM_QUADS = ADAM_CHUNK / (256 * 4);

static bool type_ok(int t) { return t == SEMSEG_TYPE_F32 || t == SEMSEG_TYPE_BF16 || t == SEMSEG_TYPE_F16; }
static int type_bytes(int t) { return t == SEMSEG_TYPE_F32 ? 4 : 2; }
static bool aligned_to(const void* p, int bytes) { return (((uintptr_t)p) & (uintptr_t)(bytes - 1)) == 0; }

// four gradients from element 4 * quad; `type` is the same for the whole block
__device__ __forceinline__ f32x4 load_quad(const void* g, int type, int64_t quad) {
    if (type == SEMSEG_TYPE_F32) return reinterpret_cast<const f32x4*>(g)[quad];
    if (type == SEMSEG_TYPE_BF16) return __builtin_convertvector(reinterpret_cast<const bf16x4*>(g)[quad], f32x4);
    return __builtin_convertvector(reinterpret_cast<const f16x4*>(g)[quad], f32x4);
}
__device__ __forceinline__ float load_one(const void* g, int type, int64_t i) {
    if (type == SEMSEG_TYPE_F32) return reinterpret_cast<const float*>(g)[i];
    if (type == SEMSEG_TYPE_BF16) return (float)reinterpret_cast<const __bf16*>(g)[i];
    return (float)reinterpret_cast<const _Float16*>(g)[i];
}
// the 16-bit copy of the updated parameters, rounded to nearest even from the f32 values
__device__ __forceinline__ void store_quad(void* c, int type, int64_t quad, f32x4 v) {
    if (type == SEMSEG_TYPE_BF16) reinterpret_cast<bf16x4*>(c)[quad] = __builtin_convertvector(v, bf16x4);
    else reinterpret_cast<f16x4*>(c)[quad] = __builtin_convertvector(v, f16x4);
}
__device__ __forceinline__ void store_one(void* c, int type, int64_t i, float v) {
    if (type == SEMSEG_TYPE_BF16) reinterpret_cast<__bf16*>(c)[i] = (__bf16)v;
    else reinterpret_cast<_Float16*>(c)[i] = (_Float16)v;
}

// the tensor whose chunks hold block `b`: as many first chunks are not behind it, less one.  One comparison a lane.
__device__ __forceinline__ int tensor_of(const uint32_t* first, int n, uint32_t b) {
    const int lane = threadIdx.x & 63;
    int count = 0;
    for (int base = 0; base < n; base += 64) count += __popcll(__ballot(base + lane < n && first[min(base + lane, n - 1)] <= b));
    return __builtin_amdgcn_readfirstlane(count) - 1;
}

// ---------------------------------------------------------------- step counts, coefficients, table ----------------------------
struct AdamEntry {                  // one tensor, states in 32 bits
    float* p; const void* g; void* c; float* m; float* v;
    int64_t numel;
    AdamCoef coef;
    uint8_t gtype, ctype, vec, pad;
};
struct Adam8Entry {                 // one tensor, states in 8 bits
    float* p; const void* g; void* c; uint8_t* m; float* ms; uint8_t* r; float* rs;
    int64_t numel;
    AdamCoef coef;
    uint8_t gtype, ctype, vec, pad;
};
// what the small kernel gets of a tensor in its arguments
struct AdamItem {
    float* p; const void* g; void* c; float* m; float* v; int* step;
    int64_t numel;
    float wd;
    uint32_t first;
    uint8_t gtype, ctype, vec, pad;
};
struct Adam8Item {
    float* p; const void* g; void* c; uint8_t* m; float* ms; uint8_t* r; float* rs; int* step;
    int64_t numel;
    float wd;
    uint32_t first;
    uint8_t gtype, ctype, vec, pad;
};
__device__ __forceinline__ void put_states(AdamEntry& e, const AdamItem& i) { e.m = i.m; e.v = i.v; }
__device__ __forceinline__ void put_states(Adam8Entry& e, const Adam8Item& i) { e.m = i.m; e.ms = i.ms; e.r = i.r; e.rs = i.rs; }

template <class ITEM, int MOST>
struct BeginBatch {
    static constexpr int MAX = MOST;
    ITEM item[MAX];
    int n, base;                    // tensors of this batch, and the index of the first one in the call
};
struct BeginArgs {
    const float* lr; const float* clip;
    double log_b1, log_b2;
    float grad_scale;
    uint32_t seed;
};

template <class ITEM, class ENTRY, int MOST>
__global__ __launch_bounds__(64) void adamw_begin_kernel(const BeginBatch<ITEM, MOST> b, const BeginArgs a, ENTRY* __restrict__ table,
                                                         uint32_t* __restrict__ first) {
    const int k = threadIdx.x;
    if (k >= b.n) return;
    const ITEM i = b.item[k];
    int t = *i.step;
    float factor = a.grad_scale;
    bool skip = false;
    if (a.clip) {                                            // [norm, factor] of semseg_grad_norm
        skip = !(fabsf(a.clip[0]) <= 3.402823466e38f);
        factor *= a.clip[1];
    }
    if (!skip) *i.step = ++t;
    ENTRY e;
    e.p = i.p; e.g = i.g; e.c = i.c;
    put_states(e, i);
    e.numel = i.numel;
    e.gtype = i.gtype; e.ctype = i.ctype; e.vec = i.vec; e.pad = 0;
    e.coef = adam_coef((double)a.lr[0], a.log_b1, a.log_b2, (double)i.wd, t, factor, a.seed, (uint32_t)(b.base + k));
    if (skip) e.coef.root = 0.f;
    table[b.base + k] = e;
    first[b.base + k] = i.first;
}

static bool hyper_ok(double beta1, double beta2, double eps) {
    return beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0 && eps <= 3.402823466e38;
}
static AdamHyper hyper_of(double beta1, double beta2, double eps) {
    AdamHyper h;
    h.b1 = (float)beta1; h.c1 = (float)(1.0 - beta1); h.b2 = (float)beta2; h.c2 = (float)(1.0 - beta2); h.eps = (float)eps;
    return h;
}

// ---------------------------------------------------------------- states in 32 bits -------------------------------------------
// One read and one write of everything, four 16-byte loads of each array under way per thread.  HBM-bound: 62 M elements in 168 tensors,
// f32 gradients, 327 us = 5.3 TB/s; 112 M elements in 24 tensors, bf16 gradients and copies, 588 us = 5.3 TB/s (a large copy on the same
// card: 4.9 TB/s).  Roots and divisions are the correctly rounded ones: about 50 instructions an element, a quarter of the time.
__global__ __launch_bounds__(256) void adamw_kernel(const AdamEntry* __restrict__ table, const uint32_t* __restrict__ first, int n,
                                                    AdamHyper h) {
    const int k = tensor_of(first, n, blockIdx.x);
    const AdamEntry t = table[k];
    const AdamCoef c = t.coef;
    if (c.root == 0.f) return;
    const int64_t start = (int64_t)(blockIdx.x - first[k]) * ADAM_CHUNK;
    const int tid = threadIdx.x;
    if (t.vec && start + ADAM_CHUNK <= t.numel) {
        const int64_t q0 = (start >> 2) + tid;
        f32x4* p4 = reinterpret_cast<f32x4*>(t.p);
        f32x4* m4 = reinterpret_cast<f32x4*>(t.m);
        f32x4* v4 = reinterpret_cast<f32x4*>(t.v);
        f32x4 p[ADAM_QUADS], g[ADAM_QUADS], m[ADAM_QUADS], v[ADAM_QUADS];
#pragma unroll
        for (int u = 0; u < ADAM_QUADS; ++u) {
            g[u] = load_quad(t.g, t.gtype, q0 + u * 256);
            m[u] = m4[q0 + u * 256];
            v[u] = v4[q0 + u * 256];
            p[u] = p4[q0 + u * 256];
        }
#pragma unroll
        for (int u = 0; u < ADAM_QUADS; ++u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float pj = p[u][j], mj = m[u][j], vj = v[u][j];
                adam_update32(pj, g[u][j], mj, vj, c, h);
                p[u][j] = pj; m[u][j] = mj; v[u][j] = vj;
            }
            m4[q0 + u * 256] = m[u];
            v4[q0 + u * 256] = v[u];
            p4[q0 + u * 256] = p[u];
            if (t.c) store_quad(t.c, t.ctype, q0 + u * 256, p[u]);
        }
        return;
    }
    // the last chunk of a tensor, and tensors that start at an odd address: loads that would pass the end read the last place again, so
    // that all of a thread's loads still leave together, and are not stored (one load at a time took 38 us for the 115 small tensors of a
    // ResNet50)
    const int left = (int)min(t.numel - start, (int64_t)ADAM_CHUNK);
    const int quads = t.vec ? left >> 2 : 0;
    if (quads) {
        f32x4* p4 = reinterpret_cast<f32x4*>(t.p) + (start >> 2);
        f32x4* m4 = reinterpret_cast<f32x4*>(t.m) + (start >> 2);
        f32x4* v4 = reinterpret_cast<f32x4*>(t.v) + (start >> 2);
        f32x4 p[ADAM_QUADS], g[ADAM_QUADS], m[ADAM_QUADS], v[ADAM_QUADS];
#pragma unroll
        for (int u = 0; u < ADAM_QUADS; ++u) {
            const int q = min(tid + u * 256, quads - 1);
            g[u] = load_quad(t.g, t.gtype, (start >> 2) + q);
            m[u] = m4[q];
            v[u] = v4[q];
            p[u] = p4[q];
        }
#pragma unroll
        for (int u = 0; u < ADAM_QUADS; ++u) {
            const int q = tid + u * 256;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float pj = p[u][j], mj = m[u][j], vj = v[u][j];
                adam_update32(pj, g[u][j], mj, vj, c, h);
                p[u][j] = pj; m[u][j] = mj; v[u][j] = vj;
            }
            if (q < quads) {
                m4[q] = m[u];
                v4[q] = v[u];
                p4[q] = p[u];
                if (t.c) store_quad(t.c, t.ctype, (start >> 2) + q, p[u]);
            }
        }
    }
    for (int base = quads * 4; base < left; base += 4 * 256) {
        float p[4], g[4], m[4], v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = start + min(base + tid + u * 256, left - 1);
            p[u] = t.p[i]; m[u] = t.m[i]; v[u] = t.v[i]; g[u] = load_one(t.g, t.gtype, i);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = start + base + tid + u * 256;
            adam_update32(p[u], g[u], m[u], v[u], c, h);
            if (base + tid + u * 256 < left) {
                t.m[i] = m[u];
                t.v[i] = v[u];
                t.p[i] = p[u];
                if (t.c) store_one(t.c, t.ctype, i, p[u]);
            }
        }
    }
}

static AdamItem item_of(const semseg_adamw_tensor& t) {
    AdamItem i{};
    i.p = (float*)t.param; i.g = t.grad; i.c = t.copy; i.m = (float*)t.exp_avg; i.v = (float*)t.exp_avg_sq; i.step = t.step;
    i.vec = aligned16(t.param) && aligned16(t.exp_avg) && aligned16(t.exp_avg_sq);
    return i;
}
static Adam8Item item_of(const semseg_adamw8_tensor& t) {
    Adam8Item i{};
    i.p = (float*)t.param; i.g = t.grad; i.c = t.copy; i.step = t.step;
    i.m = (uint8_t*)t.m_codes; i.ms = (float*)t.m_scales; i.r = (uint8_t*)t.r_codes; i.rs = (float*)t.r_scales;
    i.vec = aligned16(t.param) && aligned_to(t.m_codes, 4) && aligned_to(t.r_codes, 4);
    return i;
}
static bool states_ok(const semseg_adamw_tensor& t) { return t.exp_avg && t.exp_avg_sq; }
static bool states_ok(const semseg_adamw8_tensor& t) { return t.m_codes && t.m_scales && t.r_codes && t.r_scales; }

extern "C" size_t semseg_adamw_workspace_bytes(int n) {
    static_assert(sizeof(Adam8Entry) >= sizeof(AdamEntry) && sizeof(Adam8Entry) % 8 == 0, "one size for both steps");
    return n > 0 ? (size_t)n * (sizeof(Adam8Entry) + sizeof(uint32_t)) : 0;
}

// the steps' common host side: checks, the small kernel per batch of tensors, one launch of `kernel` per ADAM_MAX_TENSORS tensors
template <class ITEM, class ENTRY, class TENSOR, class KERNEL>
static int adam_step(const TENSOR* tensors, int n, const float* lr, double beta1, double beta2, double eps, float grad_scale, const float* clip,
                     uint32_t seed, int chunk, KERNEL kernel, void* workspace, size_t workspace_bytes, hipStream_t st) {
    typedef BeginBatch<ITEM, 3800 / (int)sizeof(ITEM)> Batch;
    typedef BeginBatch<ITEM, 8> SmallBatch;                  // few tensors: 0.7 KB of arguments instead of 4, 0.2 us of a call's 5.2 to 8.5
    static_assert(sizeof(Batch) + sizeof(BeginArgs) <= 4000 && Batch::MAX <= 64, "kernel arguments");
    if (n < 0 || (n && (!tensors || !lr)) || !hyper_ok(beta1, beta2, eps)) return SEMSEG_EINVAL;
    const int64_t most = (int64_t)1 << 30;                   // blocks of a launch
    for (int i = 0; i < n; ++i) {
        const TENSOR& t = tensors[i];
        if (!t.param || !t.grad || !states_ok(t) || !t.step || t.numel <= 0 || !type_ok(t.grad_type) ||
            (t.copy && (!type_ok(t.copy_type) || t.copy_type == SEMSEG_TYPE_F32)) || (t.numel + chunk - 1) / chunk > most)
            return SEMSEG_EINVAL;
    }
    if (n == 0) return 0;
    if (!workspace || workspace_bytes < semseg_adamw_workspace_bytes(n) || !aligned16(workspace)) return SEMSEG_EWORKSPACE;
    ENTRY* table = (ENTRY*)workspace;
    uint32_t* first = (uint32_t*)((char*)workspace + (size_t)n * sizeof(ENTRY));
    const AdamHyper h = hyper_of(beta1, beta2, eps);
    const BeginArgs a{lr, clip, log(beta1), log(beta2), grad_scale, seed};         // beta 0: -infinity, 1 - 0^t = 1
    for (int i = 0; i < n;) {
        const int start = i;
        uint32_t chunks = 0;
        bool room = true;
        while (room && i < n && i - start < ADAM_MAX_TENSORS) {
            Batch b;
            b.n = 0;
            b.base = i;
            for (; i < n && i - start < ADAM_MAX_TENSORS && b.n < Batch::MAX; ++i) {
                const TENSOR& t = tensors[i];
                const int64_t c = (t.numel + chunk - 1) / chunk;
                room = chunks + c <= most;
                if (!room) break;
                ITEM e = item_of(t);
                e.numel = t.numel;
                e.wd = t.weight_decay;
                e.first = chunks;
                e.gtype = (uint8_t)t.grad_type; e.ctype = (uint8_t)t.copy_type;
                e.vec = e.vec && aligned_to(t.grad, 4 * type_bytes(t.grad_type)) && (!t.copy || aligned_to(t.copy, 8));
                b.item[b.n++] = e;
                chunks += (uint32_t)c;
            }
            if (b.n == 0) break;
            if (b.n <= SmallBatch::MAX) {
                SmallBatch few;
                few.n = b.n;
                few.base = b.base;
                for (int k = 0; k < b.n; ++k) few.item[k] = b.item[k];
                auto begin = adamw_begin_kernel<ITEM, ENTRY, SmallBatch::MAX>;
                hipLaunchKernelGGL(begin, dim3(1), dim3(64), 0, st, few, a, table, first);
            } else {
                auto begin = adamw_begin_kernel<ITEM, ENTRY, Batch::MAX>;
                hipLaunchKernelGGL(begin, dim3(1), dim3(64), 0, st, b, a, table, first);
            }
            SEMSEG_LAUNCH_CHECK();
        }
        hipLaunchKernelGGL(kernel, dim3(chunks), dim3(256), 0, st, (const ENTRY*)(table + start), (const uint32_t*)(first + start), i - start, h);
        SEMSEG_LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int semseg_adamw_step(const semseg_adamw_tensor* tensors_host, int n, const float* lr, double beta1, double beta2, double eps,
                                 float grad_scale, const float* clip, void* workspace, size_t workspace_bytes, void* stream) {
    return adam_step<AdamItem, AdamEntry>(tensors_host, n, lr, beta1, beta2, eps, grad_scale, clip, 0u, ADAM_CHUNK, adamw_kernel, workspace,
                                          workspace_bytes, (hipStream_t)stream);
}

// ---------------------------------------------------------------- states in 8 bits --------------------------------------------
// A wave owns a block of 256 elements (one scale): 4 elements a lane, the block's maxima of |m| and r across the lanes, so the states are
// read and written once and never leave the registers in between.  62 M elements in 168 tensors, f32 gradients: 186 us = 5.3 TB/s of 16
// bytes an element; 112 M elements in 24 tensors, bf16 gradients and copies: 343 us = 5.2 TB/s (375 us where such passes follow each other
// without a gap).  With correctly rounded divisions, maxima by shuffles through LDS and codes rounded by bit operations it was bound by
// instructions: 386 us; now it has 90 vector instructions an element.
constexpr int ADAM8_PER_WAVE = 4;                                     // blocks of a wave, their loads in flight together
constexpr int ADAM8_CHUNK = 4 * ADAM8_PER_WAVE * ADAM8_BLOCK;         // elements of a thread block

// maximum over the wave, as a scalar.  Within a row of 16 lanes by lane permutations of the instruction itself, then across the rows:
// 6 instructions and a read of lane 63 (shuffles through LDS take 18 and their waits).  All lanes must be active.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#define SEMSEG_DPP_MAX(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, ctrl, rows, 0xf, false))
    SEMSEG_DPP_MAX(0xB1, 0xf);        // neighbours
    SEMSEG_DPP_MAX(0x4E, 0xf);        // pairs
    SEMSEG_DPP_MAX(0x141, 0xf);       // mirrored halves of a row
    SEMSEG_DPP_MAX(0x140, 0xf);       // mirrored rows
    SEMSEG_DPP_MAX(0x142, 0xa);       // lane 15 of a row to the next: rows 1 and 3
    SEMSEG_DPP_MAX(0x143, 0xc);       // lane 31 to rows 2 and 3
#undef SEMSEG_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// the e4m3 code of byte J in a word of four
template <int J>
__device__ __forceinline__ float value_of(uint32_t w) { return __builtin_amdgcn_cvt_f32_fp8((int)w, J); }

// m and r of one block after the update (4 elements a lane, elements that do not exist are 0) -> scales and words of codes
__device__ __forceinline__ void adam8_block(const float m[4], const float r[4], const uint32_t at[4], const AdamCoef& c, float& ms, float& rs,
                                            uint32_t& mc, uint32_t& rc) {
    uint32_t tm = 0, tr = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        tm = max(tm, adam_bits(m[j]) & 0x7fffffffu);
        tr = max(tr, adam_bits(r[j]) & 0x7fffffffu);
    }
    ms = adam8_scale(wave_max_u32(tm));
    rs = adam8_scale(wave_max_u32(tr));
    const float im = adam8_inverse(ms), ir = adam8_inverse(rs);
    int wm = 0, wr = 0;
#define SEMSEG_ADAM8_CODE(j)                                                                                     \
    {                                                                                                            \
        const uint32_t bits = adam_mix(at[j] + c.base);                                                          \
        wm = __builtin_amdgcn_cvt_sr_fp8_f32(adam8_scaled_m(m[j], im), bits << 16, wm, j);                       \
        wr = __builtin_amdgcn_cvt_sr_fp8_f32(adam8_scaled_r(r[j], ir), bits & 0xffff0000u, wr, j);               \
    }
    SEMSEG_ADAM8_CODE(0)
    SEMSEG_ADAM8_CODE(1)
    SEMSEG_ADAM8_CODE(2)
    SEMSEG_ADAM8_CODE(3)
#undef SEMSEG_ADAM8_CODE
    mc = (uint32_t)wm;
    rc = (uint32_t)wr;
}

__global__ __launch_bounds__(256) void adamw8_kernel(const Adam8Entry* __restrict__ table, const uint32_t* __restrict__ first, int n,
                                                     AdamHyper h) {
    const int k = tensor_of(first, n, blockIdx.x);
    const Adam8Entry t = table[k];
    const AdamCoef c = t.coef;
    if (c.root == 0.f) return;
    const int lane = threadIdx.x & 63;
    const int64_t start = (int64_t)(blockIdx.x - first[k]) * ADAM8_CHUNK + (threadIdx.x >> 6) * (ADAM8_PER_WAVE * ADAM8_BLOCK);
    if (start >= t.numel) return;                            // the same for the whole wave, as everything about blocks here
    const int full = t.vec ? (int)min((t.numel - start) >> 8, (int64_t)ADAM8_PER_WAVE) : 0;
    if (full) {
        const int64_t q0 = (start >> 2) + lane, s0 = start >> 8;
        f32x4* p4 = reinterpret_cast<f32x4*>(t.p);
        uint32_t* m4 = reinterpret_cast<uint32_t*>(t.m);
        uint32_t* r4 = reinterpret_cast<uint32_t*>(t.r);
        f32x4 p[ADAM8_PER_WAVE], g[ADAM8_PER_WAVE];
        uint32_t mc[ADAM8_PER_WAVE], rc[ADAM8_PER_WAVE];
        float ms[ADAM8_PER_WAVE], rs[ADAM8_PER_WAVE];
#pragma unroll
        for (int u = 0; u < ADAM8_PER_WAVE; ++u) {
            const int b = min(u, full - 1);                  // a block behind the last whole one is the last one again, not stored
            g[u] = load_quad(t.g, t.gtype, q0 + b * 64);
            p[u] = p4[q0 + b * 64];
            mc[u] = m4[q0 + b * 64];
            rc[u] = r4[q0 + b * 64];
            ms[u] = t.ms[s0 + b];
            rs[u] = t.rs[s0 + b];
        }
#pragma unroll
        for (int u = 0; u < ADAM8_PER_WAVE; ++u) {
            if (u >= full) break;
            float m[4], r[4];
            uint32_t at[4];
            m[0] = value_of<0>(mc[u]); m[1] = value_of<1>(mc[u]); m[2] = value_of<2>(mc[u]); m[3] = value_of<3>(mc[u]);
            r[0] = value_of<0>(rc[u]); r[1] = value_of<1>(rc[u]); r[2] = value_of<2>(rc[u]); r[3] = value_of<3>(rc[u]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                at[j] = (uint32_t)((q0 + u * 64) * 4 + j);
                float pj = p[u][j];
                m[j] *= ms[u];
                r[j] *= rs[u];
                adam_update8(pj, g[u][j], m[j], r[j], c, h);
                p[u][j] = pj;
            }
            float msn, rsn;
            uint32_t mn, rn;
            adam8_block(m, r, at, c, msn, rsn, mn, rn);
            p4[q0 + u * 64] = p[u];
            m4[q0 + u * 64] = mn;
            r4[q0 + u * 64] = rn;
            if (lane == 0) {
                t.ms[s0 + u] = msn;
                t.rs[s0 + u] = rsn;
            }
            if (t.c) store_quad(t.c, t.ctype, q0 + u * 64, p[u]);
        }
    }
    // the last block of a tensor, and tensors that start at an odd address: element lane + 64 j of the block
    for (int u = full; u < ADAM8_PER_WAVE; ++u) {
        const int64_t s = start + u * ADAM8_BLOCK;
        if (s >= t.numel) return;                            // the same for the whole wave
        const float ms = t.ms[s >> 8], rs = t.rs[s >> 8];
        float m[4], r[4], p[4];
        uint32_t at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = s + lane + 64 * j;
            at[j] = (uint32_t)i;
            m[j] = r[j] = p[j] = 0.f;
            if (i < t.numel) {
                p[j] = t.p[i];
                m[j] = value_of<0>(t.m[i]) * ms;
                r[j] = value_of<0>(t.r[i]) * rs;
                adam_update8(p[j], load_one(t.g, t.gtype, i), m[j], r[j], c, h);
            }
        }
        float msn, rsn;
        uint32_t mn, rn;
        adam8_block(m, r, at, c, msn, rsn, mn, rn);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = s + lane + 64 * j;
            if (i < t.numel) {
                t.p[i] = p[j];
                t.m[i] = (uint8_t)(mn >> (8 * j));
                t.r[i] = (uint8_t)(rn >> (8 * j));
                if (t.c) store_one(t.c, t.ctype, i, p[j]);
            }
        }
        if (lane == 0) {
            t.ms[s >> 8] = msn;
            t.rs[s >> 8] = rsn;
        }
    }
}

extern "C" int semseg_adamw8_step(const semseg_adamw8_tensor* tensors_host, int n, const float* lr, double beta1, double beta2, double eps,
                                  float grad_scale, const float* clip, uint32_t seed, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    if (eps != 0.0 && !(eps >= 0x1p-126 && eps <= 0x1p126)) return SEMSEG_EINVAL;          // the hardware's reciprocal of it would be 0 or infinite
    return adam_step<Adam8Item, Adam8Entry>(tensors_host, n, lr, beta1, beta2, eps, grad_scale, clip, seed, ADAM8_CHUNK, adamw8_kernel,
                                            workspace, workspace_bytes, (hipStream_t)stream);
}

// ---------------------------------------------------------------- global norm -------------------------------------------------
// Squares are summed in 64 bits (an f32 square leaves the range at 2e19 and below 1e-23), one partial sum per chunk in a fixed order,
// then one block sums the partials: the same bits every time.  62 M f32 elements 44 us = 5.6 TB/s, 112 M bf16 39 us = 5.8 TB/s, and 4.7
// us of the second kernel.
constexpr int NORM_MAX_TENSORS = 196;
constexpr int NORM_CHUNK = 16384;
struct NormBatch {
    const void* g[NORM_MAX_TENSORS];
    uint64_t size[NORM_MAX_TENSORS];        // elements, type and alignment: numel * 8 + type * 2 + vec
    uint32_t first[NORM_MAX_TENSORS];
    int n;
};
static_assert(sizeof(NormBatch) <= 4000, "kernel arguments");

__device__ __forceinline__ void add_square(double& s, float x) { const double d = (double)x; s = fma(d, d, s); }

__device__ __forceinline__ void add_squares(double& s, u32x4 v, int type) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t w = v[j];            // a word of its own: bit_cast of the vector's element v[j] itself reads element 0 (hipcc 7.2)
        if (type == SEMSEG_TYPE_F32) {
            add_square(s, adam_float(w));
        } else if (type == SEMSEG_TYPE_BF16) {
            add_square(s, adam_float(w << 16));
            add_square(s, adam_float(w & 0xffff0000u));
        } else {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const f16x2 x = __builtin_bit_cast(f16x2, w);
            add_square(s, (float)x[0]);
            add_square(s, (float)x[1]);
        }
    }
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const NormBatch b, double* __restrict__ partial) {
    __shared__ double sum[4];
    const int k = tensor_of(b.first, b.n, blockIdx.x);
    const uint64_t size = b.size[k];
    const struct { const void* g; int64_t numel; int type, vec; } t = {b.g[k], (int64_t)(size >> 3), (int)(size >> 1) & 3, (int)size & 1};
    const int64_t start = (int64_t)(blockIdx.x - b.first[k]) * NORM_CHUNK;
    const int64_t end = min(t.numel, start + NORM_CHUNK);
    double s = 0.0;
    if (t.vec) {
        // 16-byte loads, 8 of a thread in flight (f32: 4 elements each, 16 bits: 8); past the end the last place again, not added
        const int per = t.type == SEMSEG_TYPE_F32 ? 4 : 8;
        const int vecs = (int)(end - start) / per;
        const u32x4* g4 = reinterpret_cast<const u32x4*>(t.g) + start / per;
        for (int base = 0; base < vecs; base += 8 * 256) {
            u32x4 g[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = g4[min(base + j * 256 + (int)threadIdx.x, vecs - 1)];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (base + j * 256 + (int)threadIdx.x >= vecs) g[j] = u32x4{0u, 0u, 0u, 0u};
                add_squares(s, g[j], t.type);
            }
        }
        const int64_t i = start + (int64_t)vecs * per + threadIdx.x;
        if (i < end) add_square(s, load_one(t.g, t.type, i));           // fewer than 8 are left
    } else {
        for (int64_t i = start + threadIdx.x; i < end; i += 256) add_square(s, load_one(t.g, t.type, i));
    }
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double* __restrict__ partial, int64_t n, float grad_scale, float max_norm,
                                                                float* __restrict__ out) {
    __shared__ double sum[16];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += partial[i];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int i = 0; i < 16; ++i) total += sum[i];
        const double norm = sqrt(total) * fabs((double)grad_scale);
        const float f = (float)norm;
        float factor = 1.f;
        if (max_norm >= 0.f) factor = (float)fmin(1.0, (double)max_norm / (norm + 1e-6));
        out[0] = f;
        out[1] = fabsf(f) <= 3.402823466e38f ? factor : 0.f;
    }
}

static int64_t norm_chunks(int64_t numel) { return (numel + NORM_CHUNK - 1) / NORM_CHUNK; }

extern "C" size_t semseg_grad_norm_workspace_bytes(const semseg_grad_tensor* tensors_host, int n) {
    int64_t chunks = 0;
    for (int i = 0; tensors_host && i < n; ++i) chunks += tensors_host[i].numel > 0 ? norm_chunks(tensors_host[i].numel) : 0;
    return (size_t)(chunks ? chunks : 1) * sizeof(double);
}

extern "C" int semseg_grad_norm(const semseg_grad_tensor* tensors_host, int n, float grad_scale, float max_norm, float* out, void* workspace,
                                size_t workspace_bytes, void* stream) {
    if (n < 0 || (n && !tensors_host) || !out) return SEMSEG_EINVAL;
    for (int i = 0; i < n; ++i) {
        const semseg_grad_tensor& t = tensors_host[i];
        if (!t.grad || t.numel <= 0 || !type_ok(t.grad_type) || norm_chunks(t.numel) > (int64_t)1 << 30) return SEMSEG_EINVAL;
    }
    if (!workspace || workspace_bytes < semseg_grad_norm_workspace_bytes(tensors_host, n)) return SEMSEG_EWORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    double* partial = (double*)workspace;
    int64_t done = 0;
    for (int i = 0; i < n;) {
        NormBatch b;
        b.n = 0;
        uint32_t chunks = 0;
        for (; i < n && b.n < NORM_MAX_TENSORS; ++i) {
            const semseg_grad_tensor& t = tensors_host[i];
            const int64_t c = norm_chunks(t.numel);
            if (chunks + c > (int64_t)1 << 30) break;
            b.g[b.n] = t.grad;
            b.size[b.n] = (uint64_t)t.numel << 3 | (uint64_t)t.grad_type << 1 | (aligned16(t.grad) ? 1u : 0u);
            b.first[b.n++] = chunks;
            chunks += (uint32_t)c;
        }
        hipLaunchKernelGGL(grad_norm_kernel, dim3(chunks), dim3(256), 0, st, b, partial + done);
        SEMSEG_LAUNCH_CHECK();
        done += chunks;
    }
    hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(1024), 0, st, (const double*)partial, done, grad_scale, max_norm, out);
    SEMSEG_LAUNCH_CHECK();
    return 0;
}
