// TEST INFRASTRUCTURE: host build of the per-element code of csrc/adamw.hip (adamw_math.h) behind the same C ABI, with the same blocks
// of the 8-bit states, so that the AdamW steps and the Python entry points above them can be checked against float64 without a GPU
// (tests/test_finetune_cpu.py; the GPU's results are held to the same bounds, tests/test_gpu_finetune.py).  Never shipped.
#include <stddef.h>
#include "semseg_hip.h"
#include "adamw_math.h"

static float from_bf16(uint16_t h) { return adam_float((uint32_t)h << 16); }
static uint16_t to_bf16(float x) {
    uint32_t u = adam_bits(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
static float from_f16(uint16_t h) {
    const int e = (h >> 10) & 31, f = h & 1023;
    const float v = e == 31 ? (f ? NAN : INFINITY) : e ? ldexpf(1024.f + f, e - 25) : ldexpf((float)f, -24);
    return (h & 0x8000) ? -v : v;
}
static uint16_t to_f16(float x) {
    const uint16_t sign = (uint16_t)((adam_bits(x) >> 16) & 0x8000);
    const float a = fabsf(x);
    if (a != a) return sign | 0x7e00;
    if (a >= 65520.f) return sign | 0x7c00;
    if (a < 6.103515625e-05f) return sign | (uint16_t)nearbyintf(ldexpf(a, 24));      // subnormal (or rounds up to the first normal)
    int e;
    const float f = nearbyintf(ldexpf(frexpf(a, &e), 11));                            // [1024, 2048], to nearest even
    return sign | (uint16_t)(((e + 14) << 10) + ((int)f - 1024));
}
static float load(const void* g, int type, int64_t i) {
    if (type == SEMSEG_TYPE_F32) return ((const float*)g)[i];
    if (type == SEMSEG_TYPE_BF16) return from_bf16(((const uint16_t*)g)[i]);
    return from_f16(((const uint16_t*)g)[i]);
}
static void store(void* c, int type, int64_t i, float x) {
    if (type == SEMSEG_TYPE_BF16) ((uint16_t*)c)[i] = to_bf16(x);
    else ((uint16_t*)c)[i] = to_f16(x);
}
// e4m3: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f is NaN
static float decode(uint8_t c) {
    const int e = (c >> 3) & 15, f = c & 7;
    float v = e ? ldexpf(8.f + f, e - 10) : ldexpf((float)f, -9);
    if ((c & 0x7f) == 0x7f) v = NAN;
    return (c & 0x80) ? -v : v;
}
static uint8_t encode(float x) {                     // of values that e4m3 holds exactly
    uint8_t sign = (adam_bits(x) >> 31) ? 0x80 : 0;
    x = fabsf(x);
    if (x == 0.f) return sign;
    if (x < 0.015625f) return sign | (uint8_t)(x * 512.f);
    int e;
    const float f = frexpf(x, &e);                   // [0.5, 1)
    return sign | (uint8_t)(((e + 6) << 3) | ((int)(f * 16.f) - 8));
}

static AdamHyper hyper(double b1, double b2, double eps) {
    AdamHyper h;
    h.b1 = (float)b1; h.c1 = (float)(1.0 - b1); h.b2 = (float)b2; h.c2 = (float)(1.0 - b2); h.eps = (float)eps;
    return h;
}
static bool begin(int* step, float wd, const float* lr, double b1, double b2, float scale, const float* clip, uint32_t seed, int ordinal,
                  AdamCoef& c) {
    if (clip) {
        if (!(fabsf(clip[0]) <= 3.402823466e38f)) return false;
        scale *= clip[1];
    }
    *step += 1;
    c = adam_coef((double)lr[0], log(b1), log(b2), (double)wd, *step, scale, seed, (uint32_t)ordinal);
    return true;
}

extern "C" size_t semseg_adamw_workspace_bytes(int n) { return n > 0 ? (size_t)n * sizeof(AdamCoef) : 0; }

extern "C" int semseg_adamw_step(const semseg_adamw_tensor* t, int n, const float* lr, double b1, double b2, double eps, float scale,
                                 const float* clip, void*, size_t, void*) {
    const AdamHyper h = hyper(b1, b2, eps);
    for (int i = 0; i < n; ++i) {
        AdamCoef c;
        if (!begin(t[i].step, t[i].weight_decay, lr, b1, b2, scale, clip, 0, i, c)) continue;
        float *p = (float*)t[i].param, *m = (float*)t[i].exp_avg, *v = (float*)t[i].exp_avg_sq;
        for (int64_t j = 0; j < t[i].numel; ++j) {
            adam_update32(p[j], load(t[i].grad, t[i].grad_type, j), m[j], v[j], c, h);
            if (t[i].copy) store(t[i].copy, t[i].copy_type, j, p[j]);
        }
    }
    return 0;
}

extern "C" int semseg_adamw8_step(const semseg_adamw8_tensor* t, int n, const float* lr, double b1, double b2, double eps, float scale,
                                  const float* clip, uint32_t seed, void*, size_t, void*) {
    const AdamHyper h = hyper(b1, b2, eps);
    for (int i = 0; i < n; ++i) {
        AdamCoef c;
        if (!begin(t[i].step, t[i].weight_decay, lr, b1, b2, scale, clip, seed, i, c)) continue;
        float* p = (float*)t[i].param;
        uint8_t *mc = (uint8_t*)t[i].m_codes, *rc = (uint8_t*)t[i].r_codes;
        for (int64_t s = 0; s < t[i].numel; s += ADAM8_BLOCK) {
            const int64_t end = s + ADAM8_BLOCK < t[i].numel ? s + ADAM8_BLOCK : t[i].numel;
            float &ms = ((float*)t[i].m_scales)[s / ADAM8_BLOCK], &rs = ((float*)t[i].r_scales)[s / ADAM8_BLOCK];
            float m[ADAM8_BLOCK], r[ADAM8_BLOCK];
            uint32_t tm = 0, tr = 0;
            for (int64_t j = s; j < end; ++j) {
                float &mj = m[j - s], &rj = r[j - s];
                mj = decode(mc[j]) * ms;
                rj = decode(rc[j]) * rs;
                adam_update8(p[j], load(t[i].grad, t[i].grad_type, j), mj, rj, c, h);
                if (t[i].copy) store(t[i].copy, t[i].copy_type, j, p[j]);
                const uint32_t um = adam_bits(fabsf(mj)), ur = adam_bits(fabsf(rj));
                tm = um > tm ? um : tm;
                tr = ur > tr ? ur : tr;
            }
            ms = adam8_scale(tm);
            rs = adam8_scale(tr);
            const float im = adam8_inverse(ms), ir = adam8_inverse(rs);
            for (int64_t j = s; j < end; ++j) {
                const uint32_t bits = adam_mix((uint32_t)j + c.base);
                mc[j] = encode(adam8_round(adam8_scaled_m(m[j - s], im), bits & 0xffffu));
                rc[j] = encode(adam8_round(adam8_scaled_r(r[j - s], ir), bits >> 16));
            }
        }
    }
    return 0;
}

extern "C" size_t semseg_grad_norm_workspace_bytes(const semseg_grad_tensor*, int) { return 8; }
extern "C" int semseg_grad_norm(const semseg_grad_tensor* t, int n, float scale, float max_norm, float* out, void*, size_t, void*) {
    double s = 0.0;
    for (int i = 0; i < n; ++i)
        for (int64_t j = 0; j < t[i].numel; ++j) {
            const double x = (double)load(t[i].grad, t[i].grad_type, j);
            s += x * x;
        }
    const double norm = sqrt(s) * fabs((double)scale);
    out[0] = (float)norm;
    out[1] = fabsf(out[0]) <= 3.402823466e38f ? (max_norm >= 0.f ? (float)fmin(1.0, (double)max_norm / (norm + 1e-6)) : 1.f) : 0.f;
    return 0;
}
