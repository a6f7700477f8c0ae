// One AdamW step over many tensors in one launch, with the running means held in 32 or in 8 bits.
//
//   m' = b1 m + (1 - b1) g      v' = b2 v + (1 - b2) g^2
//   w' = w - lr wd w - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Nothing is used twice, so the step is bound by memory: 28 bytes per parameter with float32 weights and states, 16 with
// 8-bit states (and 8 bytes of scales for every 256 parameters).
#pragma once
#include "../../include/az_engine.h"
#include "az_vec.h"

#define AZ_ADAMW_THREADS 256
#define AZ_ADAMW_BLOCK AZ_STATE_BLOCK    // elements that share a scale: one wave's four elements per lane
#define AZ_ADAMW_TENSORS 56   // per launch: the table travels in the kernel's arguments, which stay under 4 KB

// The tensors of one launch.  The table goes by value: no copy to the device that would have to outlive the call, nothing
// that a later call could overwrite while this one is still queued.
struct AdamwTable {
    void *param[AZ_ADAMW_TENSORS];
    const void *grad[AZ_ADAMW_TENSORS];
    void *m[AZ_ADAMW_TENSORS], *v[AZ_ADAMW_TENSORS];
    float *m_scale[AZ_ADAMW_TENSORS], *v_scale[AZ_ADAMW_TENSORS];
    int64_t n[AZ_ADAMW_TENSORS];
    uint32_t last[AZ_ADAMW_TENSORS];   // workgroups of the launch up to and with this tensor's; 0xffffffff past the last one
};

struct AdamwScalars {
    double beta1, beta2, one_minus_beta1, one_minus_beta2;
    float decay, step_size, inv_sqrt_c2, eps;   // lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

// Which tensor a workgroup works on: every lane compares one entry of the table (one load, where a search would be a chain).
__device__ __forceinline__ int adamw_tensor(const AdamwTable &a, uint32_t block)
{
    static_assert(AZ_ADAMW_TENSORS <= 64, "one lane per tensor");
    const int lane = threadIdx.x & 63;
    const uint32_t last = lane < AZ_ADAMW_TENSORS ? a.last[lane] : 0xffffffffu;
    return __popcll(__ballot(last <= block));
}

__device__ __forceinline__ float adamw_weight(float w, float m, float v, const AdamwScalars &k)
{
    return w - k.decay * w - k.step_size * (m / (sqrtf(v) * k.inv_sqrt_c2 + k.eps));
}

__device__ __forceinline__ void adamw_32(float &w, float g, float &m, float &v, const AdamwScalars &k)
{
    m = (float)k.beta1 * m + (float)k.one_minus_beta1 * g;
    v = (float)k.beta2 * v + (float)k.one_minus_beta2 * (g * g);
    w = adamw_weight(w, m, v, k);
}

// A workgroup takes TURNS * 1024 neighbouring elements of one tensor.
template <typename T, int TURNS> __global__ __launch_bounds__(AZ_ADAMW_THREADS) void k_adamw_32(AdamwTable a, AdamwScalars k)
{
    const int i = __builtin_amdgcn_readfirstlane(adamw_tensor(a, blockIdx.x));
    const int64_t first = (int64_t)(blockIdx.x - (i ? a.last[i - 1] : 0u)) * (TURNS * 4 * AZ_ADAMW_THREADS);
    const int64_t n = a.n[i];
    T *wp = static_cast<T *>(a.param[i]);
    const T *gp = static_cast<const T *>(a.grad[i]);
    float *mp = static_cast<float *>(a.m[i]), *vp = static_cast<float *>(a.v[i]);
    float4 w[TURNS], g[TURNS], m[TURNS], v[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
        const int64_t at = first + (u * AZ_ADAMW_THREADS + threadIdx.x) * 4;
        w[u] = load4(wp, at, n); g[u] = load4(gp, at, n); m[u] = load4(mp, at, n); v[u] = load4(vp, at, n);
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
        const int64_t at = first + (u * AZ_ADAMW_THREADS + threadIdx.x) * 4;
        adamw_32(w[u].x, g[u].x, m[u].x, v[u].x, k);
        adamw_32(w[u].y, g[u].y, m[u].y, v[u].y, k);
        adamw_32(w[u].z, g[u].z, m[u].z, v[u].z, k);
        adamw_32(w[u].w, g[u].w, m[u].w, v[u].w, k);
        store4(wp, at, n, w[u]); store4(mp, at, n, m[u]); store4(vp, at, n, v[u]);
    }
}

// ---- states in 8 bits -------------------------------------------------------------------------------------------------
// A block of 256 elements shares one float32 scale S, the largest magnitude in it (rounded to nearest):
//   m = S * sgn(c) * (c / 127)^2,  c int8       v = S * (c / 255)^4,  c uint8
// The update divides m by sqrt(v), so what counts is the relative step of m and of sqrt(v): the powers put the codes where
// small values are (m down to 1.6e-5 and sqrt(v) down to 1.5e-5 of the block's largest) and still step by 1.6 % and 0.8 % at
// the top.  A code is the nearest one in the domain in which codes are evenly spaced, c = round(127 sqrt(|m| / S)),
// c = round(255 (v / S)^(1/4)), and at least 1 where v > 0, so that no element is ever divided by eps alone because its
// v was rounded away.
// Means and codes are worked out in 64 bits: a value next to a border between two codes goes to the right side of it, and
// the multiplications cost less than the memory they wait for.  Every operation of the means rounds by itself, in the order in
// which the formulas are written (no fused multiply-add): b1 S + (1 - b1) g lies exactly between two float32 values in one
// block of a hundred, and the scale must not depend on how a compiler contracts the sum.  The border is found by comparing powers, not by taking roots:
// a float32 estimate is off by one at most, and (2c - 1)^2 S <= 254^2 |m| < (2c + 1)^2 S settles it.
// A block with an infinity or a NaN in it has a scale that is not finite and reads back as NaN as a whole.

__device__ __forceinline__ double dequantize_m(int c, double s) { return s * (double)(c * abs(c)) * (1.0 / 16129.0); }

__device__ __forceinline__ double dequantize_v(int c, double s)
{
    const double q = (double)(c * c);
    return s * (q * q) * (1.0 / 4228250625.0);   // 255^4
}

// s > 0 and finite, inv = 1 / s
__device__ __forceinline__ int quantize_m(double m, double s, double inv)
{
    const double a = fabs(m), t = a * 64516.0;   // 254^2
    const int c = (int)rintf(127.0f * __builtin_amdgcn_sqrtf((float)(a * inv)));
    const double lo = (double)((2 * c - 1) * abs(2 * c - 1)) * s, hi = (double)((2 * c + 1) * (2 * c + 1)) * s;
    const int r = min(c + (t >= hi ? 1 : 0) - (t < lo ? 1 : 0), 127);
    return m < 0.0 ? -r : r;
}

__device__ __forceinline__ int quantize_v(double v, double s, double inv)
{
    const double t = v * 67652010000.0;          // 510^4
    const int c = (int)rintf(255.0f * __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)(v * inv))));
    const double l = (double)((2 * c - 1) * abs(2 * c - 1)), h = (double)((2 * c + 1) * (2 * c + 1));
    const int r = min(c + (t >= h * h * s ? 1 : 0) - (t < l * fabs(l) * s ? 1 : 0), 255);
    return v > 0.0 ? max(r, 1) : r;
}

struct __attribute__((packed)) PackedWord { uint32_t v; };

// four codes as one word (any address); those past the end are 0 / are not written
__device__ __forceinline__ uint32_t load_codes(const uint8_t *p, int64_t i, int64_t n)
{
    if (i + 4 <= n) return reinterpret_cast<const PackedWord *>(p + i)->v;
    uint32_t w = 0;
    if (i < n) w = p[i];
    if (i + 1 < n) w |= (uint32_t)p[i + 1] << 8;
    if (i + 2 < n) w |= (uint32_t)p[i + 2] << 16;
    return w;
}

__device__ __forceinline__ void store_codes(uint8_t *p, int64_t i, int64_t n, uint32_t w)
{
    if (i + 4 <= n) { reinterpret_cast<PackedWord *>(p + i)->v = w; return; }
    if (i < n) p[i] = (uint8_t)w;
    if (i + 1 < n) p[i + 1] = (uint8_t)(w >> 8);
    if (i + 2 < n) p[i + 2] = (uint8_t)(w >> 16);
}

__device__ __forceinline__ uint32_t magnitude_bits(double x) { return __float_as_uint((float)x) & 0x7fffffffu; }

// A workgroup takes TURNS * 1024 neighbouring elements of one tensor, each of its waves a block of 256 at a time.
template <typename T, int TURNS> __global__ __launch_bounds__(AZ_ADAMW_THREADS) void k_adamw_8(AdamwTable a, AdamwScalars k)
{
    const int i = __builtin_amdgcn_readfirstlane(adamw_tensor(a, blockIdx.x));
    const int64_t first = (int64_t)(blockIdx.x - (i ? a.last[i - 1] : 0u)) * (TURNS * 4 * AZ_ADAMW_THREADS);
    const int64_t n = a.n[i];
    T *wp = static_cast<T *>(a.param[i]);
    const T *gp = static_cast<const T *>(a.grad[i]);
    uint8_t *mp = static_cast<uint8_t *>(a.m[i]), *vp = static_cast<uint8_t *>(a.v[i]);
    float *msp = a.m_scale[i], *vsp = a.v_scale[i];
    float4 w[TURNS], g[TURNS];
    uint32_t mc[TURNS], vc[TURNS];
    float ms[TURNS], vs[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
        const int64_t at = first + (u * AZ_ADAMW_THREADS + threadIdx.x) * 4;
        w[u] = load4(wp, at, n); g[u] = load4(gp, at, n);
        mc[u] = load_codes(mp, at, n); vc[u] = load_codes(vp, at, n);
        const int64_t block = (at - (threadIdx.x & 63) * 4) / AZ_ADAMW_BLOCK;
        const bool in = block * AZ_ADAMW_BLOCK < n;
        ms[u] = in ? msp[block] : 0.f; vs[u] = in ? vsp[block] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
        const int64_t at = first + (u * AZ_ADAMW_THREADS + threadIdx.x) * 4;
        float *we = reinterpret_cast<float *>(&w[u]);
        const float *ge = reinterpret_cast<const float *>(&g[u]);
        double m[4], v[4];
        uint32_t mb = 0, vb = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
#pragma clang fp contract(off)
            const double gd = (double)ge[e];
            m[e] = k.beta1 * dequantize_m((int8_t)(mc[u] >> (8 * e)), (double)ms[u]) + k.one_minus_beta1 * gd;
            v[e] = k.beta2 * dequantize_v((uint8_t)(vc[u] >> (8 * e)), (double)vs[u]) + k.one_minus_beta2 * (gd * gd);
            mb = max(mb, magnitude_bits(m[e]));
            vb = max(vb, magnitude_bits(v[e]));
            we[e] = adamw_weight(we[e], (float)m[e], (float)v[e], k);
        }
        // NaN has the largest magnitude bits of all, so the integer maximum keeps it
        mb = wave_umax(mb); vb = wave_umax(vb);
        uint32_t mw = 0, vw = 0;
        if (mb != 0 && mb < 0x7f800000u) {
            const double s = (double)__uint_as_float(mb), inv = 1.0 / s;
#pragma unroll
            for (int e = 0; e < 4; e++) mw |= (uint32_t)(uint8_t)quantize_m(m[e], s, inv) << (8 * e);
        }
        if (vb != 0 && vb < 0x7f800000u) {
            const double s = (double)__uint_as_float(vb), inv = 1.0 / s;
#pragma unroll
            for (int e = 0; e < 4; e++) vw |= (uint32_t)quantize_v(v[e], s, inv) << (8 * e);
        }
        store4(wp, at, n, w[u]);
        store_codes(mp, at, n, mw); store_codes(vp, at, n, vw);
        const int64_t start = at - (threadIdx.x & 63) * 4;
        if ((threadIdx.x & 63) == 0 && start < n) {
            msp[start / AZ_ADAMW_BLOCK] = __uint_as_float(mb);
            vsp[start / AZ_ADAMW_BLOCK] = __uint_as_float(vb);
        }
    }
}

// the values that codes stand for, rounded once to float32
template <bool SIGNED> __global__ __launch_bounds__(AZ_ADAMW_THREADS) void k_dequantize_state(const uint8_t *codes, const float *scales, int64_t n, float *out)
{
    const int64_t step = (int64_t)gridDim.x * AZ_ADAMW_THREADS * 4;
    for (int64_t at = ((int64_t)blockIdx.x * AZ_ADAMW_THREADS + threadIdx.x) * 4; at < n; at += step) {
        const uint32_t w = load_codes(codes, at, n);
        const double s = (double)scales[at / AZ_ADAMW_BLOCK];
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            f[e] = (float)(SIGNED ? dequantize_m((int8_t)(w >> (8 * e)), s) : dequantize_v((uint8_t)(w >> (8 * e)), s));
        store4(out, at, n, make_float4(f[0], f[1], f[2], f[3]));
    }
}
