// One AdamW step over many tensors in one launch, with the running means held in 32 or in 8 bits.
//
//   m' = b1 m + (1 - b1) g      v' = b2 v + (1 - b2) g^2
//   w' = w - lr wd w - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Nothing is used twice, so the step is bound by memory: 28 bytes per parameter with float32 weights and states, 16 with
// 8-bit states (and 16 bytes for the scales of every 256 parameters).  Measured, 24 M float32 parameters in one tensor: 112 us
// (6.0 TB/s) and, with 8-bit state, 62 us (6.2 TB/s); a copy of 1 GiB reaches 5.1 TB/s.
#pragma once
#include "../../include/az_engine.h"
#include "az_vec.h"

#define AZ_ADAMW_THREADS 256
#define AZ_ADAMW_BLOCK AZ_STATE_BLOCK    // elements that share a scale: one wave's four elements per lane
#define AZ_ADAMW_TENSORS 64   // per launch: one for each lane; the table travels in the kernel's arguments, under 4 KB

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
    bool tiny;                                  // the root of a subnormal v is not negligible beside eps
};
static_assert(sizeof(AdamwTable) + sizeof(AdamwScalars) <= 4096, "kernel arguments");

// Which tensor a workgroup works on: every lane compares one entry of the table (one load, where a search would be a chain).
__device__ __forceinline__ int adamw_tensor(const AdamwTable &a, uint32_t block)
{
    static_assert(AZ_ADAMW_TENSORS == 64, "one lane per tensor");
    return __popcll(__ballot(a.last[threadIdx.x & 63] <= block));
}

// Square root and reciprocal by the instructions that are right to one step of float32, a third of the work of the correctly
// rounded ones: their error is in the update, not in the weight.  They take no subnormal numbers: a v below 2^-126 counts as
// nothing beside eps, or, where eps is so small that it does not (k.tiny), is scaled.
__device__ __forceinline__ float adamw_root(float v, const AdamwScalars &k)
{
    if (!k.tiny) return __builtin_amdgcn_sqrtf(v);
    const bool small = v < 0x1p-96f;
    return __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v) * (small ? 0x1p-32f : 1.0f);
}

__device__ __forceinline__ float adamw_weight(float w, float m, float root, const AdamwScalars &k)
{
    return fmaf(-k.step_size * m, __builtin_amdgcn_rcpf(fmaf(root, k.inv_sqrt_c2, k.eps)), fmaf(-k.decay, w, w));
}

// (which products are fused is written out: a tensor's result does not depend on the form of the kernel that its size selects)
__device__ __forceinline__ void adamw_32(float &w, float g, float &m, float &v, const AdamwScalars &k)
{
    m = fmaf((float)k.beta1, m, (float)k.one_minus_beta1 * g);
    v = fmaf((float)k.beta2, v, (float)k.one_minus_beta2 * (g * g));
    w = adamw_weight(w, m, adamw_root(v, k), k);
}

// What a workgroup works on: TURNS * 1024 neighbouring elements of one tensor, `left` of them before its end.
struct AdamwChunk {
    int tensor;
    int64_t first, left;
};

template <int TURNS> __device__ __forceinline__ AdamwChunk adamw_chunk(const AdamwTable &a)
{
    const int i = __builtin_amdgcn_readfirstlane(adamw_tensor(a, blockIdx.x));
    const int64_t first = (int64_t)(blockIdx.x - (i ? a.last[i - 1] : 0u)) * (TURNS * 4 * AZ_ADAMW_THREADS);
    return AdamwChunk{i, first, a.n[i] - first};
}

// FULL: the chunk ends before its tensor does, so nothing needs a check.  STREAM: the step's tensors together are larger
// than every cache, so nothing of them is kept there for the next step.
template <bool FULL, bool STREAM, typename T> __device__ __forceinline__ float4 adamw_load(const T *p, int i, int n)
{
    if constexpr (FULL) return load4<STREAM>(p + i);
    else return load4(p, (int64_t)i, (int64_t)n);
}
template <bool FULL, bool STREAM, typename T> __device__ __forceinline__ void adamw_store(T *p, int i, int n, float4 f)
{
    if constexpr (FULL) store4<STREAM>(p + i, f);
    else store4(p, (int64_t)i, (int64_t)n, f);
}

template <typename T, int TURNS, bool STREAM, bool FULL> __device__ __forceinline__ void adamw_32_chunk(const AdamwTable &a, const AdamwScalars &k, const AdamwChunk &c)
{
    T *wp = static_cast<T *>(a.param[c.tensor]) + c.first;
    const T *gp = static_cast<const T *>(a.grad[c.tensor]) + c.first;
    float *mp = static_cast<float *>(a.m[c.tensor]) + c.first, *vp = static_cast<float *>(a.v[c.tensor]) + c.first;
    const int n = (int)min(c.left, (int64_t)(TURNS * 4 * AZ_ADAMW_THREADS));
    float4 w[TURNS], g[TURNS], m[TURNS], v[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
        const int at = (u * AZ_ADAMW_THREADS + threadIdx.x) * 4;
        w[u] = adamw_load<FULL, STREAM>(wp, at, n); g[u] = adamw_load<FULL, STREAM>(gp, at, n); m[u] = adamw_load<FULL, STREAM>(mp, at, n); v[u] = adamw_load<FULL, STREAM>(vp, at, n);
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
        const int at = (u * AZ_ADAMW_THREADS + threadIdx.x) * 4;
        adamw_32(w[u].x, g[u].x, m[u].x, v[u].x, k);
        adamw_32(w[u].y, g[u].y, m[u].y, v[u].y, k);
        adamw_32(w[u].z, g[u].z, m[u].z, v[u].z, k);
        adamw_32(w[u].w, g[u].w, m[u].w, v[u].w, k);
        adamw_store<FULL, STREAM>(wp, at, n, w[u]); adamw_store<FULL, STREAM>(mp, at, n, m[u]); adamw_store<FULL, STREAM>(vp, at, n, v[u]);
    }
}

template <typename T, int TURNS, bool STREAM> __global__ __launch_bounds__(AZ_ADAMW_THREADS) void k_adamw_32(AdamwTable a, AdamwScalars k)
{
    const AdamwChunk c = adamw_chunk<TURNS>(a);
    if (c.left >= TURNS * 4 * AZ_ADAMW_THREADS) adamw_32_chunk<T, TURNS, STREAM, true>(a, k, c);
    else adamw_32_chunk<T, TURNS, STREAM, false>(a, k, c);
}

// ---- states in 8 bits -------------------------------------------------------------------------------------------------
// A block of 256 elements shares one float32 scale S, the largest magnitude in it (rounded to nearest):
//   m = S * sgn(c) * (c / 127)^2,  c int8       v = S * (c / 255)^4,  c uint8
// The update divides m by sqrt(v), so what counts is the relative step of m and of sqrt(v): the powers put the codes where
// small values are (m down to 1.6e-5 and sqrt(v) down to 1.5e-5 of the block's largest) and still step by 1.6 % and 0.8 % at
// the top.  A code is the nearest one in the domain in which codes are evenly spaced, c = round(127 sqrt(|m| / S)),
// c = round(255 (v / S)^(1/4)), and at least 1 where v > 0, so that no element is ever divided by eps alone because its
// v was rounded away.
// Means are worked out in 64 bits, every operation rounded by itself in the order in which the formulas are written (no fused
// multiply-add): b1 S + (1 - b1) g lies exactly between two float32 values in one block of a hundred, and the scale must not
// depend on how a compiler contracts the sum.
// Codes are those of the 64-bit means too: a value next to a border between two codes goes to the right side of it.  A
// float32 estimate of 127 sqrt(|m| / S) or 255 sqrt(sqrt(v) / sqrt(S)) is off by less than 1e-4 (one step each of the conversion,
// the reciprocal, the roots and the products), so only what it puts within 2e-4 of a border, one wave in eight, is compared with
// that border, by powers and without roots: (2c - 1)^2 S < 254^2 |m| < (2c + 1)^2 S.  A value on a border goes to the even code
// (with b2 = 0 and 16-bit gradients that happens: both sides of the comparison round the same product then, and are equal).  With that, 95 M bfloat16 parameters take
// 180 to 192 us (950 MB, 5.0 to 5.3 TB/s); with the comparison for every element they took 360 us and were bound by arithmetic.
// A block with an infinity or a NaN in it has a scale that is not finite and reads back as NaN as a whole.

// byte e of a word as int8 / uint8, in float32: c |c| and c^2 are exact there
__device__ __forceinline__ float signed_code(uint32_t w, int e) { return (float)(int8_t)(w >> (8 * e)); }
__device__ __forceinline__ float unsigned_code(uint32_t w, int e) { return (float)(uint8_t)(w >> (8 * e)); }

__device__ __forceinline__ double dequantize_m(float c, double s) { return s * (double)(c * fabsf(c)) * (1.0 / 16129.0); }

__device__ __forceinline__ double dequantize_v(float c, double s)
{
    const double q = (double)(c * c);
    return s * (q * q) * (1.0 / 4228250625.0);   // 255^4
}

// the codes (as float32) from their borders; s > 0 and finite, inv = 1 / s
__device__ __forceinline__ float border_m(double m, double s, double inv)
{
    const double a = fabs(m), t = a * 64516.0;   // 254^2
    const int c = (int)rintf(127.0f * __builtin_amdgcn_sqrtf((float)(a * inv)));
    const double lo = (double)((2 * c - 1) * abs(2 * c - 1)) * s, hi = (double)((2 * c + 1) * (2 * c + 1)) * s;
    const bool odd = c & 1;
    return (float)min(c + (t > hi || (t == hi && odd) ? 1 : 0) - (t < lo || (t == lo && odd) ? 1 : 0), 127);
}

__device__ __forceinline__ float border_v(double v, double s, double inv)
{
    const double t = v * 67652010000.0;          // 510^4
    const int c = (int)rintf(255.0f * __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)(v * inv))));
    const double l = (double)((2 * c - 1) * abs(2 * c - 1)), h = (double)((2 * c + 1) * (2 * c + 1));
    const double lo = l * fabs(l) * s, hi = h * h * s;
    const bool odd = c & 1;
    return (float)min(c + (t > hi || (t == hi && odd) ? 1 : 0) - (t < lo || (t == lo && odd) ? 1 : 0), 255);
}

// Four codes as the bytes of a word; `bits` are the scale's, the same in the whole wave.  v comes with its root, which the
// update has needed already.
__device__ __forceinline__ uint32_t quantize_m(const double (&m)[4], const float (&f)[4], uint32_t bits)
{
    if (bits == 0 || bits >= 0x7f800000u) return 0;
    const float s = __uint_as_float(bits), inv = __builtin_amdgcn_rcpf(s);
    float c[4], off = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float x = 127.0f * __builtin_amdgcn_sqrtf(fabsf(f[e]) * inv);
        c[e] = rintf(x);
        off = fmaxf(off, fabsf(x - c[e]));
    }
    // (also where the reciprocal is no longer a normal number, or close to it)
    if (off > 0.4998f || s < 0x1p-100f || s > 0x1p100f) {
        const double d = (double)s, dinv = 1.0 / d;
#pragma unroll
        for (int e = 0; e < 4; e++) c[e] = border_m(m[e], d, dinv);
    }
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) w = __builtin_amdgcn_cvt_pk_u8_f32(copysignf(c[e], f[e]) + 128.0f, e, w);
    return w ^ 0x80808080u;
}

__device__ __forceinline__ uint32_t quantize_v(const double (&v)[4], const float (&root)[4], uint32_t bits)
{
    if (bits == 0 || bits >= 0x7f800000u) return 0;
    const float s = __uint_as_float(bits), inv = __builtin_amdgcn_rsqf(s);
    float c[4], off = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float x = 255.0f * __builtin_amdgcn_sqrtf(root[e] * inv);
        c[e] = rintf(x);
        off = fmaxf(off, fabsf(x - c[e]));
    }
    // (also where a subnormal v, whose root may read as 0, is not yet a code of 0)
    if (off > 0.4998f || s < 0x1p-60f || s > 0x1p100f) {
        const double d = (double)s, dinv = 1.0 / d;
#pragma unroll
        for (int e = 0; e < 4; e++) c[e] = border_v(v[e], d, dinv);
    }
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) w = __builtin_amdgcn_cvt_pk_u8_f32(v[e] > 0.0 ? fmaxf(c[e], 1.0f) : 0.0f, e, w);
    return w;
}

struct __attribute__((packed)) PackedWord { uint32_t v; };

// four codes as one word (any address); those past the end are 0 / are not written
template <bool FULL> __device__ __forceinline__ uint32_t load_codes(const uint8_t *p, int64_t i, int64_t n)
{
    if (FULL || i + 4 <= n) return reinterpret_cast<const PackedWord *>(p + i)->v;
    uint32_t w = 0;
    if (i < n) w = p[i];
    if (i + 1 < n) w |= (uint32_t)p[i + 1] << 8;
    if (i + 2 < n) w |= (uint32_t)p[i + 2] << 16;
    return w;
}

template <bool FULL> __device__ __forceinline__ void store_codes(uint8_t *p, int i, int n, uint32_t w)
{
    if (FULL || i + 4 <= n) { reinterpret_cast<PackedWord *>(p + i)->v = w; return; }
    if (i < n) p[i] = (uint8_t)w;
    if (i + 1 < n) p[i + 1] = (uint8_t)(w >> 8);
    if (i + 2 < n) p[i + 2] = (uint8_t)(w >> 16);
}

// A workgroup's chunk in blocks of 256, one for each of its waves at a time.
template <typename T, int TURNS, bool STREAM, bool FULL> __device__ __forceinline__ void adamw_8_chunk(const AdamwTable &a, const AdamwScalars &k, const AdamwChunk &ch)
{
    T *wp = static_cast<T *>(a.param[ch.tensor]) + ch.first;
    const T *gp = static_cast<const T *>(a.grad[ch.tensor]) + ch.first;
    uint8_t *mp = static_cast<uint8_t *>(a.m[ch.tensor]) + ch.first, *vp = static_cast<uint8_t *>(a.v[ch.tensor]) + ch.first;
    float *msp = a.m_scale[ch.tensor] + ch.first / AZ_ADAMW_BLOCK, *vsp = a.v_scale[ch.tensor] + ch.first / AZ_ADAMW_BLOCK;
    const int n = (int)min(ch.left, (int64_t)(TURNS * 4 * AZ_ADAMW_THREADS));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    static_assert(AZ_ADAMW_THREADS * 4 == 4 * AZ_ADAMW_BLOCK, "four waves, a block each");
    float4 w[TURNS], g[TURNS];
    uint32_t mc[TURNS], vc[TURNS];
    float ms[TURNS], vs[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
        const int at = (u * AZ_ADAMW_THREADS + threadIdx.x) * 4, block = u * 4 + wave;
        w[u] = adamw_load<FULL, STREAM>(wp, at, n); g[u] = adamw_load<FULL, STREAM>(gp, at, n);
        mc[u] = load_codes<FULL>(mp, at, n); vc[u] = load_codes<FULL>(vp, at, n);
        const bool in = FULL || block * AZ_ADAMW_BLOCK < n;
        ms[u] = in ? msp[block] : 0.f; vs[u] = in ? vsp[block] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
        const int at = (u * AZ_ADAMW_THREADS + threadIdx.x) * 4, block = u * 4 + wave;
        float *we = reinterpret_cast<float *>(&w[u]);
        const float *ge = reinterpret_cast<const float *>(&g[u]);
        double m[4], v[4];
        float mf[4], root[4];
        uint32_t mb = 0, vb = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
#pragma clang fp contract(off)
            const double gd = (double)ge[e];
            m[e] = k.beta1 * dequantize_m(signed_code(mc[u], e), (double)ms[u]) + k.one_minus_beta1 * gd;
            v[e] = k.beta2 * dequantize_v(unsigned_code(vc[u], e), (double)vs[u]) + k.one_minus_beta2 * (gd * gd);
            mf[e] = (float)m[e];
            const float vf = (float)v[e];
            mb = max(mb, __float_as_uint(mf[e]) & 0x7fffffffu);
            vb = max(vb, __float_as_uint(vf));     // (never negative)
            root[e] = adamw_root(vf, k);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) we[e] = adamw_weight(we[e], mf[e], root[e], k);
        // NaN has the largest magnitude bits of all, so the integer maximum keeps it
        mb = wave_umax(mb); vb = wave_umax(vb);
        const uint32_t mw = quantize_m(m, mf, mb), vw = quantize_v(v, root, vb);
        adamw_store<FULL, STREAM>(wp, at, n, w[u]);
        store_codes<FULL>(mp, at, n, mw); store_codes<FULL>(vp, at, n, vw);
        if ((threadIdx.x & 63) == 0 && (FULL || block * AZ_ADAMW_BLOCK < n)) {
            msp[block] = __uint_as_float(mb);
            vsp[block] = __uint_as_float(vb);
        }
    }
}

template <typename T, int TURNS, bool STREAM> __global__ __launch_bounds__(AZ_ADAMW_THREADS) void k_adamw_8(AdamwTable a, AdamwScalars k)
{
    const AdamwChunk c = adamw_chunk<TURNS>(a);
    if (c.left >= TURNS * 4 * AZ_ADAMW_THREADS) adamw_8_chunk<T, TURNS, STREAM, true>(a, k, c);
    else adamw_8_chunk<T, TURNS, STREAM, false>(a, k, c);
}

// the values that codes stand for, rounded once to float32
template <bool SIGNED> __global__ __launch_bounds__(AZ_ADAMW_THREADS) void k_dequantize_state(const uint8_t *codes, const float *scales, int64_t n, float *out)
{
    const int64_t step = (int64_t)gridDim.x * AZ_ADAMW_THREADS * 4;
    for (int64_t at = ((int64_t)blockIdx.x * AZ_ADAMW_THREADS + threadIdx.x) * 4; at < n; at += step) {
        const uint32_t w = load_codes<false>(codes, at, n);
        const double s = (double)scales[at / AZ_ADAMW_BLOCK];
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            f[e] = (float)(SIGNED ? dequantize_m(signed_code(w, e), s) : dequantize_v(unsigned_code(w, e), s));
        store4(out, at, n, make_float4(f[0], f[1], f[2], f[3]));
    }
}
