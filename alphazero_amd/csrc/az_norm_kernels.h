// Layer norm over the last axis, forward and backward.
//
//   y  = (x - mean) * r * w + b,  r = 1 / sqrt(var + eps),  var the mean of (x - mean)^2
//   dx = r * (g - mean(g) - h * mean(g * h)),  g = w * dy,  h = (x - mean) * r
//   dw = sum over rows of dy * h,   db = sum over rows of dy
//
// All sums are float32 whatever the elements' type.  The variance is taken from the row's values less their mean, in
// registers, in a second pass over those registers: a sum of squares would lose everything in rows whose mean is large
// against their spread.
//
// A row belongs to TPR threads (16: a quarter of a wave, 64: a wave, 256: a workgroup), each of which holds NV groups of four
// neighbouring elements in registers, so a row is read from memory once.  Workgroups walk the rows with a stride, so that
// weights and biases are loaded once per thread and not once per row.
#pragma once
#include "az_vec.h"

#define AZ_NORM_THREADS 256
#define AZ_NORM_WIDE_THREADS 1024

// weights and biases: float32 or the element type; absent ones are 1 and 0
template <typename T> __device__ __forceinline__ float4 load_affine(const void *p, bool f32, int64_t i, int64_t n, float absent)
{
    if (!p) return make_float4(absent, absent, absent, absent);
    return f32 ? load4(static_cast<const float *>(p), i, n) : load4(static_cast<const T *>(p), i, n);
}

__device__ __forceinline__ float sum4(float4 f) { return (f.x + f.y) + (f.z + f.w); }

// Sums of TPR threads' values in each of them.  With a whole workgroup per row the four waves meet in LDS; `slot` alternates
// between two pairs of cells, so that one barrier per sum is enough: a cell is written again only after the other sum's barrier.
template <int TPR, int N> __device__ __forceinline__ void group_sum(float (&v)[N], float (*cell)[AZ_NORM_THREADS / 64][2], int slot)
{
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = TPR == 16 ? row16_sum(v[i]) : wave_sum(v[i]);
    if constexpr (TPR == AZ_NORM_THREADS) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; i++) cell[slot][wave][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (cell[slot][0][i] + cell[slot][1][i]) + (cell[slot][2][i] + cell[slot][3][i]);
    }
}

struct NormFwd {
    const void *x, *w, *b;
    void *y;
    float *mean, *rstd;      // may be null
    int64_t rows, cols, x_stride, y_stride;
    float eps;
    bool affine_f32;
};

template <typename T, int TPR, int NV> __global__ __launch_bounds__(AZ_NORM_THREADS) void k_layer_norm_fwd(NormFwd a)
{
    __shared__ float cell[2][AZ_NORM_THREADS / 64][2];
    constexpr int GROUPS = AZ_NORM_THREADS / TPR;
    const int t = threadIdx.x % TPR;
    const float inv = 1.0f / (float)a.cols;
    float4 w[NV], b[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int64_t c = (int64_t)(k * TPR + t) * 4;
        w[k] = load_affine<T>(a.w, a.affine_f32, c, a.cols, 1.0f);
        b[k] = load_affine<T>(a.b, a.affine_f32, c, a.cols, 0.0f);
    }
    // the number of turns is the same for every thread of a workgroup: lanes whose row is past the end sum zeros
    for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < a.rows; first += (int64_t)gridDim.x * GROUPS) {
        const int64_t row = first + threadIdx.x / TPR;
        const bool in = row < a.rows;
        const int64_t cols = in ? a.cols : 0;
        const T *x = static_cast<const T *>(a.x) + (in ? row : 0) * a.x_stride;
        float4 v[NV];
        float s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; k++) v[k] = load4(x, (int64_t)(k * TPR + t) * 4, cols);
#pragma unroll
        for (int k = 0; k < NV; k++) s[0] += sum4(v[k]);
        group_sum<TPR>(s, cell, 0);
        const float mean = s[0] / (float)a.cols;   // (a division: rows of one value come out with exactly that mean)
        float q[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t c = (int64_t)(k * TPR + t) * 4;
            v[k].x = c < cols ? v[k].x - mean : 0.f;
            v[k].y = c + 1 < cols ? v[k].y - mean : 0.f;
            v[k].z = c + 2 < cols ? v[k].z - mean : 0.f;
            v[k].w = c + 3 < cols ? v[k].w - mean : 0.f;
            q[0] += (v[k].x * v[k].x + v[k].y * v[k].y) + (v[k].z * v[k].z + v[k].w * v[k].w);
        }
        group_sum<TPR>(q, cell, 1);
        const float r = 1.0f / sqrtf(q[0] * inv + a.eps);
        T *y = static_cast<T *>(a.y) + (in ? row : 0) * a.y_stride;
#pragma unroll
        for (int k = 0; k < NV; k++)
            store4(y, (int64_t)(k * TPR + t) * 4, cols,
                   make_float4(v[k].x * r * w[k].x + b[k].x, v[k].y * r * w[k].y + b[k].y, v[k].z * r * w[k].z + b[k].z, v[k].w * r * w[k].w + b[k].w));
        if (a.mean && in && t == 0) { a.mean[row] = mean; a.rstd[row] = r; }
    }
}

// Sum over a workgroup of 1024 threads, in every thread; `cell` is free again at the next call's first barrier.
__device__ __forceinline__ float block_sum(float x, float *cell)
{
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) cell[threadIdx.x >> 6] = x;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < AZ_NORM_WIDE_THREADS / 64; i++) s += cell[i];
    return s;
}

// Rows too wide for a workgroup's registers: read three times, the second and third time from cache.
template <typename T> __global__ __launch_bounds__(AZ_NORM_WIDE_THREADS) void k_layer_norm_fwd_wide(NormFwd a)
{
    __shared__ float cell[AZ_NORM_WIDE_THREADS / 64];
    const float inv = 1.0f / (float)a.cols;
    const int64_t step = AZ_NORM_WIDE_THREADS * 4;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        T *y = static_cast<T *>(a.y) + row * a.y_stride;
        float s = 0.f, q = 0.f;
        for (int64_t c = threadIdx.x * 4; c < a.cols; c += step) s += sum4(load4(x, c, a.cols));
        const float mean = block_sum(s, cell) / (float)a.cols;
        for (int64_t c = threadIdx.x * 4; c < a.cols; c += step) {
            const float4 v = load4(x, c, a.cols);
            const float d0 = v.x - mean, d1 = v.y - mean, d2 = v.z - mean, d3 = v.w - mean;
            q += d0 * d0;
            if (c + 1 < a.cols) q += d1 * d1;
            if (c + 2 < a.cols) q += d2 * d2;
            if (c + 3 < a.cols) q += d3 * d3;
        }
        const float r = 1.0f / sqrtf(block_sum(q, cell) * inv + a.eps);
        for (int64_t c = threadIdx.x * 4; c < a.cols; c += step) {
            const float4 v = load4(x, c, a.cols), w = load_affine<T>(a.w, a.affine_f32, c, a.cols, 1.0f);
            const float4 b = load_affine<T>(a.b, a.affine_f32, c, a.cols, 0.0f);
            store4(y, c, a.cols, make_float4((v.x - mean) * r * w.x + b.x, (v.y - mean) * r * w.y + b.y, (v.z - mean) * r * w.z + b.z, (v.w - mean) * r * w.w + b.w));
        }
        if (a.mean && threadIdx.x == 0) { a.mean[row] = mean; a.rstd[row] = r; }
    }
}

struct NormBwd {
    const void *dy, *x, *w;
    const float *mean, *rstd;
    void *dx;                // null: not wanted
    float *part;             // [2][parts][cols] sums of the workgroups' rows: dw, then db; null: not wanted
    int64_t rows, cols, dy_stride, x_stride, dx_stride;
    bool affine_f32;
};

// dx of the rows, and for every workgroup the sums of dy * h and dy over its rows in the order in which it meets them: no
// atomics, so the same call gives the same bits.  The threads of a workgroup that hold the same columns of different rows
// add up through LDS at the end.
template <typename T, int TPR, int NV> __global__ __launch_bounds__(AZ_NORM_THREADS) void k_layer_norm_bwd(NormBwd a)
{
    constexpr int GROUPS = AZ_NORM_THREADS / TPR, WIDTH = TPR * NV * 4;
    __shared__ float cell[2][AZ_NORM_THREADS / 64][2];
    __shared__ float4 gather[GROUPS > 1 ? GROUPS * WIDTH / 4 : 1];
    const int t = threadIdx.x % TPR;
    const float inv = 1.0f / (float)a.cols;
    float4 w[NV], dw[NV], db[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        w[k] = load_affine<T>(a.w, a.affine_f32, (int64_t)(k * TPR + t) * 4, a.cols, 1.0f);
        dw[k] = db[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < a.rows; first += (int64_t)gridDim.x * GROUPS, turn ^= 1) {
        const int64_t row = first + threadIdx.x / TPR;
        const bool in = row < a.rows;
        const int64_t cols = in ? a.cols : 0, at = in ? row : 0;
        const T *x = static_cast<const T *>(a.x) + at * a.x_stride, *dy = static_cast<const T *>(a.dy) + at * a.dy_stride;
        const float mean = a.mean[at], r = a.rstd[at];
        float4 h[NV], g[NV];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; k++) {
            h[k] = load4(x, (int64_t)(k * TPR + t) * 4, cols);
            g[k] = load4(dy, (int64_t)(k * TPR + t) * 4, cols);
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t c = (int64_t)(k * TPR + t) * 4;
            // h of an element past the row's end is 0, not -mean * r, which could be infinite
            h[k].x = c < cols ? (h[k].x - mean) * r : 0.f;
            h[k].y = c + 1 < cols ? (h[k].y - mean) * r : 0.f;
            h[k].z = c + 2 < cols ? (h[k].z - mean) * r : 0.f;
            h[k].w = c + 3 < cols ? (h[k].w - mean) * r : 0.f;
            dw[k].x += g[k].x * h[k].x; dw[k].y += g[k].y * h[k].y; dw[k].z += g[k].z * h[k].z; dw[k].w += g[k].w * h[k].w;
            db[k].x += g[k].x; db[k].y += g[k].y; db[k].z += g[k].z; db[k].w += g[k].w;
            g[k].x *= w[k].x; g[k].y *= w[k].y; g[k].z *= w[k].z; g[k].w *= w[k].w;
            s[0] += sum4(g[k]);
            s[1] += (g[k].x * h[k].x + g[k].y * h[k].y) + (g[k].z * h[k].z + g[k].w * h[k].w);
        }
        if (!a.dx) continue;
        group_sum<TPR>(s, cell, turn);
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        T *dx = static_cast<T *>(a.dx) + at * a.dx_stride;
#pragma unroll
        for (int k = 0; k < NV; k++)
            store4(dx, (int64_t)(k * TPR + t) * 4, cols,
                   make_float4(r * (g[k].x - m0 - h[k].x * m1), r * (g[k].y - m0 - h[k].y * m1), r * (g[k].z - m0 - h[k].z * m1), r * (g[k].w - m0 - h[k].w * m1)));
    }
    if (!a.part) return;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float *part = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * a.cols;
        if constexpr (GROUPS == 1) {
#pragma unroll
            for (int k = 0; k < NV; k++) store4(part, (int64_t)(k * TPR + t) * 4, a.cols, which ? db[k] : dw[k]);
        } else {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; k++) gather[(threadIdx.x / TPR) * (WIDTH / 4) + k * TPR + t] = which ? db[k] : dw[k];
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += AZ_NORM_THREADS) {
                float sum = 0.f;
#pragma unroll
                for (int g = 0; g < GROUPS; g++) sum += reinterpret_cast<const float *>(gather)[g * WIDTH + c];
                part[c] = sum;
            }
        }
    }
}

// dx of rows too wide for registers (two reads of x and dy)
template <typename T> __global__ __launch_bounds__(AZ_NORM_WIDE_THREADS) void k_layer_norm_bwd_wide(NormBwd a)
{
    __shared__ float cell[AZ_NORM_WIDE_THREADS / 64];
    const float inv = 1.0f / (float)a.cols;
    const int64_t step = AZ_NORM_WIDE_THREADS * 4;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride, *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
        T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
        const float mean = a.mean[row], r = a.rstd[row];
        float s0 = 0.f, s1 = 0.f;
        for (int64_t c = threadIdx.x * 4; c < a.cols; c += step) {
            const float4 v = load4(x, c, a.cols), g = load4(dy, c, a.cols), w = load_affine<T>(a.w, a.affine_f32, c, a.cols, 1.0f);
            const float g0 = g.x * w.x, g1 = g.y * w.y, g2 = g.z * w.z, g3 = g.w * w.w;
            s0 += g0; s1 += g0 * ((v.x - mean) * r);
            if (c + 1 < a.cols) { s0 += g1; s1 += g1 * ((v.y - mean) * r); }
            if (c + 2 < a.cols) { s0 += g2; s1 += g2 * ((v.z - mean) * r); }
            if (c + 3 < a.cols) { s0 += g3; s1 += g3 * ((v.w - mean) * r); }
        }
        const float m0 = block_sum(s0, cell) * inv, m1 = block_sum(s1, cell) * inv;
        for (int64_t c = threadIdx.x * 4; c < a.cols; c += step) {
            const float4 v = load4(x, c, a.cols), g = load4(dy, c, a.cols), w = load_affine<T>(a.w, a.affine_f32, c, a.cols, 1.0f);
            store4(dx, c, a.cols,
                   make_float4(r * (g.x * w.x - m0 - (v.x - mean) * r * m1), r * (g.y * w.y - m0 - (v.y - mean) * r * m1),
                               r * (g.z * w.z - m0 - (v.z - mean) * r * m1), r * (g.w * w.w - m0 - (v.w - mean) * r * m1)));
        }
    }
}

// The sums over rows for wide rows: a workgroup takes 1024 columns and every gridDim.y-th row.
template <typename T> __global__ __launch_bounds__(AZ_NORM_THREADS) void k_layer_norm_cols_wide(NormBwd a)
{
    const int64_t c = ((int64_t)blockIdx.x * AZ_NORM_THREADS + threadIdx.x) * 4;
    if (c >= a.cols) return;
    float4 dw = make_float4(0.f, 0.f, 0.f, 0.f), db = dw;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float4 v = load4(static_cast<const T *>(a.x) + row * a.x_stride, c, a.cols);
        const float4 g = load4(static_cast<const T *>(a.dy) + row * a.dy_stride, c, a.cols);
        const float mean = a.mean[row], r = a.rstd[row];
        dw.x += g.x * ((v.x - mean) * r); dw.y += g.y * ((v.y - mean) * r); dw.z += g.z * ((v.z - mean) * r); dw.w += g.w * ((v.w - mean) * r);
        db.x += g.x; db.y += g.y; db.z += g.z; db.w += g.w;
    }
    store4(a.part + (int64_t)blockIdx.y * a.cols, c, a.cols, dw);
    store4(a.part + ((int64_t)gridDim.y + blockIdx.y) * a.cols, c, a.cols, db);
}

// Adds the workgroups' sums: 64 columns per workgroup, its 16 waves take every 16th part and meet in LDS.  blockIdx.y: dw, db.
template <typename T> __global__ __launch_bounds__(1024) void k_layer_norm_cols(const float *part, int64_t parts, int64_t cols, void *dw, void *db, bool affine_f32)
{
    __shared__ float cell[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    void *out = blockIdx.y ? db : dw;
    if (!out) return;
    part += (int64_t)blockIdx.y * parts * cols;
    float s = 0.f;
    if (c < cols)
        for (int64_t p = wave; p < parts; p += 16) s += part[p * cols + c];
    cell[wave][lane] = s;
    __syncthreads();
    if (wave || c >= cols) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += cell[i][lane];
    if (affine_f32) static_cast<float *>(out)[c] = s;
    else static_cast<T *>(out)[c] = (T)s;
}
