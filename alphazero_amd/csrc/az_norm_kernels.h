// Layer norm over the last axis, forward and backward.
//
//   y  = (x - mean) * r * w + b,  r = 1 / sqrt(var + eps),  var the mean of (x - mean)^2
//   dx = r * (g - mean(g) - h * mean(g * h)),  g = w * dy,  h = (x - mean) * r
//   dw = sum over rows of dy * h,   db = sum over rows of dy
//
// All sums are float32 whatever the elements' type.  What is summed for the mean is the row's values less its first one, and for
// the variance those less their mean, in a second pass over the registers: sums of the values themselves, or of their squares,
// are rounded in proportion to the mean and lose everything in rows whose mean is large against their spread (1000.1 in 361
// columns: a mean one step off, and with it h = 0.02 in a row without any spread).
// The mean that is kept for the backward pass is rounded to float32 once, which moves h by up to half its last place times r.
//
// A row belongs to TPR threads (4 to 32: part of a wave, 64: a wave, more: a workgroup), each of which holds NV packs of 16
// bytes of it in registers, so a row is read from memory once; the up to 3 or 7 elements past the last whole pack are held one
// to a thread.  Workgroups walk the rows with a stride: weights and biases
// are loaded once per thread and not once per row, and the next row is asked for before the present one is worked on.
#pragma once
#include "az_vec.h"

#define AZ_NORM_WIDE_THREADS 1024
#define AZ_NORM_COLS_WIDE_THREADS 256

constexpr int norm_threads(int tpr) { return tpr > 256 ? tpr : 256; }

// weights and biases: float32 or the element type; absent ones are 1 and 0
template <typename T> __device__ __forceinline__ float4 load_affine(const void *p, bool f32, int64_t i, int64_t n, float absent)
{
    if (!p) return make_float4(absent, absent, absent, absent);
    return f32 ? load4(static_cast<const float *>(p), i, n) : load4(static_cast<const T *>(p), i, n);
}

template <typename T> __device__ __forceinline__ void load_affine_pack(const void *p, bool f32, int i, bool in, float absent, float (&out)[Pack<T>::N])
{
#pragma unroll
    for (int e = 0; e < Pack<T>::N; e += 4) {
        const float4 f = load_affine<T>(in ? p : nullptr, f32, i + e, i + e + 4, absent);
        out[e] = f.x; out[e + 1] = f.y; out[e + 2] = f.z; out[e + 3] = f.w;
    }
}

template <typename T> __device__ __forceinline__ float load_affine_one(const void *p, bool f32, int i, bool in, float absent)
{
    if (!p || !in) return absent;
    return f32 ? static_cast<const float *>(p)[i] : (float)static_cast<const T *>(p)[i];
}

__device__ __forceinline__ float sum4(float4 f) { return (f.x + f.y) + (f.z + f.w); }

// Sums of TPR threads' values in each of them.  With a whole workgroup per row the waves meet in LDS; `slot` alternates
// between two sets of cells, so that one barrier per sum is enough: a cell is written again only after the other sum's barrier.
template <int TPR, int N> __device__ __forceinline__ void group_sum(float (&v)[N], float (*cell)[N][16], int slot)
{
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = TPR == 4 ? quad_sum(v[i]) : TPR == 8 ? oct_sum(v[i]) : TPR == 16 ? row16_sum(v[i]) : TPR == 32 ? half_sum(v[i]) : wave_sum(v[i]);
    if constexpr (TPR > 64) {
        constexpr int WAVES = TPR / 64;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; i++) cell[slot][i][wave] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            // (by the lanes of a row: as many values to each thread as there are waves cost registers, and with them workgroups)
            const float x = cell[slot][i][threadIdx.x & (WAVES - 1)];
            v[i] = WAVES == 4 ? quad_sum(x) : WAVES == 8 ? oct_sum(x) : row16_sum(x);
        }
    }
}

// 1 / sqrt(t) to one step of float32; the instruction takes no subnormal numbers
__device__ __forceinline__ float inv_sqrt(float t) { return t < 0x1p-126f ? 1.0f / sqrtf(t) : __builtin_amdgcn_rsqf(t); }

// How a row's values are taken relative to its first one: d = x scale - first.  The difference of two values overflows only in
// rows of the largest numbers, which are scaled down: 2^25 of them, of either sign, then have a sum.  (A first value below
// 2^102 is less than half a step of the largest number and takes nothing past it.)  The variance of such a row is infinite in
// float32 unless it is 0.
struct RowShift {
    float scale, first;
    __device__ __forceinline__ explicit RowShift(float x0) : scale(fabsf(x0) < 0x1p102f ? 1.0f : 0x1p-30f), first(x0 * scale) {}
    __device__ __forceinline__ float operator()(float x) const { return fmaf(x, scale, -first); }
    __device__ __forceinline__ float back() const { return scale == 1.0f ? 1.0f : 0x1p30f; }
    __device__ __forceinline__ float rstd(float squares, float inv, float eps) const     // from the sum of the squares of n d's, inv = 1 / n
    {
        return inv_sqrt(fmaf(squares, scale == 1.0f ? inv : inv * 0x1p60f, eps));
    }
    __device__ __forceinline__ float value(float d) const { return fmaf(d, back(), first * back()); }   // the x whose d this is
};

// a value that all lanes of a wave hold alike, in a scalar register
__device__ __forceinline__ float of_wave(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }

// The first lane's value in each lane of groups of TPR lanes (as a load of its own for every row it took 30 us and not 28 for
// 1 M rows of 32 bfloat16 columns).
template <int TPR> __device__ __forceinline__ float first_lane(float x)
{
    const uint32_t u = __float_as_uint(x);
    if constexpr (TPR == 4) return __uint_as_float(dpp_row<AZ_QUAD_FIRST>(u));
    else if constexpr (TPR == 8)      // lane 0's in all 16, then lane 8's in the upper two banks of four
        return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)dpp_row<AZ_ROW_LANE(0)>(u), (int)u, AZ_ROW_LANE(8), 0xf, 0xc, false));
    else if constexpr (TPR == 16) return __uint_as_float(dpp_row<AZ_ROW_LANE(0)>(u));
    else if constexpr (TPR == 32) {
        const uint32_t first = dpp_row<AZ_ROW_LANE(0)>(u);
        return __uint_as_float(__builtin_amdgcn_permlane16_swap(first, first, false, false)[0]);    // of the even row of a pair
    } else return of_wave(x);
}

struct NormFwd {
    const void *x, *w, *b;
    void *y;
    float *mean, *rstd;      // may be null
    int64_t rows, cols, x_stride, y_stride;
    float eps;
    bool affine_f32, stream; // stream: y is larger than the L2 caches
};

template <typename T, int TPR, int NV> __global__ __launch_bounds__(norm_threads(TPR)) void k_layer_norm_fwd(NormFwd a)
{
    constexpr int N = Pack<T>::N, GROUPS = norm_threads(TPR) / TPR;
    __shared__ float cell[2][1][16];
    const int t = threadIdx.x % TPR, cols = (int)a.cols, packs = cols / N, last = packs * N + t;
    const bool tail = last < cols;
    const float inv = 1.0f / (float)cols;
    float w[NV][N], b[NV][N];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        load_affine_pack<T>(a.w, a.affine_f32, (k * TPR + t) * N, k * TPR + t < packs, 1.0f, w[k]);
        load_affine_pack<T>(a.b, a.affine_f32, (k * TPR + t) * N, k * TPR + t < packs, 0.0f, b[k]);
    }
    const float w1 = load_affine_one<T>(a.w, a.affine_f32, last, tail, 1.0f), b1 = load_affine_one<T>(a.b, a.affine_f32, last, tail, 0.0f);
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const int group = threadIdx.x / TPR;
    int64_t row = (int64_t)blockIdx.x * GROUPS + (TPR < 64 ? group : __builtin_amdgcn_readfirstlane(group));
    typename Pack<T>::type next[NV];
    T next1, next0;
    // a row past the end reads as zeros
    const auto ask = [&](int64_t i) {
        const T *x = static_cast<const T *>(a.x) + i * a.x_stride;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            next[k] = {};
            if (i < a.rows && k * TPR + t < packs) next[k] = load_pack<false>(x + (k * TPR + t) * N);
        }
        next1 = next0 = T(0);
        if (i < a.rows && tail) next1 = x[last];
        if (TPR > 64 && i < a.rows) next0 = x[0];
    };
    ask(row);
    // the number of turns is the same for every thread of a workgroup
    for (int64_t first_row = (int64_t)blockIdx.x * GROUPS; first_row < a.rows; first_row += step, row += step) {
        // (with a wave or less to a row its first lane holds it, in the first pack or, if there is none, past it)
        RowShift shift(TPR > 64 ? (float)next0 : first_lane<TPR>(packs ? (float)next[0][0] : (float)next1));
        if constexpr (TPR >= 64) { shift.scale = of_wave(shift.scale); shift.first = of_wave(shift.first); }
        // (packs past a row's end are zeros, and stay so if nothing is taken from them)
        float v[NV][N], v1 = tail ? shift((float)next1) : 0.f, s[1] = {v1}, q[1];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const float first = k * TPR + t < packs ? shift.first : 0.f;
#pragma unroll
            for (int e = 0; e < N; e++) v[k][e] = fmaf((float)next[k][e], shift.scale, -first);
        }
        if (first_row + step < a.rows) ask(row + step);
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < N; e += 4) s[0] += (v[k][e] + v[k][e + 1]) + (v[k][e + 2] + v[k][e + 3]);
        group_sum<TPR>(s, cell, 0);
        const float mean = s[0] * inv;     // of the row's values less its first
        v1 = tail ? v1 - mean : 0.f;
        q[0] = v1 * v1;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const float centre = k * TPR + t < packs ? mean : 0.f;
#pragma unroll
            for (int e = 0; e < N; e++) v[k][e] -= centre;
        }
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < N; e += 4)
                q[0] += (v[k][e] * v[k][e] + v[k][e + 1] * v[k][e + 1]) + (v[k][e + 2] * v[k][e + 2] + v[k][e + 3] * v[k][e + 3]);
        group_sum<TPR>(q, cell, 1);
        const float r = shift.rstd(q[0], inv, a.eps), rs = r * shift.back();
        if (row < a.rows) {
            T *y = static_cast<T *>(a.y) + row * a.y_stride;
#pragma unroll
            for (int k = 0; k < NV; k++) {
#pragma unroll
                for (int e = 0; e < N; e++) v[k][e] = v[k][e] * rs * w[k][e] + b[k][e];
                if (k * TPR + t < packs) store_pack(y + (k * TPR + t) * N, v[k], a.stream);
            }
            if (tail) y[last] = (T)(v1 * rs * w1 + b1);
            if (a.mean && t == 0) { a.mean[row] = shift.value(mean); a.rstd[row] = r; }
        }
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

// Elements c .. c+3 of a row of n as `shift` takes them, less `mean`; 0 past the row's end.
__device__ __forceinline__ float4 shifted(float4 v, const RowShift &shift, float mean, int64_t c, int64_t n)
{
    const float4 d = make_float4(shift(v.x) - mean, shift(v.y) - mean, shift(v.z) - mean, shift(v.w) - mean);
    if (c + 4 <= n) return d;
    return make_float4(c < n ? d.x : 0.f, c + 1 < n ? d.y : 0.f, c + 2 < n ? d.z : 0.f, 0.f);
}
template <typename T> __device__ __forceinline__ float4 shifted(const T *x, const RowShift &shift, float mean, int64_t c, int64_t n)
{
    if (c + 4 <= n) return shifted(load4(x + c), shift, mean, 0, 4);
    return shifted(load4(x, c, n), shift, mean, c, n);
}

__device__ __forceinline__ float squares(float4 d) { return (d.x * d.x + d.y * d.y) + (d.z * d.z + d.w * d.w); }

// Rows too wide for a workgroup's registers: read three times, the second and third time from cache.
template <typename T> __global__ __launch_bounds__(AZ_NORM_WIDE_THREADS) void k_layer_norm_fwd_wide(NormFwd a)
{
    __shared__ float cell[AZ_NORM_WIDE_THREADS / 64];
    const float inv = 1.0f / (float)a.cols;
    const int64_t step = AZ_NORM_WIDE_THREADS * 4;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        T *y = static_cast<T *>(a.y) + row * a.y_stride;
        const RowShift shift((float)x[0]);
        float s = 0.f, q = 0.f;
        for (int64_t c = threadIdx.x * 4; c < a.cols; c += step) s += sum4(shifted(x, shift, 0.f, c, a.cols));
        const float mean = block_sum(s, cell) * inv;
        for (int64_t c = threadIdx.x * 4; c < a.cols; c += step) q += squares(shifted(x, shift, mean, c, a.cols));
        const float r = shift.rstd(block_sum(q, cell), inv, a.eps), rs = r * shift.back();
        for (int64_t c = threadIdx.x * 4; c < a.cols; c += step) {
            const float4 v = shifted(x, shift, mean, c, a.cols), w = load_affine<T>(a.w, a.affine_f32, c, a.cols, 1.0f);
            const float4 b = load_affine<T>(a.b, a.affine_f32, c, a.cols, 0.0f);
            store4(y, c, a.cols, make_float4(v.x * rs * w.x + b.x, v.y * rs * w.y + b.y, v.z * rs * w.z + b.z, v.w * rs * w.w + b.w));
        }
        if (a.mean && threadIdx.x == 0) { a.mean[row] = shift.value(mean); a.rstd[row] = r; }
    }
}

// A few rows that are too wide: a workgroup to a chunk of 8192 elements, in two launches.  The first leaves each chunk's mean
// (relative to the row's first value) and its sum of squared distances from that mean; the second puts them together,
//   mean = sum n_i mean_i / n,   sum of squares = sum (M2_i + n_i (mean_i - mean)^2),
// and writes its chunk.  3 rows of 300 k float32: 9 us, with a workgroup to each row 103.
#define AZ_NORM_CHUNK 8192

// the elements of thread threadIdx.x's pack k of four in the chunk
__device__ __forceinline__ int64_t chunk_at(int k) { return (int64_t)blockIdx.x * AZ_NORM_CHUNK + (k * AZ_NORM_WIDE_THREADS + threadIdx.x) * 4; }

template <typename T> __global__ __launch_bounds__(AZ_NORM_WIDE_THREADS) void k_layer_norm_chunk_stats(NormFwd a, float2 *part)
{
    __shared__ float cell[AZ_NORM_WIDE_THREADS / 64];
    constexpr int NV = AZ_NORM_CHUNK / (AZ_NORM_WIDE_THREADS * 4);
    const T *x = static_cast<const T *>(a.x) + blockIdx.y * a.x_stride;
    const float n = (float)min((int64_t)AZ_NORM_CHUNK, a.cols - (int64_t)blockIdx.x * AZ_NORM_CHUNK);
    const RowShift shift((float)x[0]);
    float4 v[NV];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int k = 0; k < NV; k++) v[k] = load4(x, chunk_at(k), a.cols);
#pragma unroll
    for (int k = 0; k < NV; k++) s += sum4(shifted(v[k], shift, 0.f, chunk_at(k), a.cols));
    const float mean = block_sum(s, cell) / n;
#pragma unroll
    for (int k = 0; k < NV; k++) q += squares(shifted(v[k], shift, mean, chunk_at(k), a.cols));
    q = block_sum(q, cell);
    if (threadIdx.x == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = make_float2(mean, q);
}

template <typename T> __global__ __launch_bounds__(AZ_NORM_WIDE_THREADS) void k_layer_norm_chunk_write(NormFwd a, const float2 *part)
{
    __shared__ float cell[AZ_NORM_WIDE_THREADS / 64];
    constexpr int NV = AZ_NORM_CHUNK / (AZ_NORM_WIDE_THREADS * 4);
    const T *x = static_cast<const T *>(a.x) + blockIdx.y * a.x_stride;
    T *y = static_cast<T *>(a.y) + blockIdx.y * a.y_stride;
    float4 v[NV], w[NV], b[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        v[k] = load4(x, chunk_at(k), a.cols);
        w[k] = load_affine<T>(a.w, a.affine_f32, chunk_at(k), a.cols, 1.0f);
        b[k] = load_affine<T>(a.b, a.affine_f32, chunk_at(k), a.cols, 0.0f);
    }
    part += (int64_t)blockIdx.y * gridDim.x;
    const RowShift shift((float)x[0]);
    const float inv = 1.0f / (float)a.cols;
    const auto count = [&](unsigned i) { return (float)min((int64_t)AZ_NORM_CHUNK, a.cols - (int64_t)i * AZ_NORM_CHUNK); };
    float s = 0.f, q = 0.f;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += AZ_NORM_WIDE_THREADS) s += count(i) * part[i].x;
    const float mean = block_sum(s, cell) * inv;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += AZ_NORM_WIDE_THREADS) {
        const float d = part[i].x - mean;
        q += part[i].y + count(i) * d * d;
    }
    const float r = shift.rstd(block_sum(q, cell), inv, a.eps), rs = r * shift.back();
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const float4 d = shifted(v[k], shift, mean, chunk_at(k), a.cols);
        store4(y, chunk_at(k), a.cols, make_float4(d.x * rs * w[k].x + b[k].x, d.y * rs * w[k].y + b[k].y, d.z * rs * w[k].z + b[k].z, d.w * rs * w[k].w + b[k].w));
    }
    if (a.mean && blockIdx.x == 0 && threadIdx.x == 0) { a.mean[blockIdx.y] = shift.value(mean); a.rstd[blockIdx.y] = r; }
}

struct NormBwd {
    const void *dy, *x, *w;
    const float *mean, *rstd;
    void *dx;                // null: not wanted
    float *part;             // [2][parts][cols] sums of the workgroups' rows: dw, then db; null: not wanted
    int64_t parts, turns, times;   // a workgroup writes its sums after so many turns, so many times in all
    int64_t rows, cols, dy_stride, x_stride, dx_stride;
    bool affine_f32, stream; // stream: dx is larger than the L2 caches
};

// dx of the rows, and for every workgroup the sums of dy * h and dy over its rows in the order in which it meets them: no
// atomics, so the same call gives the same bits.  (A workgroup of one group writes them out after a number of rows and starts
// anew: a long chain of additions would lose what a short one keeps.)  The threads of a workgroup that hold the same columns of different rows
// add up through LDS at the end.
// Elements past a row's end read as dy = 0 and have h = 0, so they add nothing to any sum, and they are not stored.  (Their h is
// -mean times 0 and not times r: in a row without spread r is 1 / sqrt(eps), so that can overflow, and 0 times infinity is NaN.)
// STREAM: x and dy, which this pass is the last to read, go past the L2 caches.
// Without SUMS there is dx alone: a thread of a workgroup of 1024 has registers for 16 elements of x, dy and w, but not for
// their sums too.
template <typename T, int TPR, int NV, bool STREAM, bool SUMS> __global__ __launch_bounds__(norm_threads(TPR)) void k_layer_norm_bwd(NormBwd a)
{
    constexpr int N = Pack<T>::N, THREADS = norm_threads(TPR), GROUPS = THREADS / TPR, WIDTH = (TPR * NV + 1) * N;
    __shared__ float cell[2][2][16];
    __shared__ float gather[GROUPS > 1 ? GROUPS * WIDTH : 1];
    const int t = threadIdx.x % TPR, cols = (int)a.cols, packs = cols / N, last = packs * N + t;
    const bool tail = last < cols;
    const float inv = 1.0f / (float)cols;
    float w[NV][N], dw[SUMS ? NV : 1][N], db[SUMS ? NV : 1][N], dw1 = 0.f, db1 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        load_affine_pack<T>(a.w, a.affine_f32, (k * TPR + t) * N, k * TPR + t < packs, 1.0f, w[k]);
        if constexpr (SUMS) {
#pragma unroll
            for (int e = 0; e < N; e++) dw[k][e] = db[k][e] = 0.f;
        }
    }
    const float w1 = load_affine_one<T>(a.w, a.affine_f32, last, tail, 1.0f);
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / TPR;
    typename Pack<T>::type next_x[NV], next_dy[NV];
    T next_x1, next_dy1;
    float next_mean, next_r;
    const auto ask = [&](int64_t i) {
        const T *x = static_cast<const T *>(a.x) + i * a.x_stride, *dy = static_cast<const T *>(a.dy) + i * a.dy_stride;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            next_x[k] = next_dy[k] = {};
            if (i < a.rows && k * TPR + t < packs) {
                next_x[k] = load_pack<STREAM>(x + (k * TPR + t) * N);
                next_dy[k] = load_pack<STREAM>(dy + (k * TPR + t) * N);
            }
        }
        next_x1 = next_dy1 = T(0);
        if (i < a.rows && tail) { next_x1 = x[last]; next_dy1 = dy[last]; }
        next_mean = i < a.rows ? a.mean[i] : 0.f;
        next_r = i < a.rows ? a.rstd[i] : 0.f;
    };
    // one partial row of a workgroup that is a single group; its sums start anew
    int64_t left = a.turns, written = 0;
    const auto write = [&] {
        float *to = a.part + (written++ * gridDim.x + blockIdx.x) * a.cols;
#pragma unroll
        for (int k = 0; k < (SUMS ? NV : 0); k++) {
            const int at = (k * TPR + t) * N;
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                if (k * TPR + t < packs) {
                    store4(to + at + e, make_float4(dw[k][e], dw[k][e + 1], dw[k][e + 2], dw[k][e + 3]));
                    store4(to + a.parts * a.cols + at + e, make_float4(db[k][e], db[k][e + 1], db[k][e + 2], db[k][e + 3]));
                }
            }
#pragma unroll
            for (int e = 0; e < N; e++) dw[k][e] = db[k][e] = 0.f;
        }
        if (tail) { to[last] = dw1; to[a.parts * a.cols + last] = db1; }
        dw1 = db1 = 0.f;
    };
    ask(row);
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < a.rows; first += step, row += step, turn ^= 1) {
        const float mean = next_mean, r = next_r;
        const float h1 = ((float)next_x1 - mean) * (tail ? r : 0.f);
        float h[NV][N], g[NV][N], g1 = (float)next_dy1;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const float rk = k * TPR + t < packs ? r : 0.f;
#pragma unroll
            for (int e = 0; e < N; e++) { h[k][e] = ((float)next_x[k][e] - mean) * rk; g[k][e] = (float)next_dy[k][e]; }
        }
        if (first + step < a.rows) ask(row + step);
        dw1 += g1 * h1;
        db1 += g1;
        g1 *= w1;
        float s[2] = {g1, g1 * h1};
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                if constexpr (SUMS) {
                    dw[k][e] += g[k][e] * h[k][e];
                    db[k][e] += g[k][e];
                }
                g[k][e] *= w[k][e];
                s[0] += g[k][e];
                s[1] += g[k][e] * h[k][e];
            }
        if constexpr (SUMS && GROUPS == 1)
            if (a.part && --left == 0) { write(); left = a.turns; }
        if (!a.dx) continue;
        group_sum<TPR>(s, cell, turn);
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        if (row < a.rows) {
            T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
#pragma unroll
            for (int k = 0; k < NV; k++) {
#pragma unroll
                for (int e = 0; e < N; e++) g[k][e] = r * (g[k][e] - m0 - h[k][e] * m1);
                if (k * TPR + t < packs) store_pack(dx + (k * TPR + t) * N, g[k], a.stream);
            }
            if (tail) dx[last] = (T)(r * (g1 - m0 - h1 * m1));
        }
    }
    if (!a.part) return;
    if constexpr (SUMS && GROUPS == 1) {
        while (written < a.times) write();       // (zeros where this workgroup had a row less than others)
    } else if constexpr (SUMS) {
#pragma unroll
        for (int which = 0; which < 2; which++) {
            float *part = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * a.cols;
            __syncthreads();
            float *mine = gather + (threadIdx.x / TPR) * WIDTH;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                if (k * TPR + t < packs) {
#pragma unroll
                    for (int e = 0; e < N; e++) mine[(k * TPR + t) * N + e] = which ? db[k][e] : dw[k][e];
                }
            }
            if (tail) mine[last] = which ? db1 : dw1;
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += THREADS) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < GROUPS; i++) sum += gather[i * WIDTH + c];
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

// The same for a few rows, in chunks as forward: the chunks' two sums, then dx.
template <typename T> __global__ __launch_bounds__(AZ_NORM_WIDE_THREADS) void k_layer_norm_chunk_sums(NormBwd a, float2 *part)
{
    __shared__ float cell[AZ_NORM_WIDE_THREADS / 64];
    constexpr int NV = AZ_NORM_CHUNK / (AZ_NORM_WIDE_THREADS * 4);
    const T *x = static_cast<const T *>(a.x) + blockIdx.y * a.x_stride, *dy = static_cast<const T *>(a.dy) + blockIdx.y * a.dy_stride;
    const float mean = a.mean[blockIdx.y], r = a.rstd[blockIdx.y];
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int64_t c = chunk_at(k);
        const float4 v = load4(x, c, a.cols), g = load4(dy, c, a.cols), w = load_affine<T>(a.w, a.affine_f32, c, a.cols, 1.0f);
        const float g0 = g.x * w.x, g1 = g.y * w.y, g2 = g.z * w.z, g3 = g.w * w.w;
        if (c < a.cols) { s0 += g0; s1 += g0 * ((v.x - mean) * r); }
        if (c + 1 < a.cols) { s0 += g1; s1 += g1 * ((v.y - mean) * r); }
        if (c + 2 < a.cols) { s0 += g2; s1 += g2 * ((v.z - mean) * r); }
        if (c + 3 < a.cols) { s0 += g3; s1 += g3 * ((v.w - mean) * r); }
    }
    s0 = block_sum(s0, cell);
    s1 = block_sum(s1, cell);
    if (threadIdx.x == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = make_float2(s0, s1);
}

template <typename T> __global__ __launch_bounds__(AZ_NORM_WIDE_THREADS) void k_layer_norm_chunk_dx(NormBwd a, const float2 *part)
{
    __shared__ float cell[AZ_NORM_WIDE_THREADS / 64];
    constexpr int NV = AZ_NORM_CHUNK / (AZ_NORM_WIDE_THREADS * 4);
    const T *x = static_cast<const T *>(a.x) + blockIdx.y * a.x_stride, *dy = static_cast<const T *>(a.dy) + blockIdx.y * a.dy_stride;
    T *dx = static_cast<T *>(a.dx) + blockIdx.y * a.dx_stride;
    const float mean = a.mean[blockIdx.y], r = a.rstd[blockIdx.y], inv = 1.0f / (float)a.cols;
    part += (int64_t)blockIdx.y * gridDim.x;
    float s0 = 0.f, s1 = 0.f;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += AZ_NORM_WIDE_THREADS) { s0 += part[i].x; s1 += part[i].y; }
    const float m0 = block_sum(s0, cell) * inv, m1 = block_sum(s1, cell) * inv;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int64_t c = chunk_at(k);
        const float4 v = load4(x, c, a.cols), g = load4(dy, c, a.cols), w = load_affine<T>(a.w, a.affine_f32, c, a.cols, 1.0f);
        store4(dx, c, a.cols,
               make_float4(r * (g.x * w.x - m0 - (v.x - mean) * r * m1), r * (g.y * w.y - m0 - (v.y - mean) * r * m1),
                           r * (g.z * w.z - m0 - (v.z - mean) * r * m1), r * (g.w * w.w - m0 - (v.w - mean) * r * m1)));
    }
}

// The sums over rows for wide rows: a workgroup takes 1024 columns and every gridDim.y-th row.
template <typename T> __global__ __launch_bounds__(AZ_NORM_COLS_WIDE_THREADS) void k_layer_norm_cols_wide(NormBwd a)
{
    const int64_t c = ((int64_t)blockIdx.x * AZ_NORM_COLS_WIDE_THREADS + threadIdx.x) * 4;
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

// Adds the workgroups' sums.  16 columns per workgroup, so that even a row of 256 columns gives 32 of them: each row of 16 lanes
// takes every 64th part, the four rows of a wave add up by row swaps, the 16 waves in LDS.  blockIdx.y: dw, db.
template <typename T> __global__ __launch_bounds__(1024) void k_layer_norm_cols(const float *part, int64_t parts, int64_t cols, void *dw, void *db, bool affine_f32)
{
    __shared__ float cell[16][16];
    const int lane = threadIdx.x & 15, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 16 + lane;
    void *out = blockIdx.y ? db : dw;
    if (!out) return;
    part += (int64_t)blockIdx.y * parts * cols;
    float s = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int64_t p = threadIdx.x >> 4; p < parts; p += 64) s += part[p * cols + c];
    }
    s = add_halves(add_row_pairs(s));
    if ((threadIdx.x & 63) < 16) cell[wave][lane] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || c >= cols) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += cell[i][lane];
    if (affine_f32) static_cast<float *>(out)[c] = s;
    else static_cast<T *>(out)[c] = (T)s;
}
