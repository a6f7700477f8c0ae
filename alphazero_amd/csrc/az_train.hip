// Training operators of the C ABI (include/az_engine.h): layer norm with its gradient, the AdamW step.
#include "../../include/az_engine.h"
#include "az_error.h"
#include "az_norm_kernels.h"
#include "az_adamw_kernels.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <vector>

namespace {

// The caller's device for the duration of a call: kernels go to the device of the tensors, the calling thread's current
// device stays what it was.
struct DeviceScope {
    int before = -1, now;
    hipError_t error;
    explicit DeviceScope(int device) : now(device)
    {
        (void)hipGetLastError();   // (what an earlier call of this thread left there is not this call's error)
        error = hipGetDevice(&before);
        if (error == hipSuccess && before != device) error = hipSetDevice(device);
    }
    ~DeviceScope() { if (before >= 0 && before != now) (void)hipSetDevice(before); }
};

int fail_hip(const char *what, hipError_t e)
{
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", what, hipGetErrorString(e));
    return az_fail(AZ_ERR_HIP, buf);
}

bool bad_type(int32_t t) { return t != AZ_TYPE_F32 && t != AZ_TYPE_BF16 && t != AZ_TYPE_F16; }

// Whole 16-byte packs of a row.  The register forms hold up to 16384 elements in them, 16 to a thread of the largest workgroup.
int64_t norm_packs(int64_t cols, int32_t type) { return cols / (type == AZ_TYPE_F32 ? 4 : 8); }
bool norm_wide(int64_t cols, int32_t type) { return norm_packs(cols, type) > (type == AZ_TYPE_F32 ? 4096 : 2048); }

// Above 8192 elements the backward pass has no registers left for the sums over the rows: a pass of their own.
bool norm_sums_apart(int64_t cols, int32_t type) { return norm_packs(cols, type) > (type == AZ_TYPE_F32 ? 2048 : 1024); }

// Threads per row and packs per thread: the narrowest form that holds the row, one wave up to 256 packs.  (At least as many
// threads as there can be elements past the last whole pack.)  Forward, 1 M rows: 8 float32 columns 15 us with four threads to
// a row and 40 with sixteen, 32 bfloat16 columns 31 us with eight and 54 with sixteen.
template <typename T, typename Launch> void norm_form(int64_t packs, const Launch &launch)
{
    constexpr int NV = sizeof(T) == 4 ? 2 : 1;   // packs of 8 elements
    if constexpr (sizeof(T) == 4)
        if (packs <= 4) { launch.template operator()<T, 4, 1>(); return; }
    if (packs <= 8) launch.template operator()<T, 8, 1>();
    else if (packs <= 16) launch.template operator()<T, 16, 1>();
    else if (packs <= 32) launch.template operator()<T, 32, 1>();
    else if (packs <= 64) launch.template operator()<T, 64, 1>();
    else if (packs <= 128) launch.template operator()<T, 64, 2>();
    else if (packs <= 256) launch.template operator()<T, 64, 4>();
    else if (packs <= 512) launch.template operator()<T, 512 / NV, NV>();
    else if (packs <= 1024 && NV == 2) launch.template operator()<T, 1024 / NV, NV>();
    else if (packs <= 1024 * NV) launch.template operator()<T, 1024, NV>();
    else launch.template operator()<T, 1024, 2 * NV>();
}

// rows that a workgroup works on at a time, and its threads, by the same rule
int64_t norm_groups(int64_t packs, int32_t type)
{
    if (packs <= 4 && type == AZ_TYPE_F32) return 64;
    return packs <= 8 ? 32 : packs <= 16 ? 16 : packs <= 32 ? 8 : packs <= 256 ? 4 : 1;
}
int64_t norm_block(int64_t packs, int32_t type)
{
    const int64_t nv = type == AZ_TYPE_F32 ? 2 : 1;
    return packs <= 256 * nv ? 256 : packs <= 512 * nv ? 512 : 1024;
}

// Workgroups of a pass over many rows, each of which walks over its share of them.  More than the memory needs in flight only
// spread the accesses: rows of 256 float32 (whole cache lines) take 65 us with 1024 workgroups forward and 74 with 2048
// (185 k rows), 94 us backward with 768 and 96 with 1024.  Rows that end inside a line wait for each other's lines and want
// more: 361 16-bit columns, 100 k rows: 27 us with 2048 and 29 with 1024; backward 48 with 1024 and 53 with 768.  Forms with a
// workgroup to a row wait at its barriers and want all that fit (30 k rows of 2500 16-bit columns: 62 us with 1024, 77 with 512).
bool norm_lines(int64_t cols, int32_t type) { return cols * (type == AZ_TYPE_F32 ? 4 : 2) % 128 == 0; }

int64_t norm_fwd_blocks(int64_t cols, int32_t type)
{
    const int64_t packs = norm_packs(cols, type);
    if (norm_sums_apart(cols, type)) return 256;          // (as many as its registers leave room for)
    if (packs > 256) return 256 * 2048 / norm_block(packs, type);
    if (packs > 128 && type != AZ_TYPE_F32) return 768;   // (the same)
    return norm_lines(cols, type) ? 1024 : 2048;
}

int64_t norm_bwd_blocks(int64_t cols, int32_t type)
{
    const int64_t packs = norm_packs(cols, type);
    if (packs <= 64) return norm_lines(cols, type) ? 768 : 1024;
    if (packs <= 128) return 768;
    if (packs <= 256) return type == AZ_TYPE_F32 ? 512 : 256;
    return packs <= 512 ? 512 : 256;
}

// Of the eight L2 caches together.  What is larger is written, and read for the last time, past them: 256 float32 columns, 185 k
// rows, backward 94 us against 106; 4096 rows of 16384 bfloat16, backward 150 against 157.  (In some sizes it is the other way
// round, by less: 361 16-bit columns, 100 k rows, 48 us against 47; 1500 float32 columns, 100 k rows, 384 against 367.)
#define AZ_L2_BYTES (32 << 20)

template <typename Launch> void by_type(int32_t type, const Launch &launch)
{
    if (type == AZ_TYPE_F32) launch.template operator()<float>();
    else if (type == AZ_TYPE_BF16) launch.template operator()<__bf16>();
    else launch.template operator()<_Float16>();
}

// Chunks of a wide row where the rows alone would not give every compute unit a workgroup; 0: a workgroup to each row.
int64_t norm_chunks(int64_t rows, int64_t cols, int32_t type)
{
    return norm_wide(cols, type) && rows < 256 ? (cols + AZ_NORM_CHUNK - 1) / AZ_NORM_CHUNK : 0;
}

struct FwdForm {
    const NormFwd &a; hipStream_t st; int64_t packs; int32_t type;
    template <typename T, int TPR, int NV> void operator()() const
    {
        const int64_t groups = norm_groups(packs, type), blocks = (a.rows + groups - 1) / groups;
        k_layer_norm_fwd<T, TPR, NV><<<(unsigned)std::min(blocks, norm_fwd_blocks(a.cols, type)), norm_threads(TPR), 0, st>>>(a);
    }
};
struct FwdType {
    const NormFwd &a; float2 *part; hipStream_t st; int32_t type;
    template <typename T> void operator()() const
    {
        const int64_t chunks = norm_chunks(a.rows, a.cols, type);
        if (chunks) {
            const dim3 grid((unsigned)chunks, (unsigned)a.rows);
            k_layer_norm_chunk_stats<T><<<grid, AZ_NORM_WIDE_THREADS, 0, st>>>(a, part);
            k_layer_norm_chunk_write<T><<<grid, AZ_NORM_WIDE_THREADS, 0, st>>>(a, part);
        } else if (norm_wide(a.cols, type)) k_layer_norm_fwd_wide<T><<<(unsigned)std::min<int64_t>(a.rows, 2 * 256), AZ_NORM_WIDE_THREADS, 0, st>>>(a);
        else norm_form<T>(norm_packs(a.cols, type), FwdForm{a, st, norm_packs(a.cols, type), type});
    }
};

// Workgroups of the backward pass and how many rows of partial sums each of them leaves: functions of the sizes alone, so the
// order of the sums is the same on every call.  Four rows or more for each group of threads where there are rows enough,
// since every partial row is written and read again, but so many partial rows that no thread adds up more than 64 rows, or
// rows / 1024 if that is more.  With the groups' sums and the partial rows' added to that, a float32 sum over the rows is a
// chain of at most rows / 1024 + 96 additions in every form.
// (Several partial rows to a workgroup cost less than more workgroups: 40 000 rows of 8192 bfloat16 361 us and 414, 344
// with a chain of 157.)
struct BwdParts {
    int64_t blocks = 0, turns = 0, times = 1;     // a workgroup writes its sums after so many turns, so many times
    int64_t parts() const { return blocks * times; }
    BwdParts(int64_t rows, int64_t cols, int32_t type)
    {
        if (rows <= 0) return;
        const int64_t longest = std::max<int64_t>(64, (rows + 1023) / 1024);
        if (norm_sums_apart(cols, type)) { blocks = std::max(std::min<int64_t>(rows, 64), (rows + longest - 1) / longest); return; }
        const int64_t packs = norm_packs(cols, type), groups = norm_groups(packs, type), each = (rows + groups - 1) / groups;
        blocks = std::min(norm_bwd_blocks(cols, type), std::max((each + 3) / 4, std::min<int64_t>(each, 64)));
        turns = (each + blocks - 1) / blocks;
        if (groups > 1) return;      // (with several groups to a workgroup 1024 of them or more in all)
        times = (turns + longest - 1) / longest;
        turns = longest;
    }
};
int64_t bwd_parts(int64_t rows, int64_t cols, int32_t type) { return BwdParts(rows, cols, type).parts(); }

struct BwdForm {
    const NormBwd &a; hipStream_t st; int64_t grid;
    template <typename T, int TPR, int NV> void operator()() const
    {
        if constexpr (TPR * NV * Pack<T>::N > 8192) {
            const unsigned blocks = (unsigned)std::min<int64_t>(a.rows, 256);
            if (!a.dx) return;
            if (a.stream) k_layer_norm_bwd<T, TPR, NV, true, false><<<blocks, norm_threads(TPR), 0, st>>>(a);
            else k_layer_norm_bwd<T, TPR, NV, false, false><<<blocks, norm_threads(TPR), 0, st>>>(a);
        } else if (a.stream) k_layer_norm_bwd<T, TPR, NV, true, true><<<(unsigned)grid, norm_threads(TPR), 0, st>>>(a);
        else k_layer_norm_bwd<T, TPR, NV, false, true><<<(unsigned)grid, norm_threads(TPR), 0, st>>>(a);
    }
};
struct BwdType {
    const NormBwd &a; float2 *part; void *dw, *db; hipStream_t st; int32_t type;
    template <typename T> void operator()() const
    {
        const int64_t parts = a.parts;
        if (parts > 0) {
            const int64_t chunks = norm_chunks(a.rows, a.cols, type);
            // (the pass for dx comes after it: it is the last to read x and dy and may take them past the caches; 4096 rows of 16384
            // bfloat16 with the forward pass 200 us, the other way round 205, and 209 with dx first but through the caches)
            if (a.part && norm_sums_apart(a.cols, type))
                k_layer_norm_cols_wide<T><<<dim3((unsigned)((a.cols + 1023) / 1024), (unsigned)parts), AZ_NORM_COLS_WIDE_THREADS, 0, st>>>(a);
            if (!norm_wide(a.cols, type)) {
                norm_form<T>(norm_packs(a.cols, type), BwdForm{a, st, BwdParts(a.rows, a.cols, type).blocks});
            } else if (a.dx && chunks) {
                const dim3 grid((unsigned)chunks, (unsigned)a.rows);
                k_layer_norm_chunk_sums<T><<<grid, AZ_NORM_WIDE_THREADS, 0, st>>>(a, part);
                k_layer_norm_chunk_dx<T><<<grid, AZ_NORM_WIDE_THREADS, 0, st>>>(a, part);
            } else if (a.dx) {
                k_layer_norm_bwd_wide<T><<<(unsigned)std::min<int64_t>(a.rows, 2 * 256), AZ_NORM_WIDE_THREADS, 0, st>>>(a);
            }
        }
        if (dw || db)
            k_layer_norm_cols<T><<<dim3((unsigned)((a.cols + 15) / 16), 2), 1024, 0, st>>>(a.part, parts, a.cols, dw, db, a.affine_f32);
    }
};

int norm_sizes(int64_t rows, int64_t cols, int32_t type, int32_t affine_type, double eps)
{
    if (bad_type(type) || bad_type(affine_type)) return az_fail(AZ_ERR_ARG, "layer norm: unknown element type");
    if (affine_type != type && affine_type != AZ_TYPE_F32) return az_fail(AZ_ERR_ARG, "layer norm: weight and bias are float32 or of the input's type");
    // (a grid has less than 2^32 threads, of which the sums over the rows take 64 for each column)
    if (rows < 0 || cols < 1 || cols > ((int64_t)1 << 25) || rows > ((int64_t)1 << 50) / cols) return az_fail(AZ_ERR_ARG, "layer norm: bad number of rows or columns");
    if (!(eps >= 0.0)) return az_fail(AZ_ERR_ARG, "layer norm: eps must not be negative");
    return AZ_OK;
}

}  // namespace

extern "C" int64_t az_layer_norm_fwd_workspace(int32_t type, int64_t rows, int64_t cols)
{
    return rows < 1 || cols < 1 || bad_type(type) ? 0 : 2 * rows * norm_chunks(rows, cols, type);
}

extern "C" int az_layer_norm_fwd_dev(int32_t device, void *stream, int32_t type, int32_t affine_type, int64_t rows, int64_t cols, double eps,
                                     const void *x, int64_t x_stride, const void *weight, const void *bias, void *y, int64_t y_stride, float *mean, float *rstd,
                                     float *workspace, int64_t workspace_floats)
{
    const int rc = norm_sizes(rows, cols, type, affine_type, eps);
    if (rc) return rc;
    if (rows == 0) return AZ_OK;
    if (!x || !y) return az_fail(AZ_ERR_ARG, "layer norm: null array");
    if (!mean != !rstd) return az_fail(AZ_ERR_ARG, "layer norm: mean and rstd go together");
    const int64_t need = az_layer_norm_fwd_workspace(type, rows, cols);
    if (need > 0 && (!workspace || workspace_floats < need || (uintptr_t)workspace % 8)) return az_fail(AZ_ERR_ARG, "layer norm: workspace smaller than az_layer_norm_fwd_workspace, or not aligned to 8 bytes");
    if (x_stride < 0 || (y_stride < cols && rows > 1)) return az_fail(AZ_ERR_ARG, "layer norm: bad row stride");
    DeviceScope scope(device);
    if (scope.error != hipSuccess) return fail_hip("layer norm: device", scope.error);
    const NormFwd a{x, weight, bias, y, mean, rstd, rows, cols, x_stride, y_stride, (float)eps, affine_type == AZ_TYPE_F32,
                    rows * cols * (type == AZ_TYPE_F32 ? 4 : 2) > AZ_L2_BYTES};
    by_type(type, FwdType{a, reinterpret_cast<float2 *>(workspace), static_cast<hipStream_t>(stream), type});
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? AZ_OK : fail_hip("layer norm", e);
}

extern "C" int64_t az_layer_norm_bwd_workspace(int32_t type, int64_t rows, int64_t cols)
{
    return rows < 1 || cols < 1 || bad_type(type) ? 0 : 2 * rows * norm_chunks(rows, cols, type) + 2 * bwd_parts(rows, cols, type) * cols;
}

extern "C" int az_layer_norm_bwd_dev(int32_t device, void *stream, int32_t type, int32_t affine_type, int64_t rows, int64_t cols, const void *dy, int64_t dy_stride,
                                     const void *x, int64_t x_stride, const void *weight, const float *mean, const float *rstd, void *dx, int64_t dx_stride,
                                     void *dweight, void *dbias, float *workspace, int64_t workspace_floats)
{
    const int rc = norm_sizes(rows, cols, type, affine_type, 0.0);
    if (rc) return rc;
    if (rows > 0 && (!dy || !x || !mean || !rstd)) return az_fail(AZ_ERR_ARG, "layer norm backward: null array");
    if (dy_stride < 0 || x_stride < 0 || (dx && dx_stride < cols && rows > 1)) return az_fail(AZ_ERR_ARG, "layer norm backward: bad row stride");
    const bool sums = dweight || dbias;
    const int64_t chunk_floats = 2 * rows * norm_chunks(rows, cols, type);   // first in the workspace: pairs, so its start is aligned
    const int64_t need = sums ? az_layer_norm_bwd_workspace(type, rows, cols) : dx ? chunk_floats : 0;
    if (need > 0 && (!workspace || workspace_floats < need || (uintptr_t)workspace % 8)) return az_fail(AZ_ERR_ARG, "layer norm backward: workspace smaller than az_layer_norm_bwd_workspace, or not aligned to 8 bytes");
    if (!dx && !sums) return AZ_OK;
    DeviceScope scope(device);
    if (scope.error != hipSuccess) return fail_hip("layer norm backward: device", scope.error);
    const BwdParts plan(rows, cols, type);
    const NormBwd a{dy, x, weight, mean, rstd, dx, sums && need ? workspace + chunk_floats : nullptr, plan.parts(), plan.turns, plan.times, rows, cols, dy_stride, x_stride, dx_stride,
                    affine_type == AZ_TYPE_F32, rows * cols * (type == AZ_TYPE_F32 ? 4 : 2) > AZ_L2_BYTES};
    by_type(type, BwdType{a, reinterpret_cast<float2 *>(workspace), dweight, dbias, static_cast<hipStream_t>(stream), type});
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? AZ_OK : fail_hip("layer norm backward", e);
}

namespace {

struct Range {
    uintptr_t first, end;
    bool written;
    bool operator<(const Range &o) const { return first < o.first; }
};

// Every element that a step writes belongs to one tensor only, and no gradient lies where something is written: workgroups
// that share memory would race.  Gradients may share memory with each other.
bool overlap(std::vector<Range> &r)
{
    std::sort(r.begin(), r.end());
    uintptr_t read_end = 0, write_end = 0;   // of the ranges that start at or before the present one
    for (const Range &x : r) {
        if (x.first < write_end || (x.written && x.first < read_end)) return true;
        uintptr_t &end = x.written ? write_end : read_end;
        end = std::max(end, x.end);
    }
    return false;
}

struct AdamwType {
    const AdamwTable &t; const AdamwScalars &k; unsigned blocks; bool eight; int turns; hipStream_t st;
    template <typename T> void operator()() const
    {
        if (eight) {
            if (turns == 1) k_adamw_8<T, 1, false><<<blocks, AZ_ADAMW_THREADS, 0, st>>>(t, k);
            else k_adamw_8<T, 4, true><<<blocks, AZ_ADAMW_THREADS, 0, st>>>(t, k);
        } else {
            if (turns == 1) k_adamw_32<T, 1, false><<<blocks, AZ_ADAMW_THREADS, 0, st>>>(t, k);
            else if (turns == 2) k_adamw_32<T, 2, false><<<blocks, AZ_ADAMW_THREADS, 0, st>>>(t, k);
            else k_adamw_32<T, 4, true><<<blocks, AZ_ADAMW_THREADS, 0, st>>>(t, k);
        }
    }
};

int adamw_step(int32_t device, void *stream, int64_t tensors, void *const *params, const void *const *grads, void *const *m, void *const *v, float *const *m_scales,
               float *const *v_scales, const int64_t *numels, int32_t type, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step)
{
    if (tensors < 0 || (tensors > 0 && (!params || !grads || !m || !v || !numels))) return az_fail(AZ_ERR_ARG, "adamw: null table");
    if (bad_type(type)) return az_fail(AZ_ERR_ARG, "adamw: unknown element type");
    if (!m_scales != !v_scales) return az_fail(AZ_ERR_ARG, "adamw: the scales of both states or of neither");
    if (!(lr >= 0.0) || !(eps >= 0.0) || !(weight_decay >= 0.0)) return az_fail(AZ_ERR_ARG, "adamw: lr, eps and weight_decay must not be negative");
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return az_fail(AZ_ERR_ARG, "adamw: betas must lie in [0, 1)");
    if (step < 1) return az_fail(AZ_ERR_ARG, "adamw: steps are counted from 1");
    const bool eight = m_scales != nullptr;
    const int64_t size = type == AZ_TYPE_F32 ? 4 : 2;
    std::vector<Range> ranges;
    ranges.reserve((size_t)tensors * (eight ? 6 : 4));
    int64_t total = 0;
    for (int64_t i = 0; i < tensors; i++) {
        const int64_t n = numels[i];
        if (n < 0 || n > ((int64_t)1 << 33)) return az_fail(AZ_ERR_ARG, "adamw: bad tensor size");
        if (n == 0) continue;
        if (!params[i] || !grads[i] || !m[i] || !v[i] || (eight && (!m_scales[i] || !v_scales[i]))) return az_fail(AZ_ERR_ARG, "adamw: null tensor");
        const auto add = [&](const void *p, int64_t bytes, bool written = true) { ranges.push_back(Range{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, written}); };
        add(grads[i], n * size, false);
        add(params[i], n * size);
        add(m[i], eight ? n : n * 4);
        add(v[i], eight ? n : n * 4);
        if (eight) {
            add(m_scales[i], (n + AZ_ADAMW_BLOCK - 1) / AZ_ADAMW_BLOCK * 4);
            add(v_scales[i], (n + AZ_ADAMW_BLOCK - 1) / AZ_ADAMW_BLOCK * 4);
        }
        total += n;
    }
    if (total == 0) return AZ_OK;
    if (overlap(ranges)) return az_fail(AZ_ERR_ARG, "adamw: two tensors share memory that the step writes");
    DeviceScope scope(device);
    if (scope.error != hipSuccess) return fail_hip("adamw: device", scope.error);
    AdamwScalars k;
    k.beta1 = beta1; k.beta2 = beta2; k.one_minus_beta1 = 1.0 - beta1; k.one_minus_beta2 = 1.0 - beta2;
    k.decay = (float)(lr * weight_decay);
    k.step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    k.inv_sqrt_c2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    k.eps = eps > 0.0 ? std::max((float)eps, 1.17549435e-38f) : 0.f;   // (subnormal numbers do not survive the reciprocal)
    k.tiny = !(k.inv_sqrt_c2 * 1.1e-19f < k.eps * 0x1p-25f);   // 1.1e-19: the root of the smallest normal number
    // What fits the 256 MB memory-side cache is still there at the next step (9 M float32 parameters, 252 MB: 40 us, past the
    // caches 45); what does not only gets in its own way (24 M: 126 us through the caches, 112 past them; with 8-bit state 75
    // and 62).
    const bool stream_past = total * (3 * size + (eight ? 4 : 16)) > ((int64_t)256 << 20);
    AdamwTable t;
    for (int64_t i = 0; i < tensors;) {
        // a launch is full at 64 tensors, or when its threads would no longer fit a grid (less than 2^32)
        int held = 0;
        int64_t elements = 0, widest = 0;
        for (; i < tensors && held < AZ_ADAMW_TENSORS; i++) {
            const int64_t n = numels[i];
            if (n == 0) continue;
            if (held && widest + n / 1024 + 1 > 0xffffff) break;
            widest += n / 1024 + 1;
            elements += n;
            t.param[held] = params[i]; t.grad[held] = grads[i]; t.m[held] = m[i]; t.v[held] = v[i];
            t.m_scale[held] = eight ? m_scales[i] : nullptr; t.v_scale[held] = eight ? v_scales[i] : nullptr;
            t.n[held++] = n;
        }
        if (!held) break;
        // Packs of four elements to a thread.  Small launches want many workgroups (1 M: 5.4 us with one pack, 5.8 with two; 4 M:
        // 18.2 and 17.8), launches with 8-bit state, which wait for arithmetic too, at any size (2 M: 9.0 and 9.6).
        const int turns = elements <= ((int64_t)1 << 20) ? 1 : stream_past ? 4 : eight ? 1 : 2;
        const int64_t chunk = turns * 4 * AZ_ADAMW_THREADS;
        uint32_t blocks = 0;
        for (int j = 0; j < AZ_ADAMW_TENSORS; j++) t.last[j] = j < held ? blocks += (uint32_t)((t.n[j] + chunk - 1) / chunk) : 0xffffffffu;
        by_type(type, AdamwType{t, k, blocks, eight, turns, static_cast<hipStream_t>(stream)});
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return fail_hip("adamw", e);
    }
    return AZ_OK;
}

}  // namespace

extern "C" int az_adamw_step_dev(int32_t device, void *stream, int64_t tensors, void *const *params, const void *const *grads, void *const *exp_avg,
                                 void *const *exp_avg_sq, float *const *exp_avg_scale, float *const *exp_avg_sq_scale, const int64_t *numels, int32_t type,
                                 double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step)
{
    try {
        return adamw_step(device, stream, tensors, params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, numels, type, lr, beta1, beta2, eps, weight_decay, step);
    } catch (...) {   // (the list of ranges could not be allocated: nothing has been launched)
        return az_fail(AZ_ERR_ARG, "adamw: out of host memory");
    }
}

extern "C" int az_dequantize_state_dev(int32_t device, void *stream, const void *codes, const float *scales, int64_t n, int32_t is_signed, float *out)
{
    if (n < 0 || n > ((int64_t)1 << 40)) return az_fail(AZ_ERR_ARG, "dequantize: bad size");
    if (n == 0) return AZ_OK;
    if (!codes || !scales || !out) return az_fail(AZ_ERR_ARG, "dequantize: null array");
    DeviceScope scope(device);
    if (scope.error != hipSuccess) return fail_hip("dequantize: device", scope.error);
    const int64_t per = AZ_ADAMW_THREADS * 4;
    const unsigned blocks = (unsigned)std::min<int64_t>((n + per - 1) / per, 16 * 256);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const uint8_t *c = static_cast<const uint8_t *>(codes);
    if (is_signed) k_dequantize_state<true><<<blocks, AZ_ADAMW_THREADS, 0, st>>>(c, scales, n, out);
    else k_dequantize_state<false><<<blocks, AZ_ADAMW_THREADS, 0, st>>>(c, scales, n, out);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? AZ_OK : fail_hip("dequantize", e);
}
