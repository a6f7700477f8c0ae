// Element types and vector loads shared by the training kernels (az_norm_kernels.h, az_adamw_kernels.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// Four elements of T as one load or store.  The alignment asked for is that of one element only: rows of odd length and
// views into larger buffers start anywhere, and gfx950 takes a wide global access at any address (an unaligned one costs
// at most one more cache line).
template <typename T> struct Vec4 { typedef T type __attribute__((ext_vector_type(4))); };
template <typename T> struct __attribute__((packed, aligned(alignof(T)))) Packed4 { typename Vec4<T>::type v; };

template <typename T> __device__ __forceinline__ float4 load4(const T *p)
{
    const auto v = reinterpret_cast<const Packed4<T> *>(p)->v;
    return make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]);
}

// every conversion to 16 bits rounds to nearest even, once, from the float32 result
template <typename T> __device__ __forceinline__ void store4(T *p, float4 f)
{
    Packed4<T> out;
    out.v = typename Vec4<T>::type{(T)f.x, (T)f.y, (T)f.z, (T)f.w};
    *reinterpret_cast<Packed4<T> *>(p) = out;
}

// elements i .. i+3 of a run of n (those past its end are 0 / are not written)
template <typename T> __device__ __forceinline__ float4 load4(const T *p, int64_t i, int64_t n)
{
    if (i + 4 <= n) return load4(p + i);
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n) f.x = (float)p[i];
    if (i + 1 < n) f.y = (float)p[i + 1];
    if (i + 2 < n) f.z = (float)p[i + 2];
    return f;
}

template <typename T> __device__ __forceinline__ void store4(T *p, int64_t i, int64_t n, float4 f)
{
    if (i + 4 <= n) { store4(p + i, f); return; }
    if (i < n) p[i] = (T)f.x;
    if (i + 1 < n) p[i + 1] = (T)f.y;
    if (i + 2 < n) p[i + 2] = (T)f.z;
}

template <int CTRL> __device__ __forceinline__ uint32_t dpp_row(uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
#define AZ_ROW_ROR(n) (0x120 + (n))   // DPP row_ror: rotation within 16 lanes

// Sum over the 16 lanes of a DPP row, in every lane, the same bits in all of them (each step adds the same two partial
// sums in both of the lanes that hold them).
__device__ __forceinline__ float row16_sum(float x)
{
    x += __uint_as_float(dpp_row<AZ_ROW_ROR(8)>(__float_as_uint(x)));
    x += __uint_as_float(dpp_row<AZ_ROW_ROR(4)>(__float_as_uint(x)));
    x += __uint_as_float(dpp_row<AZ_ROW_ROR(2)>(__float_as_uint(x)));
    x += __uint_as_float(dpp_row<AZ_ROW_ROR(1)>(__float_as_uint(x)));
    return x;
}

__device__ __forceinline__ float lane_value(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }

// Sum over a wave's 64 lanes, in every lane; needs all lanes active.
__device__ __forceinline__ float wave_sum(float x)
{
    x = row16_sum(x);
    return (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
}

// Largest of 64 unsigned values, in every lane; needs all lanes active.
__device__ __forceinline__ uint32_t wave_umax(uint32_t x)
{
    x = max(x, dpp_row<AZ_ROW_ROR(8)>(x));
    x = max(x, dpp_row<AZ_ROW_ROR(4)>(x));
    x = max(x, dpp_row<AZ_ROW_ROR(2)>(x));
    x = max(x, dpp_row<AZ_ROW_ROR(1)>(x));
    const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
    const uint32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
    return max(max(a, b), max(c, d));
}
