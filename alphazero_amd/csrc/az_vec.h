// Element types and vector loads shared by the training kernels (az_norm_kernels.h, az_adamw_kernels.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// Four elements of T as one load or store.  The alignment asked for is that of one element only: rows of odd length and
// views into larger buffers start anywhere, and gfx950 takes a wide global access at any address (an unaligned one costs
// at most one more cache line).
template <typename T> struct Vec4 {
    typedef T type __attribute__((ext_vector_type(4)));
    typedef type any __attribute__((aligned(alignof(T))));
};

// STREAM: past the caches, for what will not be read again before something else has taken its place in them
template <bool STREAM = false, typename T> __device__ __forceinline__ float4 load4(const T *p)
{
    const typename Vec4<T>::any *from = reinterpret_cast<const typename Vec4<T>::any *>(p);
    typename Vec4<T>::type v;
    if constexpr (STREAM) v = __builtin_nontemporal_load(from);
    else v = *from;
    return make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]);
}

// every conversion to 16 bits rounds to nearest even, once, from the float32 result
template <bool STREAM = false, typename T> __device__ __forceinline__ void store4(T *p, float4 f)
{
    const typename Vec4<T>::type v = {(T)f.x, (T)f.y, (T)f.z, (T)f.w};
    typename Vec4<T>::any *to = reinterpret_cast<typename Vec4<T>::any *>(p);
    if constexpr (STREAM) __builtin_nontemporal_store(v, to);
    else *to = v;
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

// As many neighbouring elements as one 16-byte access holds (4 of float32, 8 of 16 bits), as they lie in memory.
template <typename T> struct Pack {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(N)));
    typedef type any __attribute__((aligned(alignof(T))));   // at any element's address
};

template <bool STREAM, typename T> __device__ __forceinline__ typename Pack<T>::type load_pack(const T *p)
{
    const typename Pack<T>::any *from = reinterpret_cast<const typename Pack<T>::any *>(p);
    if constexpr (STREAM) return __builtin_nontemporal_load(from);
    else return *from;
}

template <typename T> __device__ __forceinline__ void store_pack(T *p, const float (&f)[Pack<T>::N], bool stream)
{
    typename Pack<T>::type out;
#pragma unroll
    for (int e = 0; e < Pack<T>::N; e++) out[e] = (T)f[e];
    typename Pack<T>::any *to = reinterpret_cast<typename Pack<T>::any *>(p);
    if (stream) __builtin_nontemporal_store(out, to);
    else *to = out;
}

template <int CTRL> __device__ __forceinline__ uint32_t dpp_row(uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
#define AZ_ROW_ROR(n) (0x120 + (n))   // DPP row_ror: rotation within 16 lanes

#define AZ_QUAD_XOR1 0xb1               // DPP quad_perm 1,0,3,2
#define AZ_QUAD_XOR2 0x4e               // DPP quad_perm 2,3,0,1
#define AZ_QUAD_FIRST 0x00              // DPP quad_perm 0,0,0,0
#define AZ_ROW_LANE(n) (0x150 + (n))    // DPP row_newbcast: lane n of 16 in all of them
#define AZ_ROW_HALF_MIRROR 0x141        // DPP row_half_mirror: lane i of eight takes lane 7 - i

// Sums over 4 and 8 neighbouring lanes and over the 16 lanes of a DPP row, in every lane, the same bits in all of them (each step adds the same two partial
// sums in both of the lanes that hold them).
__device__ __forceinline__ float quad_sum(float x)
{
    x += __uint_as_float(dpp_row<AZ_QUAD_XOR1>(__float_as_uint(x)));
    x += __uint_as_float(dpp_row<AZ_QUAD_XOR2>(__float_as_uint(x)));
    return x;
}
__device__ __forceinline__ float oct_sum(float x)
{
    x = quad_sum(x);
    return x + __uint_as_float(dpp_row<AZ_ROW_HALF_MIRROR>(__float_as_uint(x)));
}
__device__ __forceinline__ float row16_sum(float x)
{
    x += __uint_as_float(dpp_row<AZ_ROW_ROR(8)>(__float_as_uint(x)));
    x += __uint_as_float(dpp_row<AZ_ROW_ROR(4)>(__float_as_uint(x)));
    x += __uint_as_float(dpp_row<AZ_ROW_ROR(2)>(__float_as_uint(x)));
    x += __uint_as_float(dpp_row<AZ_ROW_ROR(1)>(__float_as_uint(x)));
    return x;
}

// gfx950's row swaps hand every lane the values of both rows (or both halves) of a pair, in the same order: what is added up
// from them has the same bits in all lanes.
__device__ __forceinline__ float add_row_pairs(float x)     // lane i of rows 2j and 2j+1: x of row 2j + x of row 2j+1
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_halves(float x)        // lane i of both halves of the wave
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sum over groups of 32 neighbouring lanes / over a wave's 64, in every lane; needs all lanes active.
__device__ __forceinline__ float half_sum(float x) { return add_row_pairs(row16_sum(x)); }
__device__ __forceinline__ float wave_sum(float x) { return add_halves(half_sum(x)); }

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
