// Storage types of the operators that take fp32 or bf16 (HIPGPT_TYPE_*): 16 bytes of either as fp32 values and back.
#pragma once

#include "tc_primitives.cuh"

#include <cuda_bf16.h>

#include <initializer_list>

namespace hipgpt {

template <typename T> constexpr int kPer16 = 16 / (int)sizeof(T);      // values in 16 bytes

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// W consecutive values: 16 bytes (or 32 of fp32 results of 16-bit inputs) at a time where W fills them, else one by one
template <int W>
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[W], float)
{
    static_assert(W == 4, "16 bytes of fp32");
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
}
template <int W>
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[W], __nv_bfloat16)
{
    static_assert(W == 8, "16 bytes of bf16");
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

template <typename T, int W>
__device__ __forceinline__ void load_values(const T *p, float (&v)[W])
{
    if constexpr (W == 1) {
        v[0] = to_float(*p);
    } else if constexpr (W * sizeof(T) == 16) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        unpack(u, v, T());
    } else if constexpr (W * sizeof(T) == 8) {
        static_assert(sizeof(T) == 2, "four of bf16");
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xFFFF0000u);
        v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xFFFF0000u);
    } else {
        static_assert(W * sizeof(T) == 32 && sizeof(T) == 4, "whole 16-byte words");
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
}

template <typename T, int W>
__device__ __forceinline__ void store_values(T *p, const float (&v)[W])
{
    if constexpr (W == 1) {
        *p = from_float<T>(v[0]);
    } else if constexpr (sizeof(T) == 2 && W == 4) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    } else if constexpr (sizeof(T) == 2) {
        static_assert(W == 8, "16 bytes of bf16");
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) reinterpret_cast<float4 *>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
}

inline bool ranges_overlap(const void *a, size_t na, const void *b, size_t nb)
{
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    return a0 < b0 + nb && b0 < a0 + na;
}

// A call's arrays; the first `outputs` of them are written
struct Extent { const void *at; size_t bytes; };
inline int refuse_overlaps(int outputs, std::initializer_list<Extent> arrays)
{
    int i = 0;
    for (const Extent *a = arrays.begin(); a != arrays.end() && i < outputs; ++a, ++i)
        for (const Extent *b = a + 1; b != arrays.end(); ++b)
            if (a->at && b->at && a->bytes && b->bytes && ranges_overlap(a->at, a->bytes, b->at, b->bytes)) return fail(HIPGPT_ERR_BAD_ARG, "an output overlaps another of the call's arrays");
    return HIPGPT_OK;
}

inline bool all_aligned16(std::initializer_list<const void *> ps)
{
    uintptr_t all = 0;
    for (const void *p : ps) all |= reinterpret_cast<uintptr_t>(p);
    return (all & 15) == 0;
}

}  // namespace hipgpt
