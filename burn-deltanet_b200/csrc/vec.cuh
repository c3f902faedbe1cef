// vec.cuh — runs of consecutive elements (float32 or bfloat16, chosen at compile time) between global memory and
// float registers: one or two 16-byte accesses where the caller has checked the alignment, single elements
// otherwise.
#pragma once

#include "common.cuh"

namespace dc {

__host__ __device__ __forceinline__ bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

namespace vec {

// `n` of N elements from p (the others 0).  ALIGNED: p is aligned to the run's size (16 bytes at most) and n == N.
template <bool ALIGNED, int N>
__device__ __forceinline__ void load(const float *p, float (&v)[N], int n = N) {
    if constexpr (ALIGNED && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 t = *reinterpret_cast<const float4 *>(p + i);
            v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? p[i] : 0.f;
    }
}
__device__ __forceinline__ void unpack(uint32_t w, float &lo, float &hi) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
    lo = f.x, hi = f.y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}
template <bool ALIGNED, int N>
__device__ __forceinline__ void load(const __nv_bfloat16 *p, float (&v)[N], int n = N) {
    if constexpr (ALIGNED && N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const uint4 t = *reinterpret_cast<const uint4 *>(p + i);
            unpack(t.x, v[i], v[i + 1]), unpack(t.y, v[i + 2], v[i + 3]);
            unpack(t.z, v[i + 4], v[i + 5]), unpack(t.w, v[i + 6], v[i + 7]);
        }
    } else if constexpr (ALIGNED && N == 4) {
        const uint2 t = *reinterpret_cast<const uint2 *>(p);
        unpack(t.x, v[0], v[1]), unpack(t.y, v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
    }
}
template <bool ALIGNED, int N>
__device__ __forceinline__ void store(float *p, const float (&v)[N], int n = N) {
    if constexpr (ALIGNED && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = v[i];
    }
}
template <bool ALIGNED, int N>
__device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&v)[N], int n = N) {
    if constexpr (ALIGNED && N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 8)
            *reinterpret_cast<uint4 *>(p + i) = make_uint4(pack(v[i], v[i + 1]), pack(v[i + 2], v[i + 3]),
                                                           pack(v[i + 4], v[i + 5]), pack(v[i + 6], v[i + 7]));
    } else if constexpr (ALIGNED && N == 4) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack(v[0], v[1]), pack(v[2], v[3]));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = __float2bfloat16_rn(v[i]);
    }
}
// the same with the element type chosen at run time (0: float32, 1: bfloat16; uniform over the launch)
template <bool ALIGNED, int N>
__device__ __forceinline__ void load_as(int dtype, const void *p, int64_t at, float (&v)[N], int n = N) {
    if (dtype) load<ALIGNED>(static_cast<const __nv_bfloat16 *>(p) + at, v, n);
    else load<ALIGNED>(static_cast<const float *>(p) + at, v, n);
}
template <bool ALIGNED, int N>
__device__ __forceinline__ void store_as(int dtype, void *p, int64_t at, const float (&v)[N], int n = N) {
    if (dtype) store<ALIGNED>(static_cast<__nv_bfloat16 *>(p) + at, v, n);
    else store<ALIGNED>(static_cast<float *>(p) + at, v, n);
}

}  // namespace vec
}  // namespace dc
