// vec.cuh — pairs of float32 in one register, and runs of consecutive elements (float32 or bfloat16, chosen at compile time) between global memory and
// float registers: one or two 16-byte accesses where the caller has checked the alignment, single elements
// otherwise.
#pragma once

#include "common.cuh"

namespace dc {

__host__ __device__ __forceinline__ bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

namespace vec {

// Pairs of float32 in one instruction (both lanes rounded as the single forms round them).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// p[first * stride] + p[(first + step) * stride] + .. below `lines`, in order, eight loads under way together whatever their
// number (an unrolled loop does its last few one by one: 2 us for the 50 lines of 6 x 2049 x 1536 in the convolution).
__device__ __forceinline__ float sum_lines(const float *p, int64_t first, int64_t lines, int64_t step, int64_t stride) {
    constexpr int kBatch = 8;
    float v = 0.f;
    for (int64_t i = first; i < lines; i += kBatch * step) {
        float x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) x[k] = i + k * step < lines ? p[(i + k * step) * stride] : 0.f;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) v += x[k];
    }
    return v;
}


// `n` of N elements from p (the others 0).  ALIGNED: p is aligned to the run's size (16 bytes at most) and n == N.
template <bool ALIGNED, int N>
__device__ __forceinline__ void load(const float *p, float (&v)[N], int n = N) {
    if constexpr (ALIGNED && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 t = *reinterpret_cast<const float4 *>(p + i);
            v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
        }
    } else if constexpr (ALIGNED && N == 2) {
        const float2 t = *reinterpret_cast<const float2 *>(p);
        v[0] = t.x, v[1] = t.y;
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
    } else if constexpr (ALIGNED && N == 2) {
        unpack(*reinterpret_cast<const uint32_t *>(p), v[0], v[1]);
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
    } else if constexpr (ALIGNED && N == 2) {
        *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
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
    } else if constexpr (ALIGNED && N == 2) {
        *reinterpret_cast<uint32_t *>(p) = pack(v[0], v[1]);
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

// N elements as they are in memory, to be converted later: loads in flight take the registers of the type, not of float32.
template <typename T, int N>
struct Raw {
    uint32_t w[N * sizeof(T) / 4];
};
template <bool ALIGNED, typename T, int N>
__device__ __forceinline__ void load_raw(const T *p, Raw<T, N> &r, int n) {
    constexpr int kWords = N * sizeof(T) / 4;
    if constexpr (ALIGNED && kWords % 4 == 0) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i / 4];
            r.w[i] = v.x, r.w[i + 1] = v.y, r.w[i + 2] = v.z, r.w[i + 3] = v.w;
        }
    } else {
        static_assert(!ALIGNED, "aligned runs are whole 16-byte accesses");
        T v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            dc::st(&v[i], 0.f);
            if (i < n) v[i] = p[i];
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) r.w[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const __nv_bfloat162 b = __halves2bfloat162(v[i], v[i + 1]);
                r.w[i / 2] = *reinterpret_cast<const uint32_t *>(&b);
            }
        }
    }
}
// pair i (elements 2 i and 2 i + 1)
template <typename T, int N>
__device__ __forceinline__ float2 pair_of(const Raw<T, N> &r, int i) {
    float2 f;
    if constexpr (sizeof(T) == 4) f = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    else unpack(r.w[i], f.x, f.y);
    return f;
}

}  // namespace vec
}  // namespace dc
