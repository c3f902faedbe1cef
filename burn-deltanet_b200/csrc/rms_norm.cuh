// rms_norm.cuh — the residual stream's addition with the RMS norm of the sum, and its backward.
//
//   forward   s = x + residual;  y = s w / sqrt(mean(s^2) + eps);  optionally y as e4m3 with scales
//   backward  with inv = 1 / sqrt(mean(r^2) + eps) of the stored sum r, and m = mean(w dy r):
//             d = inv w dy - r inv^3 m + d_r,  d_w = sum over rows of dy r inv
//
// HBM-bound: the forward reads x and the residual and writes the sum and y once, the backward reads dy, d_r and r
// and writes d once; the row stays in registers between the reduction and its use.  A row is spread over TPR
// threads (a power of two, 32 to 1024), eight consecutive columns per access, VPT accesses per thread; narrow
// rows share a CTA.  The inverse root is recomputed in the backward from the row it reads anyway, so the forward
// saves nothing beside r.
#pragma once

#include <cuda_fp8.h>
#include <float.h>

#include "common.cuh"
#include "vec.cuh"

namespace dc {
namespace rms {

constexpr int kVec = 8;  // columns per access

struct Params {
    int64_t rows;
    int32_t width, group;  // group: columns per scale (e4m3), 0 = the whole row
    int64_t x_stride, rin_stride, rout_stride, y_stride;
    int32_t x_dt, r_dt, y_dt;  // 0 float32, 1 bfloat16
    float eps;
    const void *x, *rin;
    const float *weight;
    void *rout, *y;
    float *scale;
};

// Sum (or maximum) over the TPR threads of a row; every thread of the CTA calls it.  `red` holds one float per warp.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, int tpr, float *red) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, w) : v + w;
    }
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tpr >> 5, first = warp & ~(per - 1);
    __syncthreads();  // the last reduction's values have been read
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    v = red[first];
    for (int i = 1; i < per; ++i) v = MAX ? fmaxf(v, red[first + i]) : v + red[first + i];
    return v;
}

// e4m3 values of v[i] * inv in one 8-byte word
__device__ __forceinline__ uint2 to_e4m3(const float (&v)[kVec], float inv) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
        w[i] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    return make_uint2(w[0], w[1]);
}

// ALIGNED: width a multiple of 8 and every row of every tensor 16-byte aligned (8-byte for e4m3).
template <int VPT, bool ALIGNED, bool F8>
__global__ void rms_norm_kernel(const Params p, int tpr) {
    __shared__ float red[32];
    const int tx = threadIdx.x & (tpr - 1), ty = threadIdx.x / tpr;
    const int rows_per_cta = blockDim.x / tpr;
    const float inv_width = 1.f / (float)p.width;
    int n[VPT];  // columns of each access inside the row
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int left = p.width - (tx + i * tpr) * kVec;
        n[i] = left < 0 ? 0 : left > kVec ? kVec : left;
    }
    // every thread takes the same number of rounds, for the barriers in row_reduce
    for (int64_t row0 = (int64_t)blockIdx.x * rows_per_cta; row0 < p.rows; row0 += (int64_t)gridDim.x * rows_per_cta) {
        const int64_t row = row0 + ty;
        const bool on = row < p.rows;
        float s[VPT][kVec];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int col = (tx + i * tpr) * kVec;
            float r[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) s[i][e] = 0.f, r[e] = 0.f;
            if (on && n[i] > 0) {
                vec::load_as<ALIGNED>(p.x_dt, p.x, row * p.x_stride + col, s[i], n[i]);
                if (p.rin) vec::load_as<ALIGNED>(p.r_dt, p.rin, row * p.rin_stride + col, r, n[i]);
            }
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                s[i][e] += r[e];
                ss = fmaf(s[i][e], s[i][e], ss);
            }
        }
        if (p.rout && on) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (n[i] > 0) vec::store_as<ALIGNED>(p.r_dt, p.rout, row * p.rout_stride + (tx + i * tpr) * kVec, s[i], n[i]);
        }
        ss = row_reduce<false>(ss, tpr, red);
        const float inv = 1.f / sqrtf(fmaf(ss, inv_width, p.eps));
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            if (n[i] > 0) {
                float w[kVec];
                vec::load<ALIGNED>(p.weight + (tx + i * tpr) * kVec, w, n[i]);
#pragma unroll
                for (int e = 0; e < kVec; ++e) s[i][e] *= inv * w[e];
            }
        }
        if constexpr (!F8) {
            if (on) {
#pragma unroll
                for (int i = 0; i < VPT; ++i)
                    if (n[i] > 0) vec::store_as<ALIGNED>(p.y_dt, p.y, row * p.y_stride + (tx + i * tpr) * kVec, s[i], n[i]);
            }
        } else {
            uint8_t *Y = static_cast<uint8_t *>(p.y);
            float amax[VPT], all = 0.f;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                amax[i] = 0.f;  // fmaxf drops a NaN: its row is NaN throughout, and keeps scale 1
#pragma unroll
                for (int e = 0; e < kVec; ++e) amax[i] = fmaxf(amax[i], fabsf(s[i][e]));
                all = fmaxf(all, amax[i]);
            }
            const int lanes = p.group ? p.group / kVec : 0;  // lanes of a group: 4 .. 32, a power of two
            if (lanes) {
#pragma unroll
                for (int i = 0; i < VPT; ++i)
                    for (int o = lanes / 2; o >= 1; o >>= 1) amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], o));
            } else {
                all = row_reduce<true>(all, tpr, red);
#pragma unroll
                for (int i = 0; i < VPT; ++i) amax[i] = all;
            }
            if (on) {
#pragma unroll
                for (int i = 0; i < VPT; ++i) {
                    if (n[i] <= 0) continue;
                    const int v = tx + i * tpr;
                    const float scale = amax[i] > 0.f ? fmaxf(amax[i] * (1.f / 448.f), FLT_MIN) : 1.f;
                    if (lanes) {
                        if (v % lanes == 0) p.scale[row * (p.width / p.group) + v / lanes] = scale;
                    } else if (v == 0) {
                        p.scale[row] = scale;
                    }
                    const uint2 q = to_e4m3(s[i], 1.f / scale);
                    uint8_t *o = Y + row * p.y_stride + v * kVec;
                    if constexpr (ALIGNED) {
                        *reinterpret_cast<uint2 *>(o) = q;
                    } else {
#pragma unroll
                        for (int e = 0; e < kVec; ++e)
                            if (e < n[i]) o[e] = (uint8_t)((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
                    }
                }
            }
        }
    }
}

struct BwdParams {
    int64_t rows;
    int32_t width;
    int64_t dy_stride, dr_stride, r_stride, dx_stride, dres_stride;
    int32_t y_dt, r_dt, x_dt;
    float eps;
    const void *dy, *dr, *r;
    const float *weight;
    void *dx, *dres;
    float *part;  // [gridDim.x, width] partial sums of d_weight, or null
};

// Persistent CTAs: each keeps its rows' share of d_weight in registers and writes it once, to its own line of
// `part` (column_sum_kernel adds the lines in order).
template <int VPT, bool ALIGNED>
__global__ void __launch_bounds__(512) rms_norm_bwd_kernel(const BwdParams p, int tpr) {
    __shared__ float red[32];
    extern __shared__ float lines[];  // [rows per CTA - 1][width], when several rows share the CTA
    const int tx = threadIdx.x & (tpr - 1), ty = threadIdx.x / tpr;
    const int rows_per_cta = blockDim.x / tpr;
    const float inv_width = 1.f / (float)p.width;
    int n[VPT];
    float dw[VPT][kVec];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int left = p.width - (tx + i * tpr) * kVec;
        n[i] = left < 0 ? 0 : left > kVec ? kVec : left;
#pragma unroll
        for (int e = 0; e < kVec; ++e) dw[i][e] = 0.f;
    }
    for (int64_t row0 = (int64_t)blockIdx.x * rows_per_cta; row0 < p.rows; row0 += (int64_t)gridDim.x * rows_per_cta) {
        const int64_t row = row0 + ty;
        const bool on = row < p.rows;
        float r[VPT][kVec], g[VPT][kVec];
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) r[i][e] = 0.f, g[i][e] = 0.f;
            if (on && n[i] > 0) {
                const int col = (tx + i * tpr) * kVec;
                vec::load_as<ALIGNED>(p.r_dt, p.r, row * p.r_stride + col, r[i], n[i]);
                vec::load_as<ALIGNED>(p.y_dt, p.dy, row * p.dy_stride + col, g[i], n[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float w[kVec];
            if (n[i] > 0) vec::load<ALIGNED>(p.weight + (tx + i * tpr) * kVec, w, n[i]);
            if (on && n[i] > 0) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    ss = fmaf(r[i][e], r[i][e], ss);
                    dot = fmaf(w[e] * g[i][e], r[i][e], dot);
                }
            }
        }
        ss = row_reduce<false>(ss, tpr, red);
        dot = row_reduce<false>(dot, tpr, red);
        const float inv = 1.f / sqrtf(fmaf(ss, inv_width, p.eps));
        const float back = inv * inv * inv * (dot * inv_width);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            if (!on || n[i] <= 0) continue;
            const int col = (tx + i * tpr) * kVec;
            float w[kVec], d[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) d[e] = 0.f;
            if (p.dr) vec::load_as<ALIGNED>(p.r_dt, p.dr, row * p.dr_stride + col, d, n[i]);
            vec::load<ALIGNED>(p.weight + col, w, n[i]);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                dw[i][e] = fmaf(g[i][e], r[i][e] * inv, dw[i][e]);
                d[e] += fmaf(inv * w[e], g[i][e], -r[i][e] * back);
            }
            if (p.dx) vec::store_as<ALIGNED>(p.x_dt, p.dx, row * p.dx_stride + col, d, n[i]);
            if (p.dres) vec::store_as<ALIGNED>(p.r_dt, p.dres, row * p.dres_stride + col, d, n[i]);
        }
    }
    if (!p.part) return;
    // rows that share the CTA: row group 0 adds the others' sums in order
    if (rows_per_cta > 1) {
        if (ty > 0) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (e < n[i]) lines[(int64_t)(ty - 1) * p.width + (tx + i * tpr) * kVec + e] = dw[i][e];
        }
        __syncthreads();
    }
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (e < n[i]) {
                    const int col = (tx + i * tpr) * kVec + e;
                    float v = dw[i][e];
                    for (int q = 1; q < rows_per_cta; ++q) v += lines[(int64_t)(q - 1) * p.width + col];
                    p.part[(int64_t)blockIdx.x * p.width + col] = v;
                }
    }
}

}  // namespace rms

// out[c] = sum over i < lines of in[i * stride + c], c < cols, in a fixed order: 32 columns per CTA, eight threads
// down each, then the eight sums in order.
constexpr int kColThreads = 256, kColDown = kColThreads / 32;
__global__ void __launch_bounds__(kColThreads) column_sum_kernel(const float *in, int64_t lines, int64_t stride, int64_t cols,
                                                                 float *out) {
    __shared__ float sum[kColDown][33];
    const int lane = threadIdx.x & 31, down = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    float v = 0.f;
    if (c < cols)
#pragma unroll 8
        for (int64_t i = down; i < lines; i += kColDown) v += in[i * stride + c];
    sum[down][lane] = v;
    __syncthreads();
    if (down == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < kColDown; ++i) v += sum[i][lane];
        out[c] = v;
    }
}

}  // namespace dc
