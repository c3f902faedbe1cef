// rms_norm.cuh — the residual stream's addition with the RMS norm of the sum, and its backward.
//
//   forward   s = x + residual;  y = s w / sqrt(mean(s^2) + eps);  optionally y as e4m3 with scales
//   backward  with inv = 1 / sqrt(mean(r^2) + eps) of the stored sum r, and m = mean(w dy r inv):
//             d = inv (w dy - r inv m) + d_r,  d_w = sum over rows of dy r inv
//
// HBM-bound: the forward reads x and the residual and writes the sum and y once, the backward reads dy, d_r and r
// and writes d once; the row stays in registers between the reduction and its use.  A row is spread over TPR
// threads (a power of two, 32 to 512), eight consecutive columns per access, VPT accesses per thread; narrow
// rows share a CTA.  CTAs stay and take row after row: the next row's loads are under way, as raw words, while this
// one is reduced and written, and the weights stay in registers.  The inverse root is recomputed in the backward from the
// row it reads anyway, so the forward saves nothing beside r.
//
// Measured: 32768 x 2048 bfloat16 88 us (6.1 TB/s), 16384 x 4096 with a float32 residual into e4m3 125 us (6.0 TB/s),
// 16381 x 1560 with a float32 residual, forward and backward, 127 us (5.6 TB/s): 0.86 to 0.93 of a plain copy.
#pragma once

#include <cuda_fp8.h>
#include <float.h>

#include "common.cuh"
#include "vec.cuh"

namespace dc {
namespace rms {

constexpr int kVec = 8;  // columns per access

// How an access's eight columns lie in a row: side by side, in aligned or single accesses, or (where rows start anywhere)
// TPR columns apart, so that a warp's single accesses meet in few lines.
enum class Lay { kAligned, kSide, kApart };

template <Lay LAY>
__device__ __forceinline__ int column(int i, int tx, int tpr) { return LAY == Lay::kApart ? i * tpr * kVec + tx : (tx + i * tpr) * kVec; }
// columns of access i inside a row of `width`
template <Lay LAY>
__device__ __forceinline__ int inside(int i, int tx, int tpr, int width) {
    const int left = width - column<LAY>(i, tx, tpr);
    const int n = LAY == Lay::kApart ? (left + tpr - 1) / tpr : left;
    return left <= 0 ? 0 : n > kVec ? kVec : n;
}
template <Lay LAY>
__device__ __forceinline__ void load_cols(int dtype, const void *p, int64_t row, int i, int tx, int tpr, float (&v)[kVec], int n) {
    const int64_t at = row + column<LAY>(i, tx, tpr);
    if constexpr (LAY == Lay::kApart) {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
            v[e] = e >= n ? 0.f : dtype ? ld(static_cast<const __nv_bfloat16 *>(p) + at + e * tpr) : static_cast<const float *>(p)[at + e * tpr];
    } else {
        vec::load_as<LAY == Lay::kAligned>(dtype, p, at, v, n);
    }
}
template <Lay LAY>
__device__ __forceinline__ void store_cols(int dtype, void *p, int64_t row, int i, int tx, int tpr, const float (&v)[kVec], int n) {
    const int64_t at = row + column<LAY>(i, tx, tpr);
    if constexpr (LAY == Lay::kApart) {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
            if (e < n) {
                if (dtype) st(static_cast<__nv_bfloat16 *>(p) + at + e * tpr, v[e]);
                else static_cast<float *>(p)[at + e * tpr] = v[e];
            }
    } else {
        vec::store_as<LAY == Lay::kAligned>(dtype, p, at, v, n);
    }
}

struct Params {
    int64_t rows;
    int32_t width, group;  // group: columns per scale (e4m3), 0 = the whole row
    int32_t groups, group_shift;  // width / group; log2(group / kVec)
    int64_t x_stride, rin_stride, rout_stride, y_stride;
    int32_t x_dt, r_dt, y_dt;  // 0 float32, 1 bfloat16
    float eps;
    const void *x, *rin;
    const float *weight;
    void *rout, *y;
    float *scale;
};

// Sums (or maxima) over the TPR threads of a row; every thread of the CTA calls it.  `red` holds a pair per warp.
template <bool MAX>
__device__ __forceinline__ float2 row_reduce(float2 v, int tpr, float2 *red) {
    auto join = [](float2 a, float2 b) { return MAX ? make_float2(fmaxf(a.x, b.x), fmaxf(a.y, b.y)) : make_float2(a.x + b.x, a.y + b.y); };
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v = join(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tpr >> 5, first = warp & ~(per - 1);
    __syncthreads();  // the last reduction's values have been read
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    v = red[first];
    for (int i = 1; i < per; ++i) v = join(v, red[first + i]);
    return v;
}
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, int tpr, float2 *red) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, w) : v + w;
    }
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tpr >> 5, first = warp & ~(per - 1);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[warp].x = v;
    __syncthreads();
    v = red[first].x;
    for (int i = 1; i < per; ++i) v = MAX ? fmaxf(v, red[first + i].x) : v + red[first + i].x;
    return v;
}

// e4m3 values of v[i] * inv in one 8-byte word.  With inv = 1 / scale this is the quotient to about 2^-22 before its rounding to
// e4m3: next to a tie the other neighbour may come out.
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

// From the sum of one row on (s, n[i] columns of each access): its sum of squares, the stores, and y.  Every thread of the
// CTA calls it, with s = 0 and on = false where it has no row.
template <int VPT, Lay LAY, bool F8>
__device__ __forceinline__ void norm_row(const Params &p, float (&s)[VPT][kVec], const int (&n)[VPT], const float (&w)[VPT][kVec], int64_t row,
                                         bool on, int tx, int tpr, float2 *red) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) ss = fmaf(s[i][e], s[i][e], ss);
    if (p.rout && on) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (n[i] > 0) store_cols<LAY>(p.r_dt, p.rout, row * p.rout_stride, i, tx, tpr, s[i], n[i]);
    }
    ss = row_reduce<false>(ss, tpr, red);
    const float inv = 1.f / sqrtf(fmaf(ss, 1.f / (float)p.width, p.eps));
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) s[i][e] *= inv * w[i][e];
    if constexpr (!F8) {
        if (on) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (n[i] > 0) store_cols<LAY>(p.y_dt, p.y, row * p.y_stride, i, tx, tpr, s[i], n[i]);
        }
    } else {
        uint8_t *Y = static_cast<uint8_t *>(p.y);
        float amax[VPT], all = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            amax[i] = 0.f;  // fmaxf drops a NaN: its row is NaN throughout, and keeps scale 1
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (LAY == Lay::kAligned || e < n[i]) amax[i] = fmaxf(amax[i], fabsf(s[i][e]));
            all = fmaxf(all, amax[i]);
        }
        const int lanes = p.group ? p.group / kVec : 0;  // lanes of a group: 4 .. 32, a power of two
        if (lanes) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1)
                    if (o < lanes) amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], o));
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
                    if ((v & (lanes - 1)) == 0) p.scale[row * p.groups + (v >> p.group_shift)] = scale;
                } else if (v == 0) {
                    p.scale[row] = scale;
                }
                const uint2 q = to_e4m3(s[i], __fdividef(1.f, scale));
                uint8_t *o = Y + row * p.y_stride + v * kVec;
                if constexpr (LAY == Lay::kAligned) {
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

// This thread's part of a row: columns of each access, and the weights.
template <int VPT, Lay LAY>
__device__ __forceinline__ void columns(int width, const float *weight, int tx, int tpr, int (&n)[VPT], float (&w)[VPT][kVec]) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        n[i] = inside<LAY>(i, tx, tpr, width);
#pragma unroll
        for (int e = 0; e < kVec; ++e) w[i][e] = 0.f;
        if (n[i] > 0) load_cols<LAY>(0, weight, 0, i, tx, tpr, w[i], n[i]);
    }
}

// Whole 16-byte accesses: width a multiple of 8 and every row of every tensor 16-byte aligned (8-byte for e4m3).  80
// registers leave three CTAs of 256 an SM; two hold too few loads (16384 x 4096 into e4m3: 125 us, 140 at 96 registers).
template <typename TX, typename TR, int VPT, bool F8>
__global__ void __maxnreg__(VPT == 4 ? 128 : 80) rms_norm_vec_kernel(const Params p, int tpr) {
    __shared__ float2 red[32];
    const int tx = threadIdx.x & (tpr - 1), ty = threadIdx.x / tpr, rows_per_cta = blockDim.x / tpr;
    int n[VPT];
    float w[VPT][kVec];
    columns<VPT, Lay::kAligned>(p.width, p.weight, tx, tpr, n, w);
    const TX *X = static_cast<const TX *>(p.x) + tx * kVec;
    const TR *R = p.rin ? static_cast<const TR *>(p.rin) + tx * kVec : nullptr;
    vec::Raw<TX, kVec> x[VPT];
    vec::Raw<TR, kVec> r[VPT];
    auto load = [&](int64_t row) {
        if (row >= p.rows) return;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (n[i] > 0) vec::load_raw<true>(X + row * p.x_stride + i * tpr * kVec, x[i], kVec);
        if (R)
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (n[i] > 0) vec::load_raw<true>(R + row * p.rin_stride + i * tpr * kVec, r[i], kVec);
    };
    const int64_t stride = (int64_t)gridDim.x * rows_per_cta;
    int64_t row0 = (int64_t)blockIdx.x * rows_per_cta;
    load(row0 + ty);
    for (; row0 < p.rows; row0 += stride) {  // every thread takes the same number of rounds, for the barriers
        const int64_t row = row0 + ty;
        const bool on = row < p.rows;
        float s[VPT][kVec];
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < kVec; e += 2) {
                float2 v = vec::both(0.f);
                if (on && n[i] > 0) {
                    v = vec::pair_of(x[i], e / 2);
                    if (R) v = vec::add2(v, vec::pair_of(r[i], e / 2));
                }
                s[i][e] = v.x, s[i][e + 1] = v.y;
            }
        load(row + stride);
        norm_row<VPT, Lay::kAligned, F8>(p, s, n, w, row, on, tx, tpr, red);
    }
}

// Any width, stride and alignment.
template <int VPT, bool F8, Lay LAY>
__global__ void __launch_bounds__(512) rms_norm_kernel(const Params p, int tpr) {
    __shared__ float2 red[32];
    const int tx = threadIdx.x & (tpr - 1), ty = threadIdx.x / tpr, rows_per_cta = blockDim.x / tpr;
    int n[VPT];
    float w[VPT][kVec];
    columns<VPT, LAY>(p.width, p.weight, tx, tpr, n, w);
    for (int64_t row0 = (int64_t)blockIdx.x * rows_per_cta; row0 < p.rows; row0 += (int64_t)gridDim.x * rows_per_cta) {
        const int64_t row = row0 + ty;
        const bool on = row < p.rows;
        float s[VPT][kVec];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float r[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) s[i][e] = 0.f, r[e] = 0.f;
            if (on && n[i] > 0) {
                load_cols<LAY>(p.x_dt, p.x, row * p.x_stride, i, tx, tpr, s[i], n[i]);
                if (p.rin) load_cols<LAY>(p.r_dt, p.rin, row * p.rin_stride, i, tx, tpr, r, n[i]);
            }
#pragma unroll
            for (int e = 0; e < kVec; ++e) s[i][e] += r[e];
        }
        norm_row<VPT, LAY, F8>(p, s, n, w, row, on, tx, tpr, red);
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

// From one row's r and dy on: the reductions, d, and the row's part of d_weight.  Every thread of the CTA calls it.
// dr(i, d) and weight(i, w) give access i's d_r and weights.
template <int VPT, Lay LAY, typename DR, typename W>
__device__ __forceinline__ void bwd_row(const BwdParams &p, const float (&r)[VPT][kVec], const float (&g)[VPT][kVec], const int (&n)[VPT],
                                        W &&weight, float (&dw)[VPT][kVec], DR &&dr, int64_t row, bool on, int tx, int tpr, float2 *red) {
    float2 both = make_float2(0.f, 0.f);  // sum of r^2, sum of w dy r
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        float w[kVec];
        weight(i, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            both.x = fmaf(r[i][e], r[i][e], both.x);
            both.y = fmaf(w[e] * g[i][e], r[i][e], both.y);
        }
    }
    both = row_reduce<false>(both, tpr, red);
    const float inv_width = 1.f / (float)p.width;
    const float inv = 1.f / sqrtf(fmaf(both.x, inv_width, p.eps));
    const float mean = both.y * inv_width * inv;  // of w dy r inv.  (Powers of inv would leave float32's range before inv does.)
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        if (!on || n[i] <= 0) continue;
        float d[kVec], w[kVec];
        dr(i, d);
        weight(i, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const float unit = r[i][e] * inv;
            dw[i][e] = fmaf(g[i][e], unit, dw[i][e]);
            d[e] = fmaf(inv, fmaf(w[e], g[i][e], -unit * mean), d[e]);
        }
        if (p.dx) store_cols<LAY>(p.x_dt, p.dx, row * p.dx_stride, i, tx, tpr, d, n[i]);
        if (p.dres) store_cols<LAY>(p.r_dt, p.dres, row * p.dres_stride, i, tx, tpr, d, n[i]);
    }
}

// The CTA's line of d_weight partial sums; rows that share the CTA: row group 0 adds the others' sums in order.
template <int VPT, Lay LAY>
__device__ __forceinline__ void bwd_line(const BwdParams &p, const float (&dw)[VPT][kVec], const int (&n)[VPT], int tx, int ty, int tpr,
                                         int rows_per_cta, float *lines) {
    if (!p.part) return;
    if (rows_per_cta > 1) {
        if (ty > 0) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (e < n[i]) lines[(int64_t)(ty - 1) * p.width + column<LAY>(i, tx, tpr) + e * (LAY == Lay::kApart ? tpr : 1)] = dw[i][e];
        }
        __syncthreads();
    }
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (e < n[i]) {
                    const int col = column<LAY>(i, tx, tpr) + e * (LAY == Lay::kApart ? tpr : 1);
                    float v = dw[i][e];
                    for (int q = 1; q < rows_per_cta; ++q) v += lines[(int64_t)(q - 1) * p.width + col];
                    p.part[(int64_t)blockIdx.x * p.width + col] = v;
                }
    }
}

// CTAs that stay: each keeps its rows' share of d_weight in registers and writes it once, to its own line of `part`
// (column_sum_kernel adds the lines in order).  Whole 16-byte accesses, as in the forward.
template <typename TY, typename TR, int VPT>
__global__ void __launch_bounds__(512) rms_norm_bwd_vec_kernel(const BwdParams p, int tpr) {
    __shared__ float2 red[32];
    extern __shared__ float lines[];  // [rows per CTA - 1][width], when several rows share the CTA
    const int tx = threadIdx.x & (tpr - 1), ty = threadIdx.x / tpr, rows_per_cta = blockDim.x / tpr;
    int n[VPT];
    float w[VPT][kVec], dw[VPT][kVec];
    columns<VPT, Lay::kAligned>(p.width, p.weight, tx, tpr, n, w);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) dw[i][e] = 0.f;
    const TY *DY = static_cast<const TY *>(p.dy) + tx * kVec;
    const TR *R = static_cast<const TR *>(p.r) + tx * kVec, *DR = p.dr ? static_cast<const TR *>(p.dr) + tx * kVec : nullptr;
    vec::Raw<TY, kVec> gy[VPT];
    vec::Raw<TR, kVec> rr[VPT], gr[VPT];
    auto load = [&](int64_t row) {
        if (row >= p.rows) return;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (n[i] > 0) {
                vec::load_raw<true>(R + row * p.r_stride + i * tpr * kVec, rr[i], kVec);
                vec::load_raw<true>(DY + row * p.dy_stride + i * tpr * kVec, gy[i], kVec);
            }
    };
    auto load_dr = [&](int64_t row) {
        if (DR && row < p.rows)
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (n[i] > 0) vec::load_raw<true>(DR + row * p.dr_stride + i * tpr * kVec, gr[i], kVec);
    };
    const int64_t stride = (int64_t)gridDim.x * rows_per_cta;
    int64_t row0 = (int64_t)blockIdx.x * rows_per_cta;
    load(row0 + ty);
    for (; row0 < p.rows; row0 += stride) {
        const int64_t row = row0 + ty;
        const bool on = row < p.rows;
        float r[VPT][kVec], g[VPT][kVec];
        load_dr(row);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < kVec; e += 2) {
                const bool in = on && n[i] > 0;
                const float2 a = in ? vec::pair_of(rr[i], e / 2) : vec::both(0.f), b = in ? vec::pair_of(gy[i], e / 2) : vec::both(0.f);
                r[i][e] = a.x, r[i][e + 1] = a.y, g[i][e] = b.x, g[i][e + 1] = b.y;
            }
        load(row + stride);
        auto dr = [&](int i, float (&d)[kVec]) {
#pragma unroll
            for (int e = 0; e < kVec; e += 2) {
                const float2 v = DR ? vec::pair_of(gr[i], e / 2) : vec::both(0.f);
                d[e] = v.x, d[e + 1] = v.y;
            }
        };
        auto weight = [&](int i, float (&v)[kVec]) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) v[e] = w[i][e];
        };
        bwd_row<VPT, Lay::kAligned>(p, r, g, n, weight, dw, dr, row, on, tx, tpr, red);
    }
    bwd_line<VPT, Lay::kAligned>(p, dw, n, tx, ty, tpr, rows_per_cta, lines);
}

// Any width, stride and alignment; and, aligned, the widths whose rows leave no registers for loads under way and weights.
template <int VPT, Lay LAY>
__global__ void __launch_bounds__(512) rms_norm_bwd_kernel(const BwdParams p, int tpr) {
    __shared__ float2 red[32];
    extern __shared__ float lines[];
    const int tx = threadIdx.x & (tpr - 1), ty = threadIdx.x / tpr, rows_per_cta = blockDim.x / tpr;
    int n[VPT];
    float dw[VPT][kVec];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        n[i] = inside<LAY>(i, tx, tpr, p.width);
#pragma unroll
        for (int e = 0; e < kVec; ++e) dw[i][e] = 0.f;
    }
    for (int64_t row0 = (int64_t)blockIdx.x * rows_per_cta; row0 < p.rows; row0 += (int64_t)gridDim.x * rows_per_cta) {
        const int64_t row = row0 + ty;
        const bool on = row < p.rows;
        float r[VPT][kVec], g[VPT][kVec];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) r[i][e] = 0.f, g[i][e] = 0.f;
            if (on && n[i] > 0) {
                load_cols<LAY>(p.r_dt, p.r, row * p.r_stride, i, tx, tpr, r[i], n[i]);
                load_cols<LAY>(p.y_dt, p.dy, row * p.dy_stride, i, tx, tpr, g[i], n[i]);
            }
        }
        auto dr = [&](int i, float (&d)[kVec]) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) d[e] = 0.f;
            if (p.dr) load_cols<LAY>(p.r_dt, p.dr, row * p.dr_stride, i, tx, tpr, d, n[i]);
        };
        auto weight = [&](int i, float (&v)[kVec]) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) v[e] = 0.f;
            if (n[i] > 0) load_cols<LAY>(0, p.weight, 0, i, tx, tpr, v, n[i]);
        };
        bwd_row<VPT, LAY>(p, r, g, n, weight, dw, dr, row, on, tx, tpr, red);
    }
    bwd_line<VPT, LAY>(p, dw, n, tx, ty, tpr, rows_per_cta, lines);
}

}  // namespace rms

// out[c] = sum over i < lines of in[i * stride + c], c < cols, in a fixed order: 32 columns per CTA, 32 threads down each,
// then their sums in order.  Narrow rows give few CTAs, so loads under way are what counts: 4 us less than with eight threads
// down, at 296 lines of 1560 columns.
constexpr int kColThreads = 1024, kColDown = kColThreads / 32;
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
