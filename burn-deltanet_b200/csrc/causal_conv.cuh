// causal_conv.cuh — the short causal depthwise convolution in front of a selective scan, one decode tick of it, and
// its backward.  x [batch, seq, channels], channels contiguous:
//
//   pre_t = bias + sum_j w_j x_{t-K+1+j},  y_t = pre_t sigma(pre_t)  (or pre_t)
//   backward, with e_t = dy_t dy/dpre:  dx_t = sum_j w_j e_{t+K-1-j},  dw_j = sum_t e_t x_{t-K+1+j},  db = sum_t e_t
//
// HBM-bound.  A thread owns a few adjacent channels and a run of tokens: it reads its channels' tokens one after the
// other (a warp reads 32 such channel groups side by side, whole 128-byte lines), keeps the last K - 1 in registers,
// and so reads each input once but for the K - 1 tokens before its run, which its neighbour's loads have just brought
// into the caches.  The backward recomputes pre from x and carries the K unfinished sums of dx in registers the same
// way; its run starts at its first token and ends K - 1 tokens past its last.
#pragma once

#include "common.cuh"
#include "vec.cuh"

namespace dc {
namespace conv {

constexpr int kMaxTaps = 8;
constexpr int kThreads = 128;  // forward: four runs side by side
constexpr int kUnroll = 8;     // tokens whose loads are in flight together
constexpr int kBwdThreads = 256;
constexpr int kBwdUnroll = 4;

struct Params {
    int64_t batch, seq, channels;
    int64_t x_b, x_t, y_b, y_t;
    int32_t K, silu, run;  // run: tokens per thread, a multiple of kUnroll
    int32_t runs;          // runs of a sequence
    int32_t y_dt;
    const void *x;
    const float *weight, *bias, *window_in;
    const int32_t *lengths;
    void *y;
    float *window_out;
};

// sigma(x) with the fast exponential (x -> -inf gives 0): a few ulp
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

__device__ __forceinline__ int64_t length_of(const int32_t *lengths, int64_t b, int64_t seq) {
    if (!lengths) return seq;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n > seq ? seq : n;
}

// channel c's value of token t < len (t < 0: the window)
template <typename TI>
__device__ __forceinline__ float token(const TI *x, int64_t x_t, const float *win, int64_t K, int64_t t, int64_t c) {
    if (t >= 0) return ld(x + t * x_t + c);
    return win && t >= -K ? win[c * K + K + t] : 0.f;
}

// VEC channels per thread (with ALIGNED their loads and stores are whole vectors); KT: taps compiled in (the call's own,
// or kMaxTaps with the first KT - K of them left out).
template <typename TI, int VEC, bool ALIGNED, int KT>
__global__ void __launch_bounds__(kThreads) conv_kernel(const Params p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t item = (int64_t)blockIdx.x * (kThreads / 32) + warp;  // (sequence, run)
    if (item >= p.batch * p.runs) return;
    const int64_t b = item / p.runs, t0 = (item - b * p.runs) * (int64_t)p.run;
    const int64_t c0 = ((int64_t)blockIdx.y * 32 + lane) * VEC;
    if (c0 >= p.channels) return;
    const int n = p.channels - c0 < VEC ? (int)(p.channels - c0) : VEC;
    const int K = KT == kMaxTaps ? p.K : KT;
    const int64_t len = length_of(p.lengths, b, p.seq);
    const int64_t t1 = t0 + p.run < p.seq ? t0 + p.run : p.seq;
    const int64_t live = t1 < len ? t1 : len;  // tokens from here on are zeros
    const TI *x = static_cast<const TI *>(p.x) + b * p.x_b;
    const float *win = p.window_in ? p.window_in + b * p.channels * K : nullptr;
    const int64_t yb = b * p.y_b + c0;

    if (t0 < live) {
        // w[j] belongs to token t - (KT - 1) + j
        float w[KT][VEC], bias[VEC], hist[KT - 1][VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int64_t c = c0 + (e < n ? e : 0);
#pragma unroll
            for (int j = 0; j < KT; ++j) w[j][e] = j >= KT - K ? p.weight[c * K + j - (KT - K)] : 0.f;
            bias[e] = p.bias ? p.bias[c] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < KT - 1; ++j) {
            const int64_t t = t0 - (KT - 1) + j;
            if (t >= 0) {
                vec::load<ALIGNED>(x + t * p.x_t + c0, hist[j], n);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) hist[j][e] = e < n ? token(x, p.x_t, win, K, t, c0 + e) : 0.f;
            }
        }
        for (int64_t t = t0; t < live; t += kUnroll) {
            float in[kUnroll][VEC];
#pragma unroll
            for (int i = 0; i < kUnroll; ++i) {  // past the end: the last token again, not used
                const int64_t ti = t + i < live ? t + i : live - 1;
                vec::load<ALIGNED>(x + ti * p.x_t + c0, in[i], n);
            }
#pragma unroll
            for (int i = 0; i < kUnroll; ++i) {
                if (t + i < live) {
                    float out[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        float a = bias[e];
#pragma unroll
                        for (int j = 0; j < KT - 1; ++j)
                            if (j >= KT - K) a = fmaf(w[j][e], hist[j][e], a);
                        a = fmaf(w[KT - 1][e], in[i][e], a);
                        out[e] = p.silu ? a * sigmoid(a) : a;
                    }
                    vec::store_as<ALIGNED>(p.y_dt, p.y, yb + (t + i) * p.y_t, out, n);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
#pragma unroll
                        for (int j = 0; j < KT - 2; ++j) hist[j][e] = hist[j + 1][e];
                        hist[KT - 2][e] = in[i][e];
                    }
                }
            }
        }
    }
    if (t1 > live) {
        float zero[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) zero[e] = 0.f;
        for (int64_t t = t0 > live ? t0 : live; t < t1; ++t) vec::store_as<ALIGNED>(p.y_dt, p.y, yb + t * p.y_t, zero, n);
    }
    // the next window, from the run that holds the last token (the first run when there is none)
    if (p.window_out && (len == 0 ? t0 == 0 : t0 < len && len <= t0 + p.run)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (e < n)
                for (int j = 0; j < K; ++j)
                    p.window_out[(b * p.channels + c0 + e) * K + j] = token(x, p.x_t, win, K, len - K + j, c0 + e);
    }
}

// One token per sequence: a thread per channel, the window shifted in place or copied.
template <typename TI>
__global__ void __launch_bounds__(256) conv_step_kernel(const Params p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.batch * p.channels) return;
    const int64_t b = i / p.channels, c = i - b * p.channels;
    const int K = p.K;
    const bool on = length_of(p.lengths, b, 1) > 0;
    const float *win = p.window_in ? p.window_in + i * K : nullptr;
    float *out = p.window_out ? p.window_out + i * K : nullptr;
    const float *w = p.weight + c * K;
    float a = p.bias ? p.bias[c] : 0.f;
    if (K == 4 && aligned16(p.weight) && (!win || aligned16(p.window_in)) && (!out || aligned16(p.window_out))) {
        const float4 o = win ? *reinterpret_cast<const float4 *>(win) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 v = *reinterpret_cast<const float4 *>(w);
        const float x = on ? ld(static_cast<const TI *>(p.x) + b * p.x_b + c) : 0.f;
        a = fmaf(v.x, o.y, a), a = fmaf(v.y, o.z, a), a = fmaf(v.z, o.w, a), a = fmaf(v.w, x, a);
        if (out) *reinterpret_cast<float4 *>(out) = on ? make_float4(o.y, o.z, o.w, x) : o;
    } else {
        const float x = on ? ld(static_cast<const TI *>(p.x) + b * p.x_b + c) : 0.f;
        float old = win ? win[0] : 0.f;  // column j, read before column j is written
        for (int j = 0; j < K; ++j) {
            const float next = j + 1 < K ? (win ? win[j + 1] : 0.f) : x;
            a = fmaf(w[j], next, a);
            if (out) out[j] = on ? next : old;
            old = next;
        }
    }
    const float y = on ? (p.silu ? a * sigmoid(a) : a) : 0.f;
    if (p.y_dt) st(static_cast<__nv_bfloat16 *>(p.y) + b * p.y_b + c, y);
    else st(static_cast<float *>(p.y) + b * p.y_b + c, y);
}

struct BwdParams {
    int64_t batch, seq, channels;
    int64_t x_b, x_t, dy_b, dy_t, dx_b, dx_t;
    int32_t K, silu, run, runs, y_dt;
    const void *dy, *x;
    const float *dwin_out, *weight, *bias, *window_in;
    const int32_t *lengths;
    void *dx;
    float *dwin_in;
    float *part;  // [gridDim.x][K + 1][channels]: each CTA's sums of d_weight (K lines) and d_bias
};

// Channels of a warp: 32 * VEC.  The CTA's warps take consecutive runs of the same channels and add their sums in
// order in shared memory.
template <typename TI, int VEC, bool ALIGNED, int KT>
__global__ void __launch_bounds__(kBwdThreads) conv_bwd_kernel(const BwdParams p) {
    constexpr int kWarps = kBwdThreads / 32;
    __shared__ float sums[kWarps][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
    const int64_t c0 = ((int64_t)blockIdx.y * 32 + lane) * VEC;
    const int n = c0 >= p.channels ? 0 : p.channels - c0 < VEC ? (int)(p.channels - c0) : VEC;
    const int K = KT == kMaxTaps ? p.K : KT;
    float dw[KT][VEC], db[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        db[e] = 0.f;
#pragma unroll
        for (int j = 0; j < KT; ++j) dw[j][e] = 0.f;
    }
    if (item < p.batch * p.runs && n > 0) {
        const int64_t b = item / p.runs, t0 = (item - b * p.runs) * (int64_t)p.run;
        const int64_t len = length_of(p.lengths, b, p.seq);
        const int64_t t1 = t0 + p.run < p.seq ? t0 + p.run : p.seq;
        const TI *x = static_cast<const TI *>(p.x) + b * p.x_b;
        TI *dx = static_cast<TI *>(p.dx) + b * p.dx_b + c0;
        const float *win = p.window_in ? p.window_in + b * p.channels * K : nullptr;
        const float *dnext = p.dwin_out ? p.dwin_out + b * p.channels * K : nullptr;
        float *dwin = p.dwin_in ? p.dwin_in + b * p.channels * K : nullptr;
        float w[KT][VEC], bias[VEC], hist[KT - 1][VEC], d[KT][VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int64_t c = c0 + (e < n ? e : 0);
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                w[j][e] = j >= KT - K ? p.weight[c * K + j - (KT - K)] : 0.f;
                d[j][e] = 0.f;
            }
            bias[e] = p.bias ? p.bias[c] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < KT - 1; ++j) {
            const int64_t t = t0 - (KT - 1) + j;
#pragma unroll
            for (int e = 0; e < VEC; ++e) hist[j][e] = 0.f;
            if (j >= KT - K && t < len) {
                if (t >= 0) {
                    vec::load<ALIGNED>(x + t * p.x_t + c0, hist[j], n);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) hist[j][e] = e < n ? token(x, p.x_t, win, K, t, c0 + e) : 0.f;
                }
            }
        }
        // d[j] gathers dx of token t - (KT - 1) + j while e_t passes by; after token t, d[0] is complete
        const int64_t end = t1 + KT - 1;  // tokens past t1 only finish the run's last sums
        for (int64_t t = t0; t < end; t += kBwdUnroll) {
            float in[kBwdUnroll][VEC], go[kBwdUnroll][VEC];
#pragma unroll
            for (int i = 0; i < kBwdUnroll; ++i) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) in[i][e] = 0.f, go[i][e] = 0.f;
                if (t + i < len) {
                    vec::load<ALIGNED>(x + (t + i) * p.x_t + c0, in[i], n);
                    vec::load_as<ALIGNED>(p.y_dt, p.dy, b * p.dy_b + (t + i) * p.dy_t + c0, go[i], n);
                }
            }
#pragma unroll
            for (int i = 0; i < kBwdUnroll; ++i) {
                const int64_t ti = t + i;
                if (ti < end) {
                    const bool mine = ti < t1;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        float pre = bias[e];
#pragma unroll
                        for (int j = 0; j < KT - 1; ++j) pre = fmaf(w[j][e], hist[j][e], pre);
                        pre = fmaf(w[KT - 1][e], in[i][e], pre);
                        float g = go[i][e];
                        if (p.silu) {
                            const float s = sigmoid(pre);
                            g *= s * fmaf(pre, 1.f - s, 1.f);
                        }
                        if (ti >= len) g = 0.f;
#pragma unroll
                        for (int j = 0; j < KT; ++j) d[j][e] = fmaf(w[j][e], g, d[j][e]);
                        if (mine) {
                            db[e] += g;
#pragma unroll
                            for (int j = 0; j < KT - 1; ++j) dw[j][e] = fmaf(g, hist[j][e], dw[j][e]);
                            dw[KT - 1][e] = fmaf(g, in[i][e], dw[KT - 1][e]);
                        }
                    }
                    const int64_t tau = ti - (KT - 1);  // d[0]'s token
                    if (tau >= t0 && tau < p.seq) {
                        if (dnext && tau < len && tau >= len - K) {
#pragma unroll
                            for (int e = 0; e < VEC; ++e)
                                if (e < n) d[0][e] += dnext[(c0 + e) * K + (int)(tau - len + K)];
                        }
                        vec::store<ALIGNED>(dx + tau * p.dx_t, d[0], n);
                    } else if (dwin && tau < 0 && tau >= -(K - 1)) {  // t0 is 0: a token of the window
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            if (e < n) {
                                const int m = K + (int)tau;
                                const float more = dnext && m >= len ? dnext[(c0 + e) * K + m - (int)len] : 0.f;
                                dwin[(c0 + e) * K + m] = d[0][e] + more;
                            }
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
#pragma unroll
                        for (int j = 0; j < KT - 1; ++j) d[j][e] = d[j + 1][e];
                        d[KT - 1][e] = 0.f;
#pragma unroll
                        for (int j = 0; j < KT - 2; ++j) hist[j][e] = j >= KT - K ? hist[j + 1][e] : 0.f;
                        if (KT - 2 >= KT - K) hist[KT - 2][e] = in[i][e];
                    }
                }
            }
        }
        if (dwin && t0 == 0) {  // column 0 reaches the output only as an unshifted window
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e < n) dwin[(c0 + e) * K] = dnext && len == 0 ? dnext[(c0 + e) * K] : 0.f;
        }
    }
    // the CTA's sums: the warps' in order, one tap at a time
    float *part = p.part + (int64_t)blockIdx.x * (K + 1) * p.channels;
#pragma unroll
    for (int j = 0; j < KT + 1; ++j) {
        if (j < KT - K) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[warp][lane * VEC + e] = j < KT ? dw[j < KT ? j : 0][e] : db[e];
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * VEC; i += kBwdThreads) {
            float v = sums[0][i];
#pragma unroll
            for (int q = 1; q < kWarps; ++q) v += sums[q][i];
            const int64_t c = (int64_t)blockIdx.y * 32 * VEC + i;
            if (c < p.channels) part[(int64_t)(j - (KT - K)) * p.channels + c] = v;
        }
    }
}

// d_weight [channels, K] and d_bias [channels] from the CTAs' sums: 32 channels and one line (tap or bias) per CTA,
// eight threads down the CTAs each, then the eight sums in order.
__global__ void __launch_bounds__(256) conv_bwd_sum_kernel(const float *part, int64_t ctas, int64_t channels, int K, float *dw, float *db) {
    __shared__ float sum[8][33];
    const int lane = threadIdx.x & 31, down = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    const int j = blockIdx.y;
    float v = 0.f;
    if (c < channels)
#pragma unroll 8
        for (int64_t i = down; i < ctas; i += 8) v += part[(i * (K + 1) + j) * channels + c];
    sum[down][lane] = v;
    __syncthreads();
    if (down == 0 && c < channels) {
#pragma unroll
        for (int i = 1; i < 8; ++i) v += sum[i][lane];
        if (j < K) dw[c * K + j] = v;
        else if (db) db[c] = v;
    }
}

}  // namespace conv
}  // namespace dc
