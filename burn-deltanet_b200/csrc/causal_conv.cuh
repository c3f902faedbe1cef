// causal_conv.cuh — the short causal depthwise convolution in front of a selective scan, one decode tick of it, and
// its backward.  x [batch, seq, channels], channels contiguous:
//
//   pre_t = bias + sum_j w_j x_{t-K+1+j},  y_t = pre_t sigma(pre_t)  (or pre_t)
//   backward, with e_t = dy_t dy/dpre:  dx_t = sum_j w_j e_{t+K-1-j},  dw_j = sum_t e_t x_{t-K+1+j},  db = sum_t e_t
//
// HBM-bound.  A thread owns a pair of adjacent channels, in two-wide arithmetic, and a run of tokens: it works on its
// channels' tokens one after the other, keeps the last K - 1 in registers, and so reads each input once but for the K - 1
// tokens before its run.  Where rows start on 16-byte boundaries each warp stages its 64 channels' tokens through a ring of
// its own in shared memory (asynchronous copies, 48 tokens ahead, no barrier beyond the warp), so that the bytes in flight
// do not depend on registers; loads into registers, eight tokens at a time, took 69 us at 8 x 4096 x 2048 bfloat16 where this
// takes 62 (4.3 TB/s).  No unit is full there (HBM 0.66, the special-function unit and the issue slots about half): 2048 CTAs
// make 2.3 waves of the 888 that the card holds, and each warp fills its ring anew for its run.
//
// The backward recomputes pre from x and carries the K unfinished sums of dx in registers the same way; its run ends
// K - 1 tokens past its last.  x and dy come through a ring each, 24 tokens ahead, and tokens that lie in the middle of a
// run are worked on eight at a time without questions about lengths and windows.  Ragged 6 x 2049 x 1536 bfloat16, forward
// and backward: 59 us (71 with loads into registers), of which the backward is 36 and the sums of the CTAs' parts 3; no unit is
// above half its rate there: 128 registers allow 16 warps an SM, whose dependent instructions show, and 1200 CTAs are two
// waves of 592 and a remnant.
#pragma once

#include "common.cuh"
#include "ptx.cuh"
#include "vec.cuh"

namespace dc {
namespace conv {

constexpr int kMaxTaps = 8;
constexpr int kThreads = 128;  // four runs side by side
constexpr int kVec = 2;        // channels of a thread
constexpr int kRow = 32 * kVec;
constexpr int kStages = 4, kStageTokens = 16;  // of a warp's ring
constexpr int kUnroll = 8;     // without it: tokens whose loads are in flight together
constexpr int kBwdThreads = 128;
constexpr int kBwdUnroll = 8;  // tokens of a stage, and of a group that is worked on without questions

struct Params {
    int64_t batch, seq, channels;
    int64_t x_b, x_t, y_b, y_t;
    int32_t K, silu, run;  // run: tokens per thread, a multiple of kUnroll
    int32_t runs;          // runs of a sequence
    int32_t y_dt;
    int32_t y_pair;        // pairs of y's channels are aligned
    const void *x;
    const float *weight, *bias, *window_in;
    const int32_t *lengths;
    void *y;
    float *window_out;
};

// sigma(x) from the fast exponential and reciprocal (x -> -inf gives 0): 3 ulp and, from the rounding of the exponential's
// argument, about 1.2 more per unit of |x|
__device__ __forceinline__ float sigmoid(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
}

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

__device__ __forceinline__ float2 sigmoid2(float2 x) {
    const float2 z = vec::mul2(x, vec::both(-1.4426950408889634f));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(z.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(z.y));
    e = vec::add2(e, vec::both(1.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    return r;
}
// silu(x) or x, of a pair
__device__ __forceinline__ float2 activate(float2 a, bool silu) { return silu ? vec::mul2(a, sigmoid2(a)) : a; }

// A warp's ring: `count` tokens of 64 channels (nch of them real) from `from` on, TOKENS of them a stage.
template <typename T, int TOKENS>
struct Ring {
    static constexpr int kPer = kRow * sizeof(T) / 16, kEl = 16 / sizeof(T);       // copies per row
    static constexpr int kRows = 32 / kPer, kEach = TOKENS / kRows;                // rows of a warp's pass, passes of a stage
    using Buffer = T[kStages][TOKENS][kRow];
    const T *src;  // this lane's first copy of the next stage
    int64_t stride;
    uint32_t dst;
    int left, row, s;  // tokens not yet asked for; stage
    bool on;
    __device__ __forceinline__ Ring(Buffer &buf, const T *from, int64_t stride, int count, int nch, int lane) : stride(stride), left(count), s(0) {
        row = lane / kPer;
        const int q = lane % kPer;
        on = q * kEl < nch;
        src = from + row * stride + (on ? q * kEl : 0);
        dst = ptx::smem_u32(&buf[0][row][q * kEl]);
    }
    __device__ __forceinline__ void load() {  // the next stage, if there is one; the caller commits
        if (left > 0) {
            const uint32_t to = dst + s * (int)sizeof(T) * TOKENS * kRow;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const bool in = on && row + i * kRows < left;
                ptx::cp_async16(to + i * (int)sizeof(T) * kRows * kRow, in ? src + i * kRows * stride : src - row * stride, in ? 16u : 0u);
            }
            src += TOKENS * stride;
            left -= TOKENS;
            s = s + 1 < kStages ? s + 1 : 0;
        }
    }
};
template <typename T>
using FwdRing = Ring<T, kStageTokens>;
template <typename TI, typename TO>
struct BwdRings {
    typename Ring<TI, kBwdUnroll>::Buffer x;
    typename Ring<TO, kBwdUnroll>::Buffer dy;
};

// STAGED: rows start on 16-byte boundaries.  KT: taps compiled in (the call's own, or kMaxTaps with the first KT - K of
// them left out).
template <typename TI, typename TO, bool STAGED, int KT>
__global__ void __launch_bounds__(kThreads) conv_kernel(const Params p) {
    extern __shared__ __align__(16) unsigned char smem_bytes[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t item = (int64_t)blockIdx.x * (kThreads / 32) + warp;  // (sequence, run)
    if (item >= p.batch * p.runs) return;
    const int64_t b = item / p.runs, t0 = (item - b * p.runs) * (int64_t)p.run;
    const int64_t c0 = (int64_t)blockIdx.y * kRow + lane * kVec;
    const int n = c0 >= p.channels ? 0 : p.channels - c0 < kVec ? (int)(p.channels - c0) : kVec;
    const int K = KT == kMaxTaps ? p.K : KT;
    const int64_t len = length_of(p.lengths, b, p.seq);
    const int64_t t1 = t0 + p.run < p.seq ? t0 + p.run : p.seq;
    const int64_t live = t1 < len ? t1 : len;  // tokens from here on are zeros
    const TI *x = static_cast<const TI *>(p.x) + b * p.x_b;
    const float *win = p.window_in ? p.window_in + b * p.channels * K : nullptr;
    TO *y = static_cast<TO *>(p.y) + b * p.y_b + c0;
    const bool pair = n == kVec && p.y_pair;  // both channels in one store

    if (t0 < live) {
        const int count = (int)(live - t0);
        const int64_t row0 = (int64_t)blockIdx.y * kRow;
        auto &buf = reinterpret_cast<typename FwdRing<TI>::Buffer *>(smem_bytes)[warp];
        FwdRing<TI> ring(buf, x + t0 * p.x_t + row0, p.x_t, STAGED ? count : 0, (int)(p.channels - row0 < kRow ? p.channels - row0 : kRow), lane);
        if (STAGED)
#pragma unroll
            for (int s = 0; s < kStages - 1; ++s) {
                ring.load();
                ptx::cp_async_commit();
            }
        // w[j] belongs to token t - (KT - 1) + j
        float2 w[KT], hist[KT - 1], bias = vec::both(0.f);
        const int64_t ca = n > 0 ? c0 : 0, cb = n > 1 ? c0 + 1 : ca;
        if (p.bias) bias = make_float2(p.bias[ca], p.bias[cb]);
#pragma unroll
        for (int j = 0; j < KT; ++j)
            w[j] = j >= KT - K ? make_float2(p.weight[ca * K + j - (KT - K)], p.weight[cb * K + j - (KT - K)]) : vec::both(0.f);
#pragma unroll
        for (int j = 0; j < KT - 1; ++j) {
            const int64_t t = t0 - (KT - 1) + j;
            hist[j] = j >= KT - K ? make_float2(token(x, p.x_t, win, K, t, ca), token(x, p.x_t, win, K, t, cb)) : vec::both(0.f);
        }
        TO *to = y + t0 * p.y_t;
        auto next = [&](float2 v, TO *to) {  // one token's output, and the history one token on
            float2 a = bias;
#pragma unroll
            for (int j = 0; j < KT - 1; ++j) a = vec::fma2(w[j], hist[j], a);
            a = activate(vec::fma2(w[KT - 1], v, a), p.silu);
#pragma unroll
            for (int j = 0; j < KT - 2; ++j) hist[j] = j >= KT - K ? hist[j + 1] : vec::both(0.f);
            if (KT - 2 >= KT - K) hist[KT - 2] = v;
            const float out[kVec] = {a.x, a.y};
            if (pair) vec::store<true>(to, out);
            else vec::store<false>(to, out, n);
        };
        if constexpr (STAGED) {
            const TI *from = &buf[0][0][lane * kVec];
            auto at = [&](int i) {
                float v[kVec];
                vec::load<true>(from + i * kRow, v);
                return make_float2(v[0], v[1]);
            };
            for (int left = count, s = 0; left > 0; left -= kStageTokens) {
                ptx::cp_async_wait<kStages - 2>();
                __syncwarp();  // every lane's copies of this stage have landed, and the last stage has been read
                ring.load();
                ptx::cp_async_commit();
                if (left >= kStageTokens) {
#pragma unroll
                    for (int i = 0; i < kStageTokens; ++i) next(at(i), to + i * p.y_t);
                } else {
                    for (int i = 0; i < left; ++i) next(at(i), to + i * p.y_t);
                }
                to += kStageTokens * p.y_t;
                s = s + 1 < kStages ? s + 1 : 0;
                from = &buf[s][0][lane * kVec];
            }
            ptx::cp_async_wait<0>();
        } else if (n > 0) {
            const TI *from = x + t0 * p.x_t + c0;
            int t = 0;
            for (; t + kUnroll <= count; t += kUnroll, from += kUnroll * p.x_t) {
                vec::Raw<TI, kVec> in[kUnroll];
#pragma unroll
                for (int i = 0; i < kUnroll; ++i) vec::load_raw<false>(from + i * p.x_t, in[i], n);
#pragma unroll
                for (int i = 0; i < kUnroll; ++i) next(vec::pair_of(in[i], 0), to + i * p.y_t);
                to += kUnroll * p.y_t;
            }
            for (; t < count; ++t, from += p.x_t) {
                vec::Raw<TI, kVec> in;
                vec::load_raw<false>(from, in, n);
                next(vec::pair_of(in, 0), to);
                to += p.y_t;
            }
        }
    }
    if (t1 > live) {
        const float zero[kVec] = {0.f, 0.f};
        for (int64_t t = t0 > live ? t0 : live; t < t1; ++t) {
            if (pair) vec::store<true>(y + t * p.y_t, zero);
            else vec::store<false>(y + t * p.y_t, zero, n);
        }
    }
    // the next window, from the run that holds the last token (the first run when there is none)
    if (p.window_out && (len == 0 ? t0 == 0 : t0 < len && len <= t0 + p.run)) {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
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
    int32_t dx_pair;  // pairs of dx's channels are aligned
    const void *dy, *x;
    const float *dwin_out, *weight, *bias, *window_in;
    const int32_t *lengths;
    void *dx;
    float *dwin_in;
    float *part;  // [gridDim.x][K + 1][channels]: each CTA's sums of d_weight (K lines) and d_bias
};

// A pair of channels per thread, 64 of a warp; STAGED as in the forward, with a ring each for x and dy.  The CTA's warps take
// consecutive runs of the same channels and add their sums in order in shared memory.
template <typename TI, typename TO, bool STAGED, int KT>
__global__ void __launch_bounds__(kBwdThreads) conv_bwd_kernel(const BwdParams p) {
    constexpr int kWarps = kBwdThreads / 32, VEC = kVec;
    extern __shared__ __align__(16) unsigned char smem_bytes[];
    __shared__ float2 sums[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
    const int64_t c0 = ((int64_t)blockIdx.y * 32 + lane) * VEC;
    const int n = c0 >= p.channels ? 0 : p.channels - c0 < VEC ? (int)(p.channels - c0) : VEC;
    const int K = KT == kMaxTaps ? p.K : KT;
    float2 dw[KT], db = vec::both(0.f);
#pragma unroll
    for (int j = 0; j < KT; ++j) dw[j] = vec::both(0.f);
    if (item < p.batch * p.runs) {
        const int64_t b = item / p.runs, t0 = (item - b * p.runs) * (int64_t)p.run;
        const int64_t len = length_of(p.lengths, b, p.seq);
        const int64_t t1 = t0 + p.run < p.seq ? t0 + p.run : p.seq;
        const TI *x = static_cast<const TI *>(p.x) + b * p.x_b;
        TI *dx = static_cast<TI *>(p.dx) + b * p.dx_b + c0;
        const float *win = p.window_in ? p.window_in + b * p.channels * K : nullptr;
        const float *dnext = p.dwin_out ? p.dwin_out + b * p.channels * K : nullptr;
        float *dwin = p.dwin_in ? p.dwin_in + b * p.channels * K : nullptr;
        const int64_t ca = n > 0 ? c0 : 0, c1 = n > 1 ? c0 + 1 : ca;  // a lane without channels reads channel 0's, writes none
        const bool pair = n == VEC && p.dx_pair;
        auto put = [&](TI *o, float2 v) {
            const float out[VEC] = {v.x, v.y};
            if (pair) vec::store<true>(o, out);
            else vec::store<false>(o, out, n);
        };
        const int count = (int)(t1 - t0), end = count + KT - 1;               // tokens past t1 only finish the run's last sums
        const int live = len - t0 < 0 ? 0 : len - t0 < end ? (int)(len - t0) : end;  // tokens that are read
        const int64_t row0 = (int64_t)blockIdx.y * kRow;
        const int nch = (int)(p.channels - row0 < kRow ? p.channels - row0 : kRow);
        auto &rings = reinterpret_cast<BwdRings<TI, TO> *>(smem_bytes)[warp];
        Ring<TI, kBwdUnroll> rx(rings.x, x + t0 * p.x_t + row0, p.x_t, STAGED ? live : 0, nch, lane);
        Ring<TO, kBwdUnroll> rg(rings.dy, static_cast<const TO *>(p.dy) + b * p.dy_b + t0 * p.dy_t + row0, p.dy_t, STAGED ? live : 0, nch, lane);
        auto load = [&] {
            rx.load();
            rg.load();
            ptx::cp_async_commit();
        };
        if (STAGED)
#pragma unroll
            for (int s = 0; s < kStages - 1; ++s) load();
        float2 w[KT], hist[KT - 1], d[KT];
        const float2 bias = p.bias ? make_float2(p.bias[ca], p.bias[c1]) : vec::both(0.f);
#pragma unroll
        for (int j = 0; j < KT; ++j) {
            w[j] = j >= KT - K ? make_float2(p.weight[ca * K + j - (KT - K)], p.weight[c1 * K + j - (KT - K)]) : vec::both(0.f);
            d[j] = vec::both(0.f);
        }
#pragma unroll
        for (int j = 0; j < KT - 1; ++j) {
            const int64_t t = t0 - (KT - 1) + j;
            hist[j] = vec::both(0.f);
            if (j >= KT - K && t < len) hist[j] = make_float2(token(x, p.x_t, win, K, t, ca), token(x, p.x_t, win, K, t, c1));
        }
        const TI *from = x + t0 * p.x_t + ca;
        const TO *gfrom = static_cast<const TO *>(p.dy) + b * p.dy_b + t0 * p.dy_t + ca;
        int stage = -1;  // of the rings
        auto advance = [&] {  // the next stage is there
            ptx::cp_async_wait<kStages - 2>();
            __syncwarp();
            load();
            stage = stage + 1 < kStages ? stage + 1 : 0;
        };
        auto fetch = [&](int t, float2 &v, float2 &g) {  // token t < live
            float a[VEC], c[VEC];
            if (STAGED) {
                vec::load<true>(&rings.x[stage][t % kBwdUnroll][lane * VEC], a);
                vec::load<true>(&rings.dy[stage][t % kBwdUnroll][lane * VEC], c);
            } else {
                vec::load<false>(from + t * p.x_t, a, n);
                vec::load<false>(gfrom + t * p.dy_t, c, n);
            }
            v = make_float2(a[0], a[1]), g = make_float2(c[0], c[1]);
        };
        // d[j] gathers dx of token t - (KT - 1) + j while the gradient of pre_t passes by; after token t, d[0] is complete
        auto pass = [&](float2 v, float2 g, bool read, bool own) {  // token t: its gradients into d, and into dw and db if its own
            float2 pre = bias;
#pragma unroll
            for (int j = 0; j < KT - 1; ++j) pre = vec::fma2(w[j], hist[j], pre);
            pre = vec::fma2(w[KT - 1], v, pre);
            if (p.silu && read) {
                const float2 s = sigmoid2(pre);
                const float2 slope = vec::fma2(vec::mul2(pre, s), vec::fma2(s, vec::both(-1.f), vec::both(1.f)), s);
                g = vec::mul2(g, slope);
            }
#pragma unroll
            for (int j = 0; j < KT; ++j) d[j] = vec::fma2(w[j], g, d[j]);
            if (own) {
                db = vec::add2(db, g);
#pragma unroll
                for (int j = 0; j < KT - 1; ++j) dw[j] = vec::fma2(g, hist[j], dw[j]);
                dw[KT - 1] = vec::fma2(g, v, dw[KT - 1]);
            }
        };
        auto shift = [&](float2 v) {
#pragma unroll
            for (int j = 0; j < KT - 1; ++j) d[j] = d[j + 1];
            d[KT - 1] = vec::both(0.f);
#pragma unroll
            for (int j = 0; j < KT - 2; ++j) hist[j] = j >= KT - K ? hist[j + 1] : vec::both(0.f);
            if (KT - 2 >= KT - K) hist[KT - 2] = v;
        };
        auto window = [&](int64_t tau, float2 v) {  // the gradient of a token of the window (t0 is 0)
            if (!dwin || tau < -(K - 1)) return;
            const int m = K + (int)tau;
            const bool more = dnext && m >= len;
            if (n > 0) dwin[c0 * K + m] = v.x + (more ? dnext[c0 * K + m - (int)len] : 0.f);
            if (n > 1) dwin[c1 * K + m] = v.y + (more ? dnext[c1 * K + m - (int)len] : 0.f);
        };
        auto any = [&](int t) {  // a token of whatever place
            const bool read = t < live;
            float2 v = vec::both(0.f), g = vec::both(0.f);
            if (STAGED && t % kBwdUnroll == 0) advance();
            if (read) fetch(t, v, g);
            pass(v, g, read, t < count);
            const int64_t tau = t0 + t - (KT - 1);  // d[0]'s token
            if (tau >= t0) {
                if (dnext && tau < len && tau >= len - K) {
                    if (n > 0) d[0].x += dnext[c0 * K + (int)(tau - len + K)];
                    if (n > 1) d[0].y += dnext[c1 * K + (int)(tau - len + K)];
                }
                put(dx + tau * p.dx_t, d[0]);
            } else if (tau < 0) {
                window(tau, d[0]);
            }
            shift(v);
        };
        // eight tokens that are read and the run's own, and finish tokens that the window's gradient does not reach
        auto group = [&](int t, bool opens) {
            if (STAGED) advance();
            TI *o = dx + (t0 + t - (KT - 1)) * p.dx_t;
            float2 v[kBwdUnroll], g[kBwdUnroll];
#pragma unroll
            for (int i = 0; i < kBwdUnroll; ++i) fetch(t + i, v[i], g[i]);
#pragma unroll
            for (int i = 0; i < kBwdUnroll; ++i) {
                pass(v[i], g[i], true, true);
                if (i < KT - 1 && opens) {
                    if (t0 == 0) window(i - (KT - 1), d[0]);
                } else {
                    put(o + i * p.dx_t, d[0]);
                }
                shift(v[i]);
            }
        };
        // from `stop` on every sum is zero; a run that lies behind the sequence's end has none at all
        const int stop = live == 0 && t0 > 0 ? 0 : live + KT - 1 < end ? live + KT - 1 : end;
        const int plain_end = (int)min((int64_t)min(count, live), dnext ? len - K + (KT - 1) - t0 : (int64_t)count);
        int t = 0;
        if (KT - 1 <= kBwdUnroll && kBwdUnroll <= plain_end) {
            group(0, true);
            for (t = kBwdUnroll; t + kBwdUnroll <= plain_end; t += kBwdUnroll) group(t, false);
        }
        for (; t < stop; ++t) any(t);
        if (STAGED) ptx::cp_async_wait<0>();
        for (int64_t tau = t0 + (stop > KT - 1 ? stop - (KT - 1) : 0); tau < t1; ++tau) put(dx + tau * p.dx_t, vec::both(0.f));
        if (dwin && t0 == 0) {  // column 0 reaches the output only as an unshifted window
            if (n > 0) dwin[c0 * K] = dnext && len == 0 ? dnext[c0 * K] : 0.f;
            if (n > 1) dwin[c1 * K] = dnext && len == 0 ? dnext[c1 * K] : 0.f;
        }
    }
    // the CTA's sums: the warps' in order, one tap at a time
    float *part = p.part + (int64_t)blockIdx.x * (K + 1) * p.channels;
#pragma unroll
    for (int j = 0; j < KT + 1; ++j) {
        if (j < KT - K) continue;
        __syncthreads();
        sums[warp][lane] = j < KT ? dw[j < KT ? j : 0] : db;
        __syncthreads();
        if (warp == 0) {
            float2 v = sums[0][lane];
#pragma unroll
            for (int q = 1; q < kWarps; ++q) v = vec::add2(v, sums[q][lane]);
            if (n > 0) part[(int64_t)(j - (KT - K)) * p.channels + c0] = v.x;
            if (n > 1) part[(int64_t)(j - (KT - K)) * p.channels + c0 + 1] = v.y;
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
    if (c < channels) v = vec::sum_lines(part + j * channels + c, down, ctas, 8, (K + 1) * channels);
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
