// selective_scan.cuh — the selective state space scan over a prompt, and one decode tick of it.
//
//   step_t = softplus(dt_t + dt_bias)       h_n <- exp(step_t a_n) h_n + step_t u_t b_tn
//   y_t = (sum_n c_tn h_n + d u_t) z_t sigma(z_t)
//
// per (sequence, channel), `state` values of h.  The exponentials bound it: state + 4 of them and their like
// (softplus, silu) per (token, channel) at 16 a clock and SM, against 4 elements read or written.
//
// Layout.  A CTA of 256 threads owns 16 channels of one sequence and walks its tokens in tiles.  Four states of a
// channel live in a thread's registers, so a channel spans P = state / 4 threads (padded to a power of two, the padding
// with a = b = c = 0), and the CTA's 16 / P segments of 16 P threads take consecutive runs of K = 8 tokens of the tile.
// The recurrence is linear, so each segment first runs its K tokens from zero while it keeps the decays and the products
// in registers (every exponential is taken once), the segments exchange (product of decays, end state) through shared
// memory, and each runs its K tokens again from the state that reaches it, now reading out: two multiply-adds per token
// and state more than a serial walk, hidden behind the exponentials, for 16 / P times the parallel work.  b and c of a
// tile are read once for the CTA's channels and kept in float32 in shared memory.
#pragma once

#include "common.cuh"
#include "ptx.cuh"
#include "vec.cuh"

namespace dc {
namespace scan {

constexpr int kThreads = 256;
constexpr int kCh = 16;   // channels of a CTA
constexpr int kK = 8;     // tokens of a segment
constexpr int kS = 4;     // states of a thread
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int P>
struct Tile {
    static constexpr int kSegs = kThreads / (kCh * P);  // 16 / P
    static constexpr int kTokens = kSegs * kK;
    static constexpr int kN = kS * P;  // padded states
};

struct Params {
    int64_t batch, seq, channels, groups, per;  // per: channels of a group
    int32_t N;
    int64_t u_b, u_t, dt_b, dt_t, z_b, z_t, b_b, b_t, c_b, c_t, y_b, y_t;
    int32_t softplus, y_dt;
    int32_t vec_x, vec_bc;  // strides allow 16-byte copies of the channel rows / of the b and c rows
    int32_t blocks;         // CTAs of a group: ceil(per / 16)
    int32_t tiles;          // checkpoints of a sequence
    const void *u, *dt, *z, *b, *c;
    const float *a, *d, *dt_bias, *state_in;
    const int32_t *lengths;
    void *y;
    float *state_out, *ckpt;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-kLog2e * x)); }

// max(x, 0) + log(1 + e), e = exp(-|x|), with log(1 + e) = 2 atanh(s) at s = e / (2 + e) <= 1/3 by its series
// s + s^3/3 + ...: full relative precision for small steps, where 1 + e would have rounded e away; the terms left out
// are below 2^-26 of the sum.  NaN stays NaN.
__device__ __forceinline__ float softplus(float x) {
    const float e = ex2(-kLog2e * fabsf(x));
    const float s = e * rcp(2.f + e), q = s * s;
    float p = 1.f / 15.f;
    p = fmaf(p, q, 1.f / 13.f);
    p = fmaf(p, q, 1.f / 11.f);
    p = fmaf(p, q, 1.f / 9.f);
    p = fmaf(p, q, 1.f / 7.f);
    p = fmaf(p, q, 1.f / 5.f);
    p = fmaf(p, q, 1.f / 3.f);
    p = fmaf(p, q, 1.f);
    return (x > 0.f ? x : x < 0.f ? 0.f : x) + 2.f * s * p;
}

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
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

struct F4 {  // four states
    float2 lo, hi;
};
__device__ __forceinline__ F4 f4(float4 v) { return {make_float2(v.x, v.y), make_float2(v.z, v.w)}; }
__device__ __forceinline__ float4 f4(F4 v) { return make_float4(v.lo.x, v.lo.y, v.hi.x, v.hi.y); }
__device__ __forceinline__ F4 mul(F4 a, F4 b) { return {mul2(a.lo, b.lo), mul2(a.hi, b.hi)}; }
__device__ __forceinline__ F4 mul(float a, F4 b) { return {mul2(both(a), b.lo), mul2(both(a), b.hi)}; }
__device__ __forceinline__ F4 fma(F4 a, F4 b, F4 c) { return {fma2(a.lo, b.lo, c.lo), fma2(a.hi, b.hi, c.hi)}; }
__device__ __forceinline__ F4 fma(float a, F4 b, F4 c) { return {fma2(both(a), b.lo, c.lo), fma2(both(a), b.hi, c.hi)}; }
__device__ __forceinline__ F4 ex2(F4 v) { return {make_float2(ex2(v.lo.x), ex2(v.lo.y)), make_float2(ex2(v.hi.x), ex2(v.hi.y))}; }
__device__ __forceinline__ float dot(F4 a, F4 b) {
    const float2 s = fma2(a.lo, b.lo, mul2(a.hi, b.hi));
    return s.x + s.y;
}
__device__ __forceinline__ F4 zero4() { return {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}; }
__device__ __forceinline__ F4 one4() { return {make_float2(1.f, 1.f), make_float2(1.f, 1.f)}; }

// four states n .. n + 3 of a row of N (states past N are 0)
__device__ __forceinline__ F4 load4(const float *row, int n, int N) {
    if ((N & 3) == 0 && aligned16(row)) return n < N ? f4(*reinterpret_cast<const float4 *>(row + n)) : zero4();
    F4 v;
    v.lo.x = n < N ? row[n] : 0.f, v.lo.y = n + 1 < N ? row[n + 1] : 0.f;
    v.hi.x = n + 2 < N ? row[n + 2] : 0.f, v.hi.y = n + 3 < N ? row[n + 3] : 0.f;
    return v;
}
__device__ __forceinline__ void store4(float *row, int n, int N, F4 v) {
    if ((N & 3) == 0 && aligned16(row)) {
        if (n < N) *reinterpret_cast<float4 *>(row + n) = f4(v);
        return;
    }
    if (n < N) row[n] = v.lo.x;
    if (n + 1 < N) row[n + 1] = v.lo.y;
    if (n + 2 < N) row[n + 2] = v.hi.x;
    if (n + 3 < N) row[n + 3] = v.hi.y;
}

// Sums of eight values over L lanes that are STRIDE apart, all at once: at each step a lane hands half of the values it
// holds to its partner and keeps the other half, while it holds more than one.  Lane q of the L (their order is q) is
// left with values first(q) .. first(q) + kOut, at v[0 ..], each summed over the L lanes.
template <int L, int STRIDE>
struct LaneSum {
    static constexpr int kOut = L >= 8 ? 1 : 8 / L;
    __device__ static __forceinline__ int first(int q) {
        int f = 0, w = 8;
#pragma unroll
        for (int o = L / 2; o >= 1; o >>= 1)
            if (w > 1) {
                w >>= 1;
                if (q & o) f += w;
            }
        return f;
    }
    __device__ static __forceinline__ void run(float (&v)[8], int q) {
        int w = 8;
#pragma unroll
        for (int o = L / 2; o >= 1; o >>= 1) {
            if (w > 1) {
                w >>= 1;
                const bool upper = (q & o) != 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < w) {
                        const float send = upper ? v[i] : v[i + w], keep = upper ? v[i + w] : v[i];
                        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o * STRIDE);
                    }
            } else {
                v[0] += __shfl_xor_sync(0xffffffffu, v[0], o * STRIDE);
            }
        }
    }
};

__device__ __forceinline__ int64_t length_of(const int32_t *lengths, int64_t b, int64_t seq) {
    if (!lengths) return seq;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n > seq ? seq : n;
}

// Where a CTA works: its sequence, group, channels d0 .. d0 + nch.
struct Place {
    int64_t b, e, d0;
    int nch;
};
__device__ __forceinline__ Place place_of(int64_t block, const Params &p, int width) {
    Place q;
    const int64_t blocks = (p.per + width - 1) / width;
    const int64_t per_seq = blocks * p.groups;
    q.b = block / per_seq;
    const int64_t r = block - q.b * per_seq;
    q.e = r / blocks;
    const int64_t off = (r - q.e * blocks) * width;
    q.d0 = q.e * p.per + off;
    q.nch = p.per - off < width ? (int)(p.per - off) : width;
    return q;
}

// `rows` rows of 16 channels (nch of them real) from src (row stride st) into dst [rows][16]; rows from `live` on and
// missing channels are zeros.  The copies are asynchronous where vec says 16-byte copies are possible.
template <typename TI>
__device__ __forceinline__ void stage_x(TI *dst, const TI *src, int64_t st, int rows, int live, int nch, bool vec) {
    constexpr int kPer = kCh * sizeof(TI) / 16, kEl = 16 / sizeof(TI);
    if (vec && nch == kCh && aligned16(src)) {
        for (int i = threadIdx.x; i < rows * kPer; i += kThreads) {
            const int r = i / kPer, q = i % kPer;
            if (r < live) ptx::cp_async16(ptx::smem_u32(dst + r * kCh + q * kEl), src + r * st + q * kEl, 16u);
            else *reinterpret_cast<uint4 *>(dst + r * kCh + q * kEl) = make_uint4(0, 0, 0, 0);
        }
    } else {
        for (int i = threadIdx.x; i < rows * kCh; i += kThreads) {
            const int r = i / kCh, q = i % kCh;
            TI v;
            dc::st(&v, 0.f);
            if (r < live && q < nch) v = src[r * st + q];
            dst[i] = v;
        }
    }
}
// the same for `rows` rows of N states into dst [rows][NP] (columns from N on were zeroed once)
template <typename TI, int NP>
__device__ __forceinline__ void stage_bc(TI *dst, const TI *src, int64_t st, int rows, int live, int N, bool vec) {
    constexpr int kEl = 16 / sizeof(TI);
    if (vec && N % kEl == 0 && aligned16(src)) {
        const int per = N / kEl;
        for (int i = threadIdx.x; i < rows * per; i += kThreads) {
            const int r = i / per, q = i % per;
            if (r < live) ptx::cp_async16(ptx::smem_u32(dst + r * NP + q * kEl), src + r * st + q * kEl, 16u);
            else *reinterpret_cast<uint4 *>(dst + r * NP + q * kEl) = make_uint4(0, 0, 0, 0);
        }
    } else {
        for (int i = threadIdx.x; i < rows * NP; i += kThreads) {
            const int r = i / NP, q = i % NP;
            TI v;
            dc::st(&v, 0.f);
            if (r < live && q < N) v = src[r * st + q];
            dst[i] = v;
        }
    }
}

// ------------------------------------------------------------------------------------------------ forward
template <typename TI, int P>
struct FwdSmem {
    using T = Tile<P>;
    struct Raw {
        TI u[T::kTokens * kCh], dt[T::kTokens * kCh], z[T::kTokens * kCh];
        TI b[T::kTokens * T::kN], c[T::kTokens * T::kN];
    };
    Raw raw[2];
    float2 step[T::kTokens * kCh];  // (step, step * u)
    float4 b[T::kTokens * P], c[T::kTokens * P];
    float4 decay[kThreads], end[kThreads];  // each segment's product of decays and end state
    float y[T::kTokens * kCh];
};

template <typename TI, int P>
__global__ void __launch_bounds__(kThreads) scan_kernel(const Params p) {
    using T = Tile<P>;
    using Smem = FwdSmem<TI, P>;
    constexpr int kTok = T::kTokens, kLanes = kCh * P;
    extern __shared__ __align__(16) unsigned char smem_bytes[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_bytes);
    const int tid = threadIdx.x, seg = tid / kLanes, r = tid % kLanes, ch = r / P, q = r % P;
    const Place at = place_of(blockIdx.x, p, kCh);
    const int64_t len = length_of(p.lengths, at.b, p.seq);
    const int N = p.N;
    const TI *U = static_cast<const TI *>(p.u) + at.b * p.u_b + at.d0, *D = static_cast<const TI *>(p.dt) + at.b * p.dt_b + at.d0;
    const TI *Z = p.z ? static_cast<const TI *>(p.z) + at.b * p.z_b + at.d0 : nullptr;
    const TI *B = static_cast<const TI *>(p.b) + at.b * p.b_b + at.e * N, *C = static_cast<const TI *>(p.c) + at.b * p.c_b + at.e * N;

    auto load_tile = [&](int64_t t0, int s) {
        const int live = len - t0 < kTok ? (int)(len - t0) : kTok;
        typename Smem::Raw &w = sm.raw[s];
        stage_x(w.u, U + t0 * p.u_t, p.u_t, kTok, live, at.nch, p.vec_x);
        stage_x(w.dt, D + t0 * p.dt_t, p.dt_t, kTok, live, at.nch, p.vec_x);
        if (Z) stage_x(w.z, Z + t0 * p.z_t, p.z_t, kTok, live, at.nch, p.vec_x);
        stage_bc<TI, T::kN>(w.b, B + t0 * p.b_t, p.b_t, kTok, live, N, p.vec_bc);
        stage_bc<TI, T::kN>(w.c, C + t0 * p.c_t, p.c_t, kTok, live, N, p.vec_bc);
        ptx::cp_async_commit();
    };

    // the padding of b and c, zeroed once
    for (int i = tid; i < kTok * T::kN; i += kThreads)
        if (i % T::kN >= N)
#pragma unroll
            for (int s = 0; s < 2; ++s) st(&sm.raw[s].b[i], 0.f), st(&sm.raw[s].c[i], 0.f);

    const bool real = ch < at.nch;
    const int64_t d = at.d0 + (real ? ch : 0);
    const F4 a2 = real ? mul(kLog2e, load4(p.a + d * N, kS * q, N)) : zero4();
    F4 carry = zero4();
    if (p.state_in && real) carry = load4(p.state_in + (at.b * p.channels + d) * N, kS * q, N);
    // the output phase: this thread's pair of channels
    const int oc = 2 * (tid % (kCh / 2));
    const float bias_pre = p.dt_bias && tid % kCh < at.nch ? p.dt_bias[at.d0 + tid % kCh] : 0.f;
    const float d0v = p.d && oc < at.nch ? p.d[at.d0 + oc] : 0.f, d1v = p.d && oc + 1 < at.nch ? p.d[at.d0 + oc + 1] : 0.f;
    const int64_t y0 = at.b * p.y_b + at.d0 + oc;
    const int64_t ysize = p.y_dt ? 2 : 4;
    const bool ypair = oc + 1 < at.nch && (reinterpret_cast<uintptr_t>(p.y) + y0 * ysize) % (2 * ysize) == 0 && p.y_t % 2 == 0;
    auto put = [&](int64_t t, float v0, float v1) {
        const int64_t o = y0 + t * p.y_t;
        if (p.y_dt) {
            __nv_bfloat16 *Y = static_cast<__nv_bfloat16 *>(p.y) + o;
            if (ypair) *reinterpret_cast<uint32_t *>(Y) = vec::pack(v0, v1);
            else {
                if (oc < at.nch) st(Y, v0);
                if (oc + 1 < at.nch) st(Y + 1, v1);
            }
        } else {
            float *Y = static_cast<float *>(p.y) + o;
            if (ypair) *reinterpret_cast<float2 *>(Y) = make_float2(v0, v1);
            else {
                if (oc < at.nch) Y[0] = v0;
                if (oc + 1 < at.nch) Y[1] = v1;
            }
        }
    };

    if (len > 0) load_tile(0, 0);
    int s = 0;
    for (int64_t t0 = 0, tile = 0; t0 < len; t0 += kTok, ++tile, s ^= 1) {
        ptx::cp_async_wait<0>();
        __syncthreads();  // the tile has landed, and the last tile's shared values are done with
        if (t0 + kTok < len) load_tile(t0 + kTok, s ^ 1);
        const int live = len - t0 < kTok ? (int)(len - t0) : kTok;
        typename Smem::Raw &w = sm.raw[s];
        for (int i = tid; i < kTok * kCh; i += kThreads) {  // kThreads is a multiple of kCh: always the same channel
            float v = ld(&w.dt[i]) + bias_pre;
            if (p.softplus) v = softplus(v);
            if (i / kCh >= live) v = 0.f;  // past the end: decay 1, nothing added
            sm.step[i] = make_float2(v, v * ld(&w.u[i]));
        }
        {
            float *fb = reinterpret_cast<float *>(sm.b), *fc = reinterpret_cast<float *>(sm.c);
            for (int i = tid; i < kTok * T::kN; i += kThreads) fb[i] = ld(&w.b[i]), fc[i] = ld(&w.c[i]);
        }
        if (p.ckpt && seg == 0 && real) store4(p.ckpt + ((at.b * p.tiles + tile) * p.channels + d) * N, kS * q, N, carry);
        __syncthreads();

        F4 av[kK], bv[kK];
        F4 prod = one4(), h = zero4();
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            const int t = seg * kK + k;
            const float2 sd = sm.step[t * kCh + ch];
            av[k] = ex2(mul(sd.x, a2));
            bv[k] = mul(sd.y, f4(sm.b[t * P + q]));
            if constexpr (T::kSegs > 1) {
                prod = mul(prod, av[k]);
                h = fma(av[k], h, bv[k]);
            }
        }
        if constexpr (T::kSegs > 1) {
            sm.decay[tid] = f4(prod);
            sm.end[tid] = f4(h);
            __syncthreads();
            h = carry;
#pragma unroll
            for (int i = 0; i < T::kSegs; ++i) {
                if (i == seg) h = carry;
                carry = fma(f4(sm.decay[i * kLanes + r]), carry, f4(sm.end[i * kLanes + r]));
            }
        } else {
            h = carry;
        }
        float y[kK];
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            h = fma(av[k], h, bv[k]);
            y[k] = dot(h, f4(sm.c[(seg * kK + k) * P + q]));
        }
        if constexpr (T::kSegs == 1) carry = h;
        LaneSum<P, 1>::run(y, q);
        const int first = seg * kK + LaneSum<P, 1>::first(q);
#pragma unroll
        for (int k = 0; k < LaneSum<P, 1>::kOut; ++k) sm.y[(first + k) * kCh + ch] = y[k];
        __syncthreads();
        for (int i = tid; i < kTok * kCh / 2; i += kThreads) {
            const int t = i / (kCh / 2);
            if (t < live) {
                const float2 yv = *reinterpret_cast<const float2 *>(&sm.y[t * kCh + oc]);
                float v0 = fmaf(d0v, ld(&w.u[t * kCh + oc]), yv.x), v1 = fmaf(d1v, ld(&w.u[t * kCh + oc + 1]), yv.y);
                if (Z) {
                    const float z0 = ld(&w.z[t * kCh + oc]), z1 = ld(&w.z[t * kCh + oc + 1]);
                    v0 *= z0 * sigmoid(z0), v1 *= z1 * sigmoid(z1);
                }
                put(t0 + t, v0, v1);
            }
        }
    }
    if (p.state_out && seg == 0 && real) store4(p.state_out + (at.b * p.channels + d) * N, kS * q, N, carry);
    for (int64_t t = len + tid / (kCh / 2); t < p.seq; t += kThreads / (kCh / 2)) put(t, 0.f, 0.f);
}

// ------------------------------------------------------------------------------------------------ one token
// Four states per thread; HBM-bound (the state read and written once, 8 bytes per state, against 4 elements per channel).
template <typename TI, int P>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const Params p) {
    const int64_t i = (int64_t)blockIdx.x * (kThreads / P) + threadIdx.x / P;  // (sequence, channel)
    const int q = threadIdx.x % P, N = p.N;
    const bool on = i < p.batch * p.channels;
    const int64_t j = on ? i : 0, b = j / p.channels, d = j - b * p.channels, e = d / p.per;
    const F4 h0 = p.state_in ? load4(p.state_in + j * N, kS * q, N) : zero4();
    const F4 a2 = mul(kLog2e, load4(p.a + d * N, kS * q, N));
    const float u = ld(static_cast<const TI *>(p.u) + b * p.u_b + d);
    float step = ld(static_cast<const TI *>(p.dt) + b * p.dt_b + d) + (p.dt_bias ? p.dt_bias[d] : 0.f);
    if (p.softplus) step = softplus(step);
    const TI *B = static_cast<const TI *>(p.b) + b * p.b_b + e * N, *C = static_cast<const TI *>(p.c) + b * p.c_b + e * N;
    float bv[kS], cv[kS];
#pragma unroll
    for (int k = 0; k < kS; ++k) {
        bv[k] = kS * q + k < N ? ld(B + kS * q + k) : 0.f;
        cv[k] = kS * q + k < N ? ld(C + kS * q + k) : 0.f;
    }
    const F4 h = fma(ex2(mul(step, a2)), h0, mul(step * u, f4(make_float4(bv[0], bv[1], bv[2], bv[3]))));
    float y = dot(h, f4(make_float4(cv[0], cv[1], cv[2], cv[3])));
#pragma unroll
    for (int o = P / 2; o >= 1; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (!on) return;
    if (p.state_out) store4(p.state_out + j * N, kS * q, N, h);
    if (q == 0) {
        if (p.d) y = fmaf(p.d[d], u, y);
        if (p.z) {
            const float z = ld(static_cast<const TI *>(p.z) + b * p.z_b + d);
            y *= z * sigmoid(z);
        }
        if (p.y_dt) st(static_cast<__nv_bfloat16 *>(p.y) + b * p.y_b + d, y);
        else st(static_cast<float *>(p.y) + b * p.y_b + d, y);
    }
}

}  // namespace scan
}  // namespace dc
