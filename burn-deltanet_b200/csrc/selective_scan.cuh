// selective_scan.cuh — the selective state space scan over a prompt, and one decode tick of it.
//
//   step_t = softplus(dt_t + dt_bias)       h_n <- exp(step_t a_n) h_n + step_t u_t b_tn
//   y_t = (sum_n c_tn h_n + d u_t) z_t sigma(z_t)
//
// per (sequence, channel), `state` values of h.  The exponentials bound it: state + 4 of them and their like
// (softplus, silu) per (token, channel) at 16 a clock and SM, against 4 elements read or written.
//
// Layout.  A CTA owns a block of channels of one sequence and walks its tokens in tiles that it stages in shared memory
// (asynchronous copies, the next tile's under this one's arithmetic).  Four states of a channel live in a thread's
// registers, so a channel spans P = state / 4 threads (padded to a power of two, the padding with a = b = c = 0).  b and c
// of a tile are read once for the CTA's channels and kept in float32.
//
// Three ways along the time axis, chosen by how many channels there are to fill the card with (selective_scan.cu):
//   * walk: a thread walks its channel's tokens one by one.  Least work.
//   * segments: the CTA's W segments of threads take consecutive runs of K = 8 tokens.  The recurrence is linear, so each
//     segment first runs its tokens from zero while it keeps the decays and products in registers (every exponential is
//     still taken once), the segments exchange (product of decays, end state) through shared memory, and each runs its
//     tokens again from the state that reaches it, now reading out: about a third more instructions for W times the threads.
//   * pieces: the time axis cut over CTAs that walk: a first launch finds each piece's end state from zero and its sum of steps (whose
//     exponential is the product of its decays), the second starts each piece from what the pieces before it give and does
//     the work: nearly twice the exponentials, for sequences long enough and channels few enough.
#pragma once

#include <float.h>

#include "common.cuh"
#include "ptx.cuh"
#include "vec.cuh"

namespace dc {
namespace scan {

constexpr int kThreads = 256;  // of the step
constexpr int kK = 8;          // tokens of a segment
constexpr int kS = 4;          // states of a thread
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

constexpr int kTile = 16;  // tokens of the walk's and the backward's tiles, and between two checkpoints

struct Params {
    int64_t batch, seq, channels, groups, per;  // per: channels of a group
    int32_t N;
    int64_t u_b, u_t, dt_b, dt_t, z_b, z_t, b_b, b_t, c_b, c_t, y_b, y_t;
    int32_t softplus, y_dt;
    int32_t vec_x, vec_bc;  // how the channel rows / the b and c rows may be copied (kVectors, kWords, kScalar)
    int32_t tiles;          // checkpoints of a sequence
    int32_t pieces;         // pieces of the time axis, `piece` tokens each (a multiple of every tile's)
    int64_t piece;
    const void *u, *dt, *z, *b, *c;
    const float *a, *d, *dt_bias, *state_in;
    const int32_t *lengths;
    void *y;
    float *state_out, *ckpt;
    float *piece_end;   // [batch, pieces, channels, N]: the state before the first token, then the pieces' end states from zero
    float *piece_step;  // [batch, pieces - 1, channels]: their sums of steps
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

using vec::both;
using vec::fma2;
using vec::mul2;

// max(x, 0) + log(1 + e), e = exp(-|x|), with log(1 + e) = 2 atanh(s) at s = e / (2 + e) <= 1/3 by its series
// s + s^3/3 + ... + s^11/11: full relative precision for small steps, where 1 + e would have rounded e away; the terms
// left out are below 1.6e-7 of the sum (at x = 0, and far less elsewhere).  Two at a time.  NaN stays NaN (through e).
__device__ __forceinline__ float2 softplus2(float2 x) {
    const float2 e = make_float2(ex2(-kLog2e * fabsf(x.x)), ex2(-kLog2e * fabsf(x.y)));
    const float2 s = mul2(e, make_float2(rcp(2.f + e.x), rcp(2.f + e.y))), q = mul2(s, s);
    float2 p = fma2(both(1.f / 11.f), q, both(1.f / 9.f));
    p = fma2(p, q, both(1.f / 7.f));
    p = fma2(p, q, both(1.f / 5.f));
    p = fma2(p, q, both(1.f / 3.f));
    p = fma2(p, q, both(1.f));
    return fma2(mul2(both(2.f), s), p, make_float2(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)));
}
__device__ __forceinline__ float softplus(float x) { return softplus2(make_float2(x, x)).x; }

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
// exp2(step * a2).  ex2.approx comes out 2e-8 low on average for arguments just below 0 (measured over [-0.2, 0]), and a state
// that remembers many tokens multiplies that up: 2^-25 in the exponent takes it off, where the argument is small enough to
// hold it.  (8 x 98 x 219 x 16 in float32, final state against 64 bits: 1.4e-6 without it, 5.6e-7 with.)  At step 0 it leaves 1.
constexpr float kTilt = 1.f / (1 << 25);
// a log2(e), held inside float32's range: a rate of -inf or near the lowest value, which switches a state off, would give -inf,
// and a step of 0 (a token behind the end, or one whose softplus vanishes) times that NaN.  So the decay is 0 for every other
// step and 1 for those.  NaN stays NaN.
__device__ __forceinline__ float rate(float a) {
    const float r = kLog2e * a;
    return r < -FLT_MAX ? -FLT_MAX : r > FLT_MAX ? FLT_MAX : r;
}
__device__ __forceinline__ F4 rates(F4 a) {
    return {make_float2(rate(a.lo.x), rate(a.lo.y)), make_float2(rate(a.hi.x), rate(a.hi.y))};
}
__device__ __forceinline__ F4 decays(float step, F4 a2) { return ex2(fma(step, a2, F4{both(kTilt), both(kTilt)})); }
__device__ __forceinline__ float dot(F4 a, F4 b) {
    const float2 s = fma2(a.lo, b.lo, mul2(a.hi, b.hi));
    return s.x + s.y;
}
__device__ __forceinline__ F4 zero4() { return {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}; }

// four values in shared memory
template <typename T>
__device__ __forceinline__ F4 four(const T *p) {
    float v[kS];
    vec::load<true>(p, v);
    return {make_float2(v[0], v[1]), make_float2(v[2], v[3])};
}

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

// How a tensor's rows may be copied, from their strides (and, for the first of these, a 16-byte first row).
enum : int { kScalar = 0, kWords = 1, kVectors = 2 };  // one by one; asynchronously, 4 bytes or 16 at a time

// ROWS rows of W values (`width` of them real) from src (row stride st) into dst [ROWS][W], by NT threads of which this is
// the tid-th; rows from `live` on and missing values are zeros.
template <int NT, int W, int ROWS, typename TI>
__device__ __forceinline__ void stage(TI *dst, const TI *src, int64_t st, int live, int width, int how, int tid) {
    constexpr int kEl = 16 / sizeof(TI), kPer = W >= kEl ? W / kEl : 1, kWord = 4 / sizeof(TI);
    if (W % kEl == 0 && how == kVectors && aligned16(src)) {
#pragma unroll 1
        for (int i = tid; i < ROWS * kPer; i += NT) {
            const int r = i / kPer, q = i % kPer, left = (width - q * kEl) * (int)sizeof(TI);
            const bool on = r < live && left > 0;
            ptx::cp_async16(ptx::smem_u32(dst + i * kEl), on ? src + r * st + q * kEl : src, !on ? 0u : left > 16 ? 16u : (uint32_t)left);
        }
    } else if (how >= kWords && (reinterpret_cast<uintptr_t>(src) & 3) == 0) {
#pragma unroll 4
        for (int i = tid; i < ROWS * W / kWord; i += NT) {
            const int r = i / (W / kWord), q = i % (W / kWord), left = (width - q * kWord) * (int)sizeof(TI);
            const bool on = r < live && left > 0;
            ptx::cp_async4(ptx::smem_u32(dst + i * kWord), on ? src + r * st + q * kWord : src, !on ? 0u : left > 4 ? 4u : (uint32_t)left);
        }
    } else {
        constexpr int kBatch = 8;  // loads under way together
#pragma unroll 1
        for (int i0 = tid; i0 < ROWS * W; i0 += kBatch * NT) {
            TI v[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int i = i0 + k * NT, r = i / W, q = i % W;
                dc::st(&v[k], 0.f);
                if (r < live && q < width) v[k] = src[r * st + q];
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
                if (i0 + k * NT < ROWS * W) dst[i0 + k * NT] = v[k];
        }
    }
}
// `n` values (a multiple of 4) in shared memory to float32, by NT threads
template <int NT, typename TI>
__device__ __forceinline__ void widen(float4 *dst, const TI *src, int n, int tid) {
#pragma unroll 2
    for (int i = tid; i < n / 4; i += NT) {
        float v[4];
        vec::load<true>(src + 4 * i, v);
        dst[i] = make_float4(v[0], v[1], v[2], v[3]);
    }
}

// ------------------------------------------------------------------------------------------------ forward
// What both forward kernels know about their CTA: where it works, and how it stages a tile and writes y.
template <typename TI, int CH, int N4>
struct Work {
    const Params &p;
    Place at;
    int64_t first, last, len;  // this CTA's tokens, and where those inside the sequence end
    const TI *U, *D, *Z, *B, *C;

    __device__ __forceinline__ Work(const Params &p, int64_t block, int64_t pieces) : p(p) {
        const int64_t piece = pieces > 1 ? block % pieces : 0;
        at = place_of(pieces > 1 ? block / pieces : block, p, CH);
        const int64_t all = length_of(p.lengths, at.b, p.seq);
        first = piece * p.piece;
        last = p.pieces > 1 && first + p.piece < p.seq ? first + p.piece : p.seq;
        len = all < last ? all : last;
        U = static_cast<const TI *>(p.u) + at.b * p.u_b + at.d0, D = static_cast<const TI *>(p.dt) + at.b * p.dt_b + at.d0;
        Z = p.z ? static_cast<const TI *>(p.z) + at.b * p.z_b + at.d0 : nullptr;
        B = static_cast<const TI *>(p.b) + at.b * p.b_b + at.e * p.N, C = static_cast<const TI *>(p.c) + at.b * p.c_b + at.e * p.N;
    }
    template <int NT, int TOK, bool FULL, typename Raw>
    __device__ __forceinline__ void load(Raw &w, int64_t t0, int tid) const {
        const int live = len - t0 < TOK ? (int)(len - t0) : TOK;
        stage<NT, CH, TOK>(w.dt, D + t0 * p.dt_t, p.dt_t, live, at.nch, p.vec_x, tid);
        stage<NT, CH, TOK>(w.u, U + t0 * p.u_t, p.u_t, live, at.nch, p.vec_x, tid);
        stage<NT, N4, TOK>(w.b, B + t0 * p.b_t, p.b_t, live, p.N, p.vec_bc, tid);
        if (FULL) {
            stage<NT, N4, TOK>(w.c, C + t0 * p.c_t, p.c_t, live, p.N, p.vec_bc, tid);
            if (Z) stage<NT, CH, TOK>(w.z, Z + t0 * p.z_t, p.z_t, live, at.nch, p.vec_x, tid);
        }
    }
};

// The part of a tile's work that goes by token and channel, four channels of a token at a time: the steps before the
// recurrence, the skip and the gate after it.  A thread of NT always has the same four channels.
template <typename TI, int P, int CH, int TOK, int NT>
struct Quads {
    static constexpr int kQuads = CH / 4, kRows = NT / kQuads;
    static_assert(NT % kQuads == 0, "one quad of channels per thread");
    const Params &p;
    int oc, orow, ny, nch;
    float bias[4], skip[4];
    int64_t y0;
    bool yquad;

    __device__ __forceinline__ Quads(const Params &p, const Place &at, int tid) : p(p) {
        oc = 4 * (tid % kQuads), orow = tid / kQuads, nch = at.nch;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bias[j] = p.dt_bias && oc + j < at.nch ? p.dt_bias[at.d0 + oc + j] : 0.f;
            skip[j] = p.d && oc + j < at.nch ? p.d[at.d0 + oc + j] : 0.f;
        }
        y0 = at.b * p.y_b + at.d0 + oc;
        const int ysize = p.y_dt ? 2 : 4;
        ny = at.nch - oc;  // channels of the quad that exist (<= 0: none)
        yquad = ny >= 4 && (reinterpret_cast<uintptr_t>(p.y) + y0 * ysize) % (4 * ysize) == 0 && p.y_t % 4 == 0;
    }
    __device__ __forceinline__ void put(int64_t t, const float (&v)[4]) const {
        if (yquad) vec::store_as<true>(p.y_dt, p.y, y0 + t * p.y_t, v);
        else vec::store_as<false>(p.y_dt, p.y, y0 + t * p.y_t, v, ny);
    }
    // raw dt and u of a token to (step, step * u)
    __device__ __forceinline__ void step_of(float2 *step, float (&v)[4], const float (&x)[4], bool live) const {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            float2 f = make_float2(v[j] + bias[j], v[j + 1] + bias[j + 1]);
            if (p.softplus) f = softplus2(f);
            v[j] = live ? f.x : 0.f, v[j + 1] = live ? f.y : 0.f;  // past the end: decay 1, nothing added
        }
        float4 *o = reinterpret_cast<float4 *>(step);
        o[0] = make_float4(v[0], v[0] * x[0], v[1], v[1] * x[1]);
        o[1] = make_float4(v[2], v[2] * x[2], v[3], v[3] * x[3]);
    }
    // a token's y, from the P shares of it: y[token][state group][channel]
    __device__ __forceinline__ void sum_of(const float *y, int t, float (&v)[4]) const {
        // from another share on in each token, so that a warp's reads meet in no bank
        const float *row = y + t * CH * P + oc;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float4 f = *reinterpret_cast<const float4 *>(row + ((i + t) & (P - 1)) * CH);
            v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
        }
    }
    __device__ __forceinline__ void finish(float (&v)[4], const float (&x)[4], const float (&z)[4], bool gated) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = fmaf(skip[j], x[j], v[j]);
            if (gated) v[j] *= z[j] * sigmoid(z[j]);
        }
    }
    __device__ __forceinline__ void steps(float2 *step, const TI *dt, const TI *u, int live) const {
#pragma unroll 2
        for (int t = orow; t < TOK; t += kRows) {
            float v[4], x[4];
            vec::load<true>(dt + t * CH + oc, v);
            vec::load<true>(u + t * CH + oc, x);
            step_of(step + t * CH + oc, v, x, t < live);
        }
    }
    __device__ __forceinline__ void outputs(const float *y, const TI *u, const TI *z, int64_t t0, int live) const {
#pragma unroll 2
        for (int t = orow; t < live; t += kRows) {
            float v[4] = {0.f, 0.f, 0.f, 0.f}, x[4], g[4];
            sum_of(y, t, v);
            vec::load<true>(u + t * CH + oc, x);
            if (z) vec::load<true>(z + t * CH + oc, g);
            finish(v, x, g, z != nullptr);
            put(t0 + t, v);
        }
    }
    __device__ __forceinline__ void zeros(int64_t from, int64_t to) const {
        const float none[4] = {0.f, 0.f, 0.f, 0.f};
        for (int64_t t = from + orow; t < to; t += kRows) put(t, none);
    }
};

template <typename TI, int CH, int TOK, int N4>
struct RawTile {
    TI u[TOK * CH], dt[TOK * CH], z[TOK * CH];
    TI b[TOK * N4], c[TOK * N4];
};

__device__ __forceinline__ void checkpoint(const Params &p, const Place &at, int64_t t, int64_t d, int q, F4 h) {
    store4(p.ckpt + ((at.b * p.tiles + t / kTile) * p.channels + d) * p.N, kS * q, p.N, h);
}

// A thread's share of the 16-byte copies of a tile, where the rows start on 16-byte boundaries: the sources move on by one
// tile a call.  What a row lacks of its last copies (missing channels, padding states) is filled with zeros.
template <typename TI, int CH, int N4, int TOK, int NT, bool FULL>
struct Stager {
    static constexpr int kEs = sizeof(TI), kEl = 16 / kEs, kXRow = CH / kEl, kBRow = N4 >= kEl ? N4 / kEl : 1;  // copies per row
    static constexpr int kX = TOK * kXRow, kB = TOK * kBRow;                                                    // and per tensor
    static constexpr int kAll = FULL ? 3 * kX + 2 * kB : 2 * kX + kB, kEach = (kAll + NT - 1) / NT;
    const char *src[kEach];
    int32_t step[kEach];    // bytes a tile
    uint32_t where[kEach];  // the copy's place in the tile | its row << 16 (TOK: none) | its bytes << 24, to save registers
    bool on;
    static_assert(kAll <= 65536 && TOK < 256, "they fit");

    __device__ __forceinline__ Stager(const Work<TI, CH, N4> &wk, int tid) {
        const Params &p = wk.p;
        on = p.vec_x == kVectors && p.vec_bc == kVectors && N4 % kEl == 0 && (!FULL || wk.Z) && aligned16(wk.U) && aligned16(wk.D) && aligned16(wk.B) &&
             (!FULL || (aligned16(wk.Z) && aligned16(wk.C)));
        const int64_t strides[] = {p.u_t, p.dt_t, p.b_t, FULL ? p.c_t : 0, FULL ? p.z_t : 0};
#pragma unroll
        for (int k = 0; k < 5; ++k) on = on && strides[k] >= 0 && strides[k] <= INT32_MAX / (TOK * kEs);
        if (!on) return;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            int c = tid + j * NT, base = 0, per = kXRow, width = wk.at.nch;  // tensors in RawTile's order: u, dt, (z,) b, (c)
            const bool used = c < kAll;
            const TI *t = wk.U;
            int64_t st = p.u_t;
            auto next = [&](int count, int at, int row_copies, int w, const TI *tensor, int64_t stride) {
                if (c < count) return false;
                c -= count, base = at, per = row_copies, width = w, t = tensor, st = stride;
                return true;
            };
            if (next(kX, kX, kXRow, wk.at.nch, wk.D, p.dt_t)) {
                if (FULL) {
                    if (next(kX, 2 * kX, kXRow, wk.at.nch, wk.Z, p.z_t) && next(kX, 3 * kX, kBRow, p.N, wk.B, p.b_t))
                        next(kB, 3 * kX + kB, kBRow, p.N, wk.C, p.c_t);
                } else {
                    next(kX, 3 * kX, kBRow, p.N, wk.B, p.b_t);
                }
            }
            const int r = used ? c / per : 0, q = used ? c % per : 0, left = (width - q * kEl) * kEs;
            const int bytes = left < 0 ? 0 : left > 16 ? 16 : left;
            where[j] = (uint32_t)(base + (used ? c : 0)) | (uint32_t)(used ? r : TOK) << 16 | (uint32_t)bytes << 24;
            src[j] = reinterpret_cast<const char *>(t + (wk.first + r) * st + (bytes ? q * kEl : 0));
            step[j] = (int32_t)(st * (TOK * kEs));
        }
    }
    template <typename Raw>
    __device__ __forceinline__ void copy(Raw &raw, int live) {
        const uint32_t to = ptx::smem_u32(&raw);
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            // past the end: no bytes, from the tile's first row, which is always inside the sequence
            const int row = (int)(where[j] >> 16 & 255);
            const bool real = row < live;
            if (row < TOK) ptx::cp_async16(to + (where[j] & 65535) * 16, real ? src[j] : src[j] - step[j] / TOK * row, real ? where[j] >> 24 : 0);
            src[j] += step[j];
        }
    }
};

// ---- token by token.  A thread of the recurrence has four states of one channel (of two where a warp would not be full, or
// where the threads would be too many for their registers).  kHelp further threads stage the tiles, take the steps of the
// next tile and write y of the last one, so that the two kinds of work, each a chain of dependent instructions, fill each
// other's gaps; one barrier per tile of 16 tokens.  8 x 4096 x 2048 x 16 bfloat16 takes 463 us: the special-function unit,
// the issue slots and the shared memory's data path are at 0.64, 0.65 and 0.72 of their rates there (294 us for the first
// alone), and what shortens one lengthens another: exponentials taken ahead of their use 495 us, b and c read as bfloat16 and widened by
// the reader 498, steps stored twice to spare the moves of two-wide arithmetic 596.  5 x 777 x 1000 x 24 float32 in 2 groups:
// 69 us, the longest sequence's chain of dependent instructions, 0.09 us a token.
// FULL: the whole scan; else only the piece's end state from zero and its sum of steps.
constexpr int walk_channels(int lanes) { return lanes >= 4 ? 16 : 64 / lanes; }       // of a CTA: a warp's at least
constexpr int walk_each(int lanes) { return lanes == 1 || lanes == 16 ? 2 : 1; }     // channels of a thread of the recurrence
// CTAs of an SM, by their registers and shared memory (float32 inputs take twice the staging space and more addresses).
constexpr int walk_ctas(int lanes, int64_t bytes) {
    return lanes == 4 ? (bytes == 2 ? 7 : 6) : lanes == 8 ? (bytes == 2 ? 4 : 3) : lanes == 16 ? (bytes == 2 ? 3 : 2) : lanes == 2 ? 4 : 2;
}
template <int P>
struct WalkShape {
    static constexpr int kCh = walk_channels(P), kV = walk_each(P), kMain = kCh * P / kV, kHelp = 4 * kCh, kNT = kMain + kHelp;
    static constexpr int kTok = kTile, kStages = 4, kN = kS * P;
};
template <typename TI, int P>
struct WalkSmem {
    using S = WalkShape<P>;
    // b and c of 16 bits once more in float32: the recurrence reads them for every channel (read as they are, and widened
    // there: slower, as above)
    static constexpr bool kWiden = sizeof(TI) < 4;
    RawTile<TI, S::kCh, S::kTok, S::kN> raw[S::kStages];
    float2 step[2][S::kTok * S::kCh];  // (step, step * u)
    float4 b[kWiden ? 2 : 1][kWiden ? S::kTok * P : 1], c[kWiden ? 2 : 1][kWiden ? S::kTok * P : 1];
    float y[2][S::kTok * S::kCh * P];
};

template <typename TI, int P, bool FULL>
__global__ void __launch_bounds__(WalkShape<P>::kNT, walk_ctas(P, sizeof(TI))) scan_walk_kernel(const Params p) {
    using S = WalkShape<P>;
    constexpr int V = S::kV, kTok = S::kTok, CH = S::kCh, kBatch = 4;
    extern __shared__ __align__(16) unsigned char smem_bytes[];
    WalkSmem<TI, P> &sm = *reinterpret_cast<WalkSmem<TI, P> *>(smem_bytes);
    constexpr bool kWiden = WalkSmem<TI, P>::kWiden;
    const int64_t pieces = FULL ? p.pieces : p.pieces - 1;  // nothing follows the last piece's end
    const Work<TI, CH, S::kN> wk(p, blockIdx.x, pieces);
    const Place &at = wk.at;
    const int64_t first = wk.first, len = wk.len;
    const int n = len > first ? (int)((len - first + kTok - 1) / kTok) : 0;  // tiles

    if (threadIdx.x >= S::kMain) {
        const int tid = threadIdx.x - S::kMain;
        const Quads<TI, P, CH, kTok, S::kHelp> quads(p, at, tid);
        Stager<TI, CH, S::kN, kTok, S::kHelp, FULL> stager(wk, tid);
        static_assert(kTok == decltype(quads)::kRows, "a helper has one token of a tile");
        constexpr int kQuad = kTok * S::kN / 4, kBc = kWiden ? (kQuad + S::kHelp - 1) / S::kHelp : 0;  // quads of b in a tile, a helper's
        const int end = n > 0 ? (int)(len - first - (int64_t)(n - 1) * kTok) : 0, row = quads.orow * CH + quads.oc;
        auto live = [&](int i) { return i + 1 < n ? kTok : end; };
        auto load = [&](int i) {
            if (i < n) {
                if (stager.on) stager.copy(sm.raw[i & (S::kStages - 1)], live(i));
                else wk.template load<S::kHelp, kTok, FULL>(sm.raw[i & (S::kStages - 1)], first + (int64_t)i * kTok, tid);
            }
            ptx::cp_async_commit();
        };
        // One token and four channels of tile i - 1's outputs and of tile i + 1's steps: two chains of dependent
        // instructions in one stretch of code, the loads of both in front.
        auto turn = [&](int i, bool before, bool after) {
            const auto &w = sm.raw[(i + 1) & (S::kStages - 1)], &o = sm.raw[(i - 1) & (S::kStages - 1)];
            float v[4] = {0.f, 0.f, 0.f, 0.f}, x[4], z[4], f[4], g[4], bv[kBc + 1][4], cv[kBc + 1][4];
            if (FULL && before) {
                quads.sum_of(sm.y[(i - 1) & 1], quads.orow, v);
                vec::load<true>(o.u + row, x);
                vec::load<true>(o.z + row, z);  // (nothing of use without a gate)
            }
            if (after) {
                vec::load<true>(w.dt + row, f);
                vec::load<true>(w.u + row, g);
#pragma unroll
                for (int j = 0; j < kBc; ++j)
                    if (kQuad % S::kHelp == 0 || tid + j * S::kHelp < kQuad) {
                        vec::load<true>(w.b + 4 * (tid + j * S::kHelp), bv[j]);
                        if (FULL) vec::load<true>(w.c + 4 * (tid + j * S::kHelp), cv[j]);
                    }
                quads.step_of(sm.step[(i + 1) & 1] + row, f, g, quads.orow < live(i + 1));
            }
            if (FULL && before) {
                quads.finish(v, x, z, wk.Z != nullptr);
                quads.put(first + (int64_t)(i - 1) * kTok + quads.orow, v);
            }
            if (after) {
#pragma unroll
                for (int j = 0; j < kBc; ++j)
                    if (kQuad % S::kHelp == 0 || tid + j * S::kHelp < kQuad) {
                        sm.b[(i + 1) & 1][tid + j * S::kHelp] = make_float4(bv[j][0], bv[j][1], bv[j][2], bv[j][3]);
                        if (FULL) sm.c[(i + 1) & 1][tid + j * S::kHelp] = make_float4(cv[j][0], cv[j][1], cv[j][2], cv[j][3]);
                    }
            }
        };
        load(0);
        load(1);
        ptx::cp_async_wait<0>();
        ptx::named_sync(1, S::kHelp);  // every helper's copies
        if (n > 0) turn(-1, false, true);
        __syncthreads();
        for (int i = 0; i < n; ++i) {
            load(i + 2);
            if (FULL && i > 0 && i + 1 < n) turn(i, true, true);
            else if (i + 1 < n) turn(i, false, true);
            else if (FULL && i > 0) turn(i, true, false);
            ptx::cp_async_wait<0>();
            __syncthreads();
        }
        if (FULL && n > 0) {
            const auto &w = sm.raw[(n - 1) & (S::kStages - 1)];
            quads.outputs(sm.y[(n - 1) & 1], w.u, wk.Z ? w.z : nullptr, first + (int64_t)(n - 1) * kTok, end);
        }
        if (FULL) quads.zeros(len > first ? len : first, wk.last);
        return;
    }

    const int ch = V * (threadIdx.x % (CH / V)), q = threadIdx.x / (CH / V), N = p.N;
    const int64_t d = at.d0 + ch, piece = pieces > 1 ? blockIdx.x % pieces : 0;
    bool real[V];
    F4 a2[V], h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        real[j] = ch + j < at.nch;
        a2[j] = real[j] ? rates(load4(p.a + (d + j) * N, kS * q, N)) : zero4();
        h[j] = zero4();
        if (FULL && p.pieces > 1 && real[j]) {  // what the pieces before this one make of the first state
            const int64_t at_end = at.b * p.pieces * p.channels + d + j, at_step = at.b * (p.pieces - 1) * p.channels + d + j;
            h[j] = load4(p.piece_end + at_end * N, kS * q, N);
#pragma unroll 4
            for (int64_t i = 0; i < piece; ++i)
                h[j] = fma(ex2(mul(p.piece_step[at_step + i * p.channels], a2[j])), h[j],
                           load4(p.piece_end + (at_end + (i + 1) * p.channels) * N, kS * q, N));
        } else if (FULL && p.state_in && real[j]) {
            h[j] = load4(p.state_in + (at.b * p.channels + d + j) * N, kS * q, N);
        }
    }
    float steps[V] = {};
    __syncthreads();
    for (int i = 0; i < n; ++i) {
        const float2 *step = sm.step[i & 1] + ch;
        const auto &raw = sm.raw[i & (S::kStages - 1)];
        const float *b = reinterpret_cast<const float *>(kWiden ? (const void *)sm.b[i & 1] : (const void *)raw.b) + kS * q;
        const float *c = reinterpret_cast<const float *>(kWiden ? (const void *)sm.c[i & 1] : (const void *)raw.c) + kS * q;
        float *y = sm.y[i & 1] + q * CH + ch;
        if (FULL && p.ckpt)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (real[j]) checkpoint(p, at, first + (int64_t)i * kTok, d + j, q, h[j]);
#pragma unroll 1
        for (int k0 = 0; k0 < kTok; k0 += kK) {
#pragma unroll
            for (int k1 = 0; k1 < kK; k1 += kBatch) {
                F4 av[kBatch][V], bv[kBatch][V];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int t = k0 + k1 + k;
                    float sd[2 * V];  // each channel's (step, step * u)
                    vec::load<true>(&step[t * CH].x, sd);
                    const F4 bt = four(b + t * S::kN);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        av[k][j] = decays(sd[2 * j], a2[j]), bv[k][j] = mul(sd[2 * j + 1], bt);
                        if (!FULL) steps[j] += sd[2 * j];
                    }
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int t = k0 + k1 + k;
                    float sum[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) h[j] = fma(av[k][j], h[j], bv[k][j]);
                    if (FULL) {
                        const F4 ct = four(c + t * S::kN);
#pragma unroll
                        for (int j = 0; j < V; ++j) sum[j] = dot(h[j], ct);
                        if constexpr (V == 2) *reinterpret_cast<float2 *>(y + t * CH * P) = make_float2(sum[0], sum[1]);
                        else y[t * CH * P] = sum[0];
                    }
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (!real[j]) continue;
        const int64_t own = (at.b * p.channels + d + j) * N;
        if (FULL) {
            if (p.state_out && piece == p.pieces - 1) store4(p.state_out + own, kS * q, N, h[j]);
            continue;
        }
        const int64_t row = at.b * p.pieces * p.channels + d + j;
        store4(p.piece_end + (row + (piece + 1) * p.channels) * N, kS * q, N, h[j]);
        if (q == 0) p.piece_step[(at.b * (p.pieces - 1) + piece) * p.channels + d + j] = steps[j];
        // the first state is kept with them: the second launch may overwrite state_in (state_out == state_in)
        if (piece == 0) store4(p.piece_end + row * N, kS * q, N, p.state_in ? load4(p.state_in + own, kS * q, N) : zero4());
    }
}

// ---- segments side by side: CH channels of P threads each, W segments of them; kSub tokens go by between two exchanges,
// kTok between two stagings.
template <int P>
struct SegShape {
    static constexpr int kCh = 8, kW = P == 1 ? 16 : 32 / P, kLanes = kCh * P, kNT = kLanes * kW;
    static constexpr int kSub = kW * kK, kTok = kSub < 32 ? 32 : kSub, kN = kS * P;
};
template <typename TI, int P>
struct SegSmem {
    using S = SegShape<P>;
    RawTile<TI, S::kCh, S::kTok, S::kN> raw[2];
    float2 step[S::kTok * S::kCh];  // (step, step * u)
    float4 b[S::kTok * P], c[S::kTok * P];
    float y[S::kTok * S::kLanes];
    float4 decay[S::kNT], end[S::kNT];  // each segment's product of decays and end state
};

template <typename TI, int P>
__global__ void __launch_bounds__(SegShape<P>::kNT, 512 / SegShape<P>::kNT) scan_segments_kernel(const Params p) {
    using S = SegShape<P>;
    constexpr int kTok = S::kTok, CH = S::kCh, kLanes = S::kLanes, kNT = S::kNT, W = S::kW;
    extern __shared__ __align__(16) unsigned char smem_bytes[];
    SegSmem<TI, P> &sm = *reinterpret_cast<SegSmem<TI, P> *>(smem_bytes);
    const int tid = threadIdx.x, seg = tid / kLanes, r = tid % kLanes, ch = r % CH, q = r / CH, N = p.N;
    const Work<TI, CH, S::kN> wk(p, blockIdx.x, 1);
    const Place &at = wk.at;
    const int64_t len = wk.len;
    const Quads<TI, P, CH, kTok, kNT> quads(p, at, tid);
    auto prepare = [&](int64_t t0, int s) {
        const auto &w = sm.raw[s];
        quads.steps(sm.step, w.dt, w.u, len - t0 < kTok ? (int)(len - t0) : kTok);
        widen<kNT>(sm.b, w.b, kTok * S::kN, tid);
        widen<kNT>(sm.c, w.c, kTok * S::kN, tid);
    };
    const bool real = ch < at.nch;
    const int64_t d = at.d0 + (real ? ch : 0);
    const F4 a2 = real ? rates(load4(p.a + d * N, kS * q, N)) : zero4();
    F4 carry = p.state_in && real ? load4(p.state_in + (at.b * p.channels + d) * N, kS * q, N) : zero4();
    if (len > 0) {
        wk.template load<kNT, kTok, true>(sm.raw[0], 0, tid);
        ptx::cp_async_commit();
        ptx::cp_async_wait<0>();
        __syncthreads();
        prepare(0, 0);
    } else {
        __syncthreads();  // every segment has read the state, which may be written below
    }
    int s = 0;
    for (int64_t t0 = 0; t0 < len; t0 += kTok, s ^= 1) {
        __syncthreads();  // this tile's values are ready, the other stage is free
        if (t0 + kTok < len) wk.template load<kNT, kTok, true>(sm.raw[s ^ 1], t0 + kTok, tid);
        ptx::cp_async_commit();
        const int live = len - t0 < kTok ? (int)(len - t0) : kTok;
#pragma unroll 1
        for (int sub = 0; sub < kTok; sub += S::kSub) {
            const int k0 = sub + seg * kK;  // this segment's first token
            F4 av[kK], bv[kK], prod, h;
#pragma unroll
            for (int k = 0; k < kK; ++k) {
                const int t = k0 + k;
                const float2 sd = sm.step[t * CH + ch];
                av[k] = decays(sd.x, a2);
                bv[k] = mul(sd.y, f4(sm.b[t * P + q]));
                prod = k ? mul(prod, av[k]) : av[k];
                h = k ? fma(av[k], h, bv[k]) : bv[k];
            }
            sm.decay[tid] = f4(prod);
            sm.end[tid] = f4(h);
            __syncthreads();
            h = carry;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if (i == seg) h = carry;
                carry = fma(f4(sm.decay[i * kLanes + r]), carry, f4(sm.end[i * kLanes + r]));
            }
            if (p.ckpt && real && k0 < live && (t0 + k0) % kTile == 0) checkpoint(p, at, t0 + k0, d, q, h);
            float *y = sm.y + k0 * kLanes + r;
#pragma unroll
            for (int k = 0; k < kK; ++k) {
                h = fma(av[k], h, bv[k]);
                y[k * kLanes] = dot(h, f4(sm.c[(k0 + k) * P + q]));
            }
            if (sub + S::kSub < kTok) __syncthreads();  // decay and end have been read
        }
        ptx::cp_async_wait<0>();
        __syncthreads();  // this tile's y is complete, the next tile has landed
        quads.outputs(sm.y, sm.raw[s].u, wk.Z ? sm.raw[s].z : nullptr, t0, live);
        if (t0 + kTok < len) prepare(t0 + kTok, s ^ 1);
    }
    if (p.state_out && seg == 0 && real) store4(p.state_out + (at.b * p.channels + d) * N, kS * q, N, carry);
    quads.zeros(len, wk.last);
}

// ------------------------------------------------------------------------------------------------ one token
// four values n .. n + 3 of a row of N of type T (values past N are 0); WHOLE: all four there and aligned
template <bool WHOLE, typename T>
__device__ __forceinline__ F4 load4_as(const T *row, int n, int N) {
    float v[4];
    if (WHOLE) vec::load<true>(row + n, v);
    else vec::load<false>(row + n, v, N - n);
    return f4(make_float4(v[0], v[1], v[2], v[3]));
}

// Four states of one channel per thread, for SEQS sequences, whose states are all under way together; HBM-bound (the state
// read and written once, 8 bytes per state, against 4 elements per channel).  A channel's P threads share out what is per
// sequence: the step, the gate and the output.  256 x 2048 x 16 in place takes 17.7 us with states that come from memory, as a
// model's layers find them (4.0 TB/s), and 13.6 with the same states again and again, which stay in L2.  Short CTAs that load,
// wait and compute hold it below the memory's rate.  One, two and four sequences per thread, from memory, bfloat16:
//   256 x 2048 x 16: 18.8, 17.7, 15.0 us      256 x 2048 x 8: 11.7, 11.2, 11.7      128 x 2048 x 64: 34.5, 28.1, 29.7
// Two is the fastest at 8 and at 64 states, four at 16.
constexpr int kStepSeqs = 2;
template <typename TI, int P, int SEQS, bool WHOLE>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const Params p) {
    constexpr int kOwn = P < SEQS ? SEQS / P : 1;  // sequences that a thread sees to: q, q + P, .. (modulo SEQS)
    // (the channels fit 32 bits, and so do the strides' products with a sequence's number where they stay 64 bits wide)
    const uint32_t at = blockIdx.x * (kThreads / P) + threadIdx.x / P, channels = (uint32_t)p.channels, d = at < channels ? at : channels - 1;
    const uint32_t e = p.groups == 1 ? 0 : d / (uint32_t)p.per;
    const int q = threadIdx.x % P, N = p.N;
    const int64_t b0 = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * SEQS;
    if (b0 >= p.batch) return;  // the last layer of a grid of more rows than its second axis holds
    const int left = p.batch - b0 < SEQS ? (int)(p.batch - b0) : SEQS;  // sequences that exist; the last one stands in for the others
    const int64_t row0 = (b0 * channels + d) * N, row = (int64_t)channels * N;
    const TI *B = static_cast<const TI *>(p.b) + b0 * p.b_b + e * (uint32_t)N, *C = static_cast<const TI *>(p.c) + b0 * p.c_b + e * (uint32_t)N;
    F4 h[SEQS], bv[SEQS], cv[SEQS];
#pragma unroll
    for (int k = 0; k < SEQS; ++k) {
        const int b = k < left ? k : left - 1;
        // (a thread behind the last channel leaves its states alone: their owner may be writing them)
        h[k] = p.state_in && at < channels ? load4_as<WHOLE>(p.state_in + row0 + b * row, kS * q, N) : zero4();
        bv[k] = load4_as<WHOLE>(B + b * p.b_b, kS * q, N);
        cv[k] = load4_as<WHOLE>(C + b * p.c_b, kS * q, N);
    }
    float u[kOwn], step[kOwn], z[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int k = (q + j * P) % SEQS;
        const int64_t b = b0 + (k < left ? k : left - 1);
        u[j] = ld(static_cast<const TI *>(p.u) + b * p.u_b + d);
        step[j] = ld(static_cast<const TI *>(p.dt) + b * p.dt_b + d);
        z[j] = p.z ? ld(static_cast<const TI *>(p.z) + b * p.z_b + d) : 0.f;
    }
    const F4 a2 = rates(load4_as<WHOLE>(p.a + (int64_t)d * N, kS * q, N));
    const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.d ? p.d[d] : 0.f;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        step[j] += bias;
        if (p.softplus) step[j] = softplus(step[j]);
    }
    float y[SEQS];
#pragma unroll
    for (int k = 0; k < SEQS; ++k) {
        const float s = __shfl_sync(0xffffffffu, step[k / P % kOwn], k % P, P), su = __shfl_sync(0xffffffffu, step[k / P % kOwn] * u[k / P % kOwn], k % P, P);
        h[k] = fma(decays(s, a2), h[k], mul(su, bv[k]));
        y[k] = dot(h[k], cv[k]);
#pragma unroll
        for (int o = P / 2; o >= 1; o >>= 1) y[k] += __shfl_xor_sync(0xffffffffu, y[k], o);
        if (p.state_out && at < channels && k < left) {
            float *o = p.state_out + row0 + k * row;
            if (WHOLE) *reinterpret_cast<float4 *>(o + kS * q) = f4(h[k]);
            else store4(o, kS * q, N, h[k]);
        }
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int k = (q + j * P) % SEQS;
        float v = y[0];
#pragma unroll
        for (int x = 1; x < SEQS; ++x) v = x == k ? y[x] : v;
        v = fmaf(skip, u[j], v);
        if (p.z) v *= z[j] * sigmoid(z[j]);
        if (at < channels && k < left && q < SEQS) {
            const int64_t o = (b0 + k) * p.y_b + d;
            if (p.y_dt) st(static_cast<__nv_bfloat16 *>(p.y) + o, v);
            else st(static_cast<float *>(p.y) + o, v);
        }
    }
}

}  // namespace scan
}  // namespace dc
