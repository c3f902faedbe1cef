// selective_scan_bwd.cuh — the backward of the selective scan, tile by tile from the last token back.
//
// With decay_t = exp(step_t a), r_t = dy_t z sigma(z) the gradient of the read-out, and for each state n
//   g_t = c_t r_t + decay_{t+1} g_{t+1}     (g of the final state from the caller)
// the gradients are, per (token, channel):
//   d_step = u sum_n b g + sum_n a w,  w = g decay h_{t-1};   d_u = step sum_n b g + r d;   d_z = dy (sum_n c h + d u) silu'(z)
// summed over the channels of a group: d_b = step u g, d_c = r h;  over tokens: d_a = step w, d_d = r u, d_dt_bias.
//
// A thread of the recurrence has four states of two neighbouring channels, as in the forward's walk.  From the last four
// tokens of a tile of 16 to its first, it takes their decays and states once more, into registers, and walks the gradients
// back through them.  The states before each four tokens come from a walk forward from the forward's checkpoint, which the
// CTA's other threads make one tile ahead; these also stage the tiles, take the steps and write the gradients of the last
// tile, so that the walk back, the longest chain, waits for nothing: one barrier per tile.  This takes 1.75 exponentials
// per token and state; the other way, segments of threads that run their tokens from zero and exchange, takes one but twice
// the shared memory traffic.  4 x 2048 x 2048 x 16 bfloat16 with the forward: 620 us, of which this kernel is about 440, with
// the shared memory at 62 % of its peak and the issue slots at 47 %; 690 us the other way.
//
// With few channels the time axis is cut into pieces, as in the forward: a first launch walks back through each piece but
// the first from zero, for the gradient that leaves it and its sum of steps, and the second starts each piece from what the
// pieces after it give.
//
// d_b and d_c sum over channels, which lie across lanes (a thread's two channels add up on the way): every four tokens a
// warp turns its sums over in shared memory, so that each lane adds the eight pairs of channels of one token and four
// states; the warps of a CTA meet in a line per token, and a second kernel adds the CTAs' lines in order.
#pragma once

#include "selective_scan.cuh"

namespace dc {
namespace scan {

struct BwdParams {
    Params f;
    int64_t dy_b, dy_t;  // d_y's strides (f.y_dt is its type)
    const void *dy;
    const float *dstate_out;
    void *du, *ddt, *dz;  // [batch, seq, channels]
    float *dstate_in;
    float *bc_part;  // [batch, groups, CTAs of a group, seq, 2, N]
    float *a_part;   // [batch, pieces, channels, N]
    float *d_part;   // [batch, pieces, 2, channels]: d_d, d_dt_bias
    // with pieces (f.pieces, f.piece; the first has none): the gradients that leave them from zero, their sums of steps
    float *piece_out;   // [batch, pieces - 1, channels, N]
    float *piece_step;  // [batch, pieces - 1, channels]
};

constexpr int bwd_channels(int lanes) { return lanes <= 2 ? 64 / lanes : lanes == 16 ? 16 : 32; }  // of a CTA
constexpr int bwd_ctas(int lanes) { return lanes == 2 || lanes == 4 ? 2 : 1; }  // of an SM, by their registers and shared memory

template <int P>
struct BwdShape {
    static constexpr int kCh = bwd_channels(P), kBlk = walk_channels(P);  // channels of a CTA, and of the threads of one block
    static constexpr int kPairs = kBlk / 2, kSegT = kPairs * P, kBlocks = kCh / kBlk, kMain = kSegT * kBlocks;
    static constexpr int kHelp = kTile * kCh / 4, kNT = kMain + kHelp, kN = kS * P, kT = 4;
    // a token's sums over the states: a share per state group, or per four of them (added up by shuffles) where there are
    // so many that the shares would not fit
    static constexpr int kShares = P >= 8 ? P / 4 : P;
    static_assert(kSegT % 32 == 0, "whole warps in a block");
};

template <typename TI, int P>
struct BwdSmem {
    using S = BwdShape<P>;
    struct Raw {  // d_y in the space of float32, whatever its type
        TI u[kTile * S::kCh], dt[kTile * S::kCh], z[kTile * S::kCh], b[kTile * S::kN], c[kTile * S::kN];
        float dy[kTile * S::kCh];
    };
    struct Shares {  // [token][share][channel]
        float y[kTile * S::kCh * S::kShares], gb[kTile * S::kCh * S::kShares], aw[kTile * S::kCh * S::kShares];
        float sums[S::kBlocks][kTile][2][S::kN];  // d_b and d_c of a tile, by block
    };
    // all twofold: the walk back is at one tile while the next is prepared or the last is written
    Raw raw[2];
    float2 step[2][kTile * S::kCh];  // (step, step * u)
    float r[2][kTile * S::kCh];
    float4 b[2][kTile * P], c[2][kTile * P];
    float4 mid[2][kTile / S::kT][2][S::kMain];  // the states before each four tokens
    Shares share[2];
    float4 turn[S::kMain / 32][S::kT * 2 * 32];  // a warp's sums of four tokens: [token][d_b, d_c][lane]
    float bias[S::kCh], skip[S::kCh];
};

// A helper's share of the 16-byte copies of a tile, where the rows start on 16-byte boundaries and d_y has the inputs' type:
// the sources move back by one tile a call (the forward's Stager, the other way).
template <typename TI, int P>
struct BwdStager {
    using S = BwdShape<P>;
    using Raw = typename BwdSmem<TI, P>::Raw;
    static constexpr int kEs = sizeof(TI), kEl = 16 / kEs, kXRow = S::kCh / kEl, kBRow = S::kN >= kEl ? S::kN / kEl : 1;
    static constexpr int kX = kTile * kXRow, kB = kTile * kBRow, kAll = 4 * kX + 2 * kB, kEach = (kAll + S::kHelp - 1) / S::kHelp;
    const char *src[kEach];
    int64_t step[kEach];  // bytes a token
    int dst[kEach], row[kEach], bytes[kEach];
    bool on;

    __device__ __forceinline__ BwdStager(const BwdParams &bp, const Place &at, int64_t t0, int tid) {
        const Params &p = bp.f;
        const struct {
            const void *at;
            int64_t batch, token, first;
            int base;  // in copies
        } in[6] = {{p.u, p.u_b, p.u_t, at.d0, 0},          {p.dt, p.dt_b, p.dt_t, at.d0, kX},        {p.z, p.z_b, p.z_t, at.d0, 2 * kX},
                   {p.b, p.b_b, p.b_t, at.e * p.N, 3 * kX}, {p.c, p.c_b, p.c_t, at.e * p.N, 3 * kX + kB}, {bp.dy, bp.dy_b, bp.dy_t, at.d0, 3 * kX + 2 * kB}};
        on = p.vec_x == kVectors && p.vec_bc == kVectors && S::kN % kEl == 0 && p.z && (p.y_dt ? 2 : 4) == kEs;
#pragma unroll
        for (int k = 0; k < 6; ++k) on = on && aligned16(static_cast<const TI *>(in[k].at) + at.b * in[k].batch + in[k].first);
        if (!on) return;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = tid + j * S::kHelp;
            row[j] = kTile;  // a row that no tile has
            bytes[j] = dst[j] = 0, step[j] = 0, src[j] = nullptr;
#pragma unroll
            for (int k = 0; k < 6; ++k) {
                const int per = k == 3 || k == 4 ? kBRow : kXRow, width = k == 3 || k == 4 ? p.N : at.nch, q = (c - in[k].base) % per;
                if (c >= in[k].base && c < in[k].base + kTile * per) {
                    const int left = (width - q * kEl) * kEs;
                    row[j] = (c - in[k].base) / per;
                    bytes[j] = left < 0 ? 0 : left > 16 ? 16 : left;
                    dst[j] = c * 16;
                    step[j] = in[k].token * kEs;
                    src[j] = reinterpret_cast<const char *>(static_cast<const TI *>(in[k].at) + at.b * in[k].batch + in[k].first + t0 * in[k].token +
                                                            (bytes[j] ? q * kEl : 0));
                }
            }
        }
    }
    __device__ __forceinline__ void copy(Raw &raw, int live) {  // src: the tile's first token
        const uint32_t to = ptx::smem_u32(&raw);
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const bool in = row[j] < live;
            if (row[j] < kTile) ptx::cp_async16(to + dst[j], src[j] + (in ? step[j] * row[j] : 0), in ? bytes[j] : 0);
            src[j] -= step[j] * kTile;
        }
    }
};

// FULL: the whole backward; else only the gradient that leaves the piece, and its sum of steps.
template <typename TI, int P, bool FULL>
__global__ void __launch_bounds__(BwdShape<P>::kNT, bwd_ctas(P)) scan_bwd_kernel(const BwdParams bp) {
    using S = BwdShape<P>;
    constexpr int CH = S::kCh, kT = S::kT;
    const Params &p = bp.f;
    extern __shared__ __align__(16) unsigned char smem_bytes[];
    BwdSmem<TI, P> &sm = *reinterpret_cast<BwdSmem<TI, P> *>(smem_bytes);
    const int64_t pieces = FULL ? p.pieces : p.pieces - 1;
    const int64_t piece = (pieces > 1 ? blockIdx.x % pieces : 0) + (FULL ? 0 : 1);
    const Place at = place_of(pieces > 1 ? blockIdx.x / pieces : blockIdx.x, p, CH);
    const int N = p.N;
    const int64_t first = p.pieces > 1 ? piece * p.piece : 0, last = p.pieces > 1 && first + p.piece < p.seq ? first + p.piece : p.seq;
    const int64_t all = length_of(p.lengths, at.b, p.seq), len = all < last ? all : last;  // this CTA's tokens: first .. len
    const int n = len > first ? (int)((len - first + kTile - 1) / kTile) : 0;              // tiles; number i from the back
    const int64_t tile_end = first / kTile + n;

    if (threadIdx.x >= S::kMain) {
        // ---------------------------------------------------------------- staging, steps, outputs
        const int tid = threadIdx.x - S::kMain, oc = 4 * (tid % (CH / 4)), t = tid / (CH / 4);  // one quad of one token
        const TI *U = static_cast<const TI *>(p.u) + at.b * p.u_b + at.d0, *D = static_cast<const TI *>(p.dt) + at.b * p.dt_b + at.d0;
        const TI *Z = p.z ? static_cast<const TI *>(p.z) + at.b * p.z_b + at.d0 : nullptr;
        const TI *B = static_cast<const TI *>(p.b) + at.b * p.b_b + at.e * N, *C = static_cast<const TI *>(p.c) + at.b * p.c_b + at.e * N;
        const int64_t dy0 = at.b * bp.dy_b + at.d0;
        const int64_t blocks = (p.per + CH - 1) / CH, blk = (at.d0 - at.e * p.per) / CH;
        float *part = bp.bc_part + ((at.b * p.groups + at.e) * blocks + blk) * p.seq * 2 * N;
        BwdStager<TI, P> stager(bp, at, (n > 0 ? tile_end - 1 : 0) * kTile, tid);
        auto load = [&](int i) {
            if (i < n) {
                const int64_t t0 = (tile_end - 1 - i) * kTile;
                const int live = len - t0 < kTile ? (int)(len - t0) : kTile;
                auto &w = sm.raw[i & 1];
                if (stager.on) {
                    stager.copy(w, live);
                } else {
                    stage<S::kHelp, CH, kTile>(w.dt, D + t0 * p.dt_t, p.dt_t, live, at.nch, p.vec_x, tid);
                    stage<S::kHelp, CH, kTile>(w.u, U + t0 * p.u_t, p.u_t, live, at.nch, p.vec_x, tid);
                    if (Z) stage<S::kHelp, CH, kTile>(w.z, Z + t0 * p.z_t, p.z_t, live, at.nch, p.vec_x, tid);
                    if (p.y_dt)
                        stage<S::kHelp, CH, kTile>(reinterpret_cast<__nv_bfloat16 *>(w.dy), static_cast<const __nv_bfloat16 *>(bp.dy) + dy0 + t0 * bp.dy_t,
                                            bp.dy_t, live, at.nch, p.vec_x, tid);
                    else
                        stage<S::kHelp, CH, kTile>(w.dy, static_cast<const float *>(bp.dy) + dy0 + t0 * bp.dy_t, bp.dy_t, live, at.nch, p.vec_x, tid);
                    stage<S::kHelp, S::kN, kTile>(w.b, B + t0 * p.b_t, p.b_t, live, N, p.vec_bc, tid);
                    stage<S::kHelp, S::kN, kTile>(w.c, C + t0 * p.c_t, p.c_t, live, N, p.vec_bc, tid);
                }
            }
            ptx::cp_async_commit();
        };
        // what this thread's four (token, channel) pairs of a tile need again when its sums come back
        struct Kept {
            float u[4], step[4], r[4], dz[4], slope[4];  // dz: d_z per read-out; slope: of softplus
        };
        Kept cur{}, nxt{};
        auto prepare = [&](int i, Kept &k) {
            const bool on = (tile_end - 1 - i) * kTile + t < len;
            const auto &w = sm.raw[i & 1];
            float v[4], z[4], gy[4];
            vec::load<true>(w.u + t * CH + oc, k.u);
            vec::load<true>(w.dt + t * CH + oc, v);
            vec::load_as<true>(p.y_dt, w.dy, t * CH + oc, gy);
            if (Z) vec::load<true>(w.z + t * CH + oc, z);
            float bias[4];
            vec::load<true>(sm.bias + oc, bias);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] += bias[j];
                k.slope[j] = p.softplus ? sigmoid(v[j]) : 1.f;
                k.r[j] = gy[j], k.dz[j] = 0.f;
                if (Z) {
                    const float s = sigmoid(z[j]);
                    k.r[j] = gy[j] * (z[j] * s);
                    k.dz[j] = gy[j] * s * fmaf(z[j], 1.f - s, 1.f);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                float2 f = make_float2(v[j], v[j + 1]);
                if (p.softplus) f = softplus2(f);
                k.step[j] = on ? f.x : 0.f, k.step[j + 1] = on ? f.y : 0.f;  // past the end: decay 1, nothing added
            }
            float4 *o = reinterpret_cast<float4 *>(sm.step[i & 1] + t * CH + oc);
            o[0] = make_float4(k.step[0], k.step[0] * k.u[0], k.step[1], k.step[1] * k.u[1]);
            o[1] = make_float4(k.step[2], k.step[2] * k.u[2], k.step[3], k.step[3] * k.u[3]);
            vec::store<true>(sm.r[i & 1] + t * CH + oc, k.r);
            widen<S::kHelp>(sm.b[i & 1], w.b, kTile * S::kN, tid);
            widen<S::kHelp>(sm.c[i & 1], w.c, kTile * S::kN, tid);
        };
        const int64_t out0 = at.b * p.seq * p.channels + at.d0 + oc;
        const int nput = at.nch - oc;  // channels of the quad that exist (<= 0: none)
        const bool quad = nput >= 4 && out0 % 4 == 0 && p.channels % 4 == 0 && aligned16(bp.du) && aligned16(bp.ddt) && aligned16(bp.dz);
        auto put = [&](void *o, int64_t token, const float (&v)[4]) {
            TI *w = static_cast<TI *>(o) + out0 + token * p.channels;
            if (quad) vec::store<true>(w, v);
            else vec::store<false>(w, v, nput);
        };
        float sd[4] = {}, sb[4] = {};  // sums over this thread's tokens: d_d, d_dt_bias
        auto finish = [&](int i, const Kept &k) {  // the gradients of tile i, from the recurrence's shares
            const auto &sh = sm.share[i & 1];
            const int64_t t0 = (tile_end - 1 - i) * kTile, token = t0 + t;
            float y[4] = {}, gb[4] = {}, aw[4] = {};
#pragma unroll
            for (int j = 0; j < S::kShares; ++j) {  // from another share on in each token, as in the forward
                const int o = (t * S::kShares + ((j + t) & (S::kShares - 1))) * CH + oc;
                const float4 f = *reinterpret_cast<const float4 *>(sh.gb + o), g = *reinterpret_cast<const float4 *>(sh.aw + o);
                gb[0] += f.x, gb[1] += f.y, gb[2] += f.z, gb[3] += f.w;
                aw[0] += g.x, aw[1] += g.y, aw[2] += g.z, aw[3] += g.w;
                if (Z) {
                    const float4 h = *reinterpret_cast<const float4 *>(sh.y + o);
                    y[0] += h.x, y[1] += h.y, y[2] += h.z, y[3] += h.w;
                }
            }
            if (token < len) {
                float skip[4], du[4], ds[4], dz[4];
                vec::load<true>(sm.skip + oc, skip);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // where softplus has no slope left, rates at the end of the range may have taken their terms past it
                    if (k.slope[j] == 0.f && !(fabsf(aw[j]) <= FLT_MAX)) aw[j] = 0.f;
                    du[j] = fmaf(gb[j], k.step[j], k.r[j] * skip[j]);
                    ds[j] = fmaf(gb[j], k.u[j], kLn2 * aw[j]) * k.slope[j];
                    dz[j] = fmaf(skip[j], k.u[j], y[j]) * k.dz[j];
                    sd[j] = fmaf(k.r[j], k.u[j], sd[j]);
                    sb[j] += ds[j];
                }
                put(bp.du, token, du);
                put(bp.ddt, token, ds);
                if (Z) put(bp.dz, token, dz);
            }
            // the tile's lines of d_b and d_c: the blocks' sums in order
            const int live = len - t0 < kTile ? (int)(len - t0) : kTile;
            for (int j = tid; j < live * 2 * S::kN; j += S::kHelp) {
                const int state = j % S::kN, row = j / S::kN;  // row: (token, which)
                if (state < N) {
                    float v = 0.f;
#pragma unroll
                    for (int q = 0; q < S::kBlocks; ++q) v += (&sh.sums[q][0][0][0])[j];
                    part[(t0 * 2 + row) * N + state] = v;
                }
            }
        };
        // the states before each four tokens of a tile: thread v walks one channel (the j-th of a pair) of a thread of the
        // recurrence; this thread is v = tid, tid + kHelp, ..
        constexpr int kWalks = (2 * S::kMain + S::kHelp - 1) / S::kHelp;
        F4 wa[kWalks], wh[kWalks];
        int wch[kWalks], wq[kWalks];
#pragma unroll
        for (int x = 0; x < kWalks; ++x) {
            const int v = tid + x * S::kHelp, of = v % S::kMain, r = of % S::kSegT;
            wch[x] = v < 2 * S::kMain ? of / S::kSegT * S::kBlk + 2 * (r % S::kPairs) + v / S::kMain : CH, wq[x] = r / S::kPairs;
            wa[x] = wch[x] < at.nch ? rates(load4(p.a + (at.d0 + wch[x]) * N, kS * wq[x], N)) : zero4();
        }
        auto fetch = [&](int i) {  // the checkpoints of tile i
#pragma unroll
            for (int x = 0; x < kWalks; ++x)
                wh[x] = wch[x] < at.nch ? load4(p.ckpt + ((at.b * p.tiles + tile_end - 1 - i) * p.channels + at.d0 + wch[x]) * N, kS * wq[x], N) : zero4();
        };
        auto walk = [&](int i) {
#pragma unroll
            for (int x = 0; x < kWalks; ++x) {
                const int v = tid + x * S::kHelp;
                if (v >= 2 * S::kMain) continue;
                const float2 *step = sm.step[i & 1] + wch[x];
                const float4 *bs = sm.b[i & 1] + wq[x];
                float4 *mid = &sm.mid[i & 1][0][v / S::kMain][v % S::kMain];
                F4 h = wh[x];
                *mid = f4(h);
#pragma unroll 1
                for (int m = 1; m < kTile / kT; ++m) {
                    F4 av[kT], bv[kT];
#pragma unroll
                    for (int k = 0; k < kT; ++k, step += CH, bs += P) {
                        const float2 s = *step;
                        av[k] = decays(s.x, wa[x]);
                        bv[k] = mul(s.y, f4(*bs));
                    }
#pragma unroll
                    for (int k = 0; k < kT; ++k) h = fma(av[k], h, bv[k]);
                    mid[m * 2 * S::kMain] = f4(h);
                }
            }
        };
        for (int i = tid; i < CH; i += S::kHelp) {
            sm.bias[i] = p.dt_bias && i < at.nch ? p.dt_bias[at.d0 + i] : 0.f;
            sm.skip[i] = p.d && i < at.nch ? p.d[at.d0 + i] : 0.f;
        }
        load(0);
        auto ahead = [&](int i) {  // make tile i ready
            if (FULL) fetch(i);
            ptx::cp_async_wait<0>();
            ptx::named_sync(1, S::kHelp);  // every helper's copies of it have landed
            load(i + 1);                   // into the other stage, which everyone has read
            prepare(i, nxt);
            ptx::named_sync(1, S::kHelp);
            if (FULL) walk(i);
        };
        if (n > 0) ahead(0);
        __syncthreads();  // the first tile is ready
        Kept old{};
        for (int i = 0; i < n; ++i) {
            old = cur, cur = nxt;
            if (i + 1 < n) ahead(i + 1);
            if (FULL && i > 0) finish(i - 1, old);
            __syncthreads();  // tile i is done, i + 1 is ready
        }
        if (!FULL) return;
        if (n > 0) finish(n - 1, cur);
        // the sums over tokens: sixteen threads' in order, through the shares' memory
        ptx::named_sync(1, S::kHelp);
        vec::store<true>(sm.share[0].y + t * CH + oc, sd);
        vec::store<true>(sm.share[0].gb + t * CH + oc, sb);
        ptx::named_sync(1, S::kHelp);
        if (tid < at.nch) {
            float d = 0.f, b = 0.f;
            for (int k = 0; k < kTile; ++k) d += sm.share[0].y[k * CH + tid], b += sm.share[0].gb[k * CH + tid];
            float *o = bp.d_part + (at.b * p.pieces + piece) * 2 * p.channels + at.d0 + tid;
            o[0] = d;
            o[p.channels] = b;
        }
        const float none[4] = {0.f, 0.f, 0.f, 0.f};
        for (int64_t token = (len > first ? len : first) + t; token < last; token += kTile) {
            put(bp.du, token, none);
            put(bp.ddt, token, none);
            if (bp.dz) put(bp.dz, token, none);
        }
        return;
    }

    // -------------------------------------------------------------------- the recurrences
    const int tid = threadIdx.x, block = tid / S::kSegT, r = tid % S::kSegT, pair = r % S::kPairs, q = r / S::kPairs;
    const int ch = block * S::kBlk + 2 * pair;
    bool real[2];
    F4 a2[2], g[2], da[2];  // g: decay_{t+1} g_{t+1}
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        real[j] = ch + j < at.nch;
        const int64_t d = at.d0 + ch + j;
        a2[j] = real[j] ? rates(load4(p.a + d * N, kS * q, N)) : zero4();
        g[j] = FULL && real[j] && bp.dstate_out ? load4(bp.dstate_out + (at.b * p.channels + d) * N, kS * q, N) : zero4();
        da[j] = zero4();
        if (FULL && real[j])
#pragma unroll 4
            for (int64_t k = p.pieces - 1; k > piece; --k) {  // what the pieces after this one make of it
                const int64_t row = (at.b * (p.pieces - 1) + k - 1) * p.channels + d;
                g[j] = fma(ex2(mul(bp.piece_step[row], a2[j])), g[j], load4(bp.piece_out + row * N, kS * q, N));
            }
    }
    if constexpr (!FULL) {
        float steps[2] = {0.f, 0.f};
        __syncthreads();  // the first tile is ready
        for (int i = 0; i < n; ++i) {
            const float2 *step = sm.step[i & 1] + ch;
            const float *rr = sm.r[i & 1] + ch;
            const float4 *cs = sm.c[i & 1] + q;
#pragma unroll 4
            for (int t = kTile - 1; t >= 0; --t) {
                const float4 sd = *reinterpret_cast<const float4 *>(step + t * CH);
                const float2 rv = *reinterpret_cast<const float2 *>(rr + t * CH);
                const F4 c = f4(cs[t * P]);
                g[0] = mul(decays(sd.x, a2[0]), fma(rv.x, c, g[0]));
                g[1] = mul(decays(sd.z, a2[1]), fma(rv.y, c, g[1]));
                steps[0] += sd.x, steps[1] += sd.z;
            }
            __syncthreads();  // tile i is done, i + 1 is ready
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (!real[j]) continue;
            const int64_t row = (at.b * (p.pieces - 1) + piece - 1) * p.channels + at.d0 + ch + j;
            store4(bp.piece_out + row * N, kS * q, N, g[j]);
            if (q == 0) bp.piece_step[row] = steps[j];
        }
        return;
    }
    // this lane's part in turning sums over: token, which of d_b (0) and d_c (1), state group of the warp, first pair
    constexpr int kGroups = 32 / S::kPairs, kPer = S::kPairs / 8;  // state groups of a warp, lanes that share a sum
    const int lane = tid & 31, out = lane / kPer, out_t = out / (2 * kGroups), out_w = out / kGroups % 2, out_q = out % kGroups;
    const int out_state = kS * (q / kGroups * kGroups + out_q);
    float4 *turn = sm.turn[tid / 32];
    auto leave = [&](float *o, int t, float v0, float v1) {  // both channels' share of token t
        if constexpr (S::kShares == P) {
            *reinterpret_cast<float2 *>(o + (t * P + q) * CH + ch) = make_float2(v0, v1);
        } else {  // the warp's four state groups, 8 lanes apart
#pragma unroll
            for (int x = 8; x <= 16; x *= 2) v0 += __shfl_xor_sync(0xffffffffu, v0, x), v1 += __shfl_xor_sync(0xffffffffu, v1, x);
            if (q % 4 == 0) *reinterpret_cast<float2 *>(o + (t * S::kShares + q / 4) * CH + ch) = make_float2(v0, v1);
        }
    };
    __syncthreads();  // the first tile is ready
    for (int i = 0; i < n; ++i) {
        const float2 *step = sm.step[i & 1] + ch;
        const float *rr = sm.r[i & 1] + ch;
        const float4 *bs = sm.b[i & 1] + q, *cs = sm.c[i & 1] + q;
        auto &sh = sm.share[i & 1];
#pragma unroll 1
        for (int m = kTile / kT - 1; m >= 0; --m) {
            F4 av[kT][2], hv[kT][2];
            const F4 h_in[2] = {f4(sm.mid[i & 1][m][0][tid]), f4(sm.mid[i & 1][m][1][tid])};
#pragma unroll
            for (int k = 0; k < kT; ++k) {
                const int t = m * kT + k;
                const float4 sd = *reinterpret_cast<const float4 *>(step + t * CH);
                const F4 b = f4(bs[t * P]);
                av[k][0] = decays(sd.x, a2[0]), av[k][1] = decays(sd.z, a2[1]);
                hv[k][0] = fma(av[k][0], k ? hv[k ? k - 1 : 0][0] : h_in[0], mul(sd.y, b));
                hv[k][1] = fma(av[k][1], k ? hv[k ? k - 1 : 0][1] : h_in[1], mul(sd.w, b));
            }
#pragma unroll
            for (int k = kT - 1; k >= 0; --k) {
                const int t = m * kT + k;
                const float4 sd = *reinterpret_cast<const float4 *>(step + t * CH);
                const float2 rv = *reinterpret_cast<const float2 *>(rr + t * CH);
                const F4 b = f4(bs[t * P]), c = f4(cs[t * P]);
                const F4 g0 = fma(rv.x, c, g[0]), g1 = fma(rv.y, c, g[1]);
                turn[(k * 2 + 0) * 32 + lane] = f4(fma(sd.w, g1, mul(sd.y, g0)));
                turn[(k * 2 + 1) * 32 + lane] = f4(fma(rv.y, hv[k][1], mul(rv.x, hv[k][0])));
                leave(sh.y, t, dot(hv[k][0], c), dot(hv[k][1], c));
                leave(sh.gb, t, dot(g0, b), dot(g1, b));
                g[0] = mul(av[k][0], g0), g[1] = mul(av[k][1], g1);
                const F4 w0 = mul(g[0], k ? hv[k ? k - 1 : 0][0] : h_in[0]), w1 = mul(g[1], k ? hv[k ? k - 1 : 0][1] : h_in[1]);
                leave(sh.aw, t, dot(w0, a2[0]), dot(w1, a2[1]));
                da[0] = fma(sd.x, w0, da[0]), da[1] = fma(sd.z, w1, da[1]);
            }
            __syncwarp();
            {
                // eight pairs of channels, from another one on in each lane so that the reads meet in no bank
                const float4 *from = turn + ((out_t * 2 + out_w) * kGroups + out_q) * S::kPairs + lane % kPer * 8;
                F4 v = f4(from[out & 7]);
#pragma unroll
                for (int x = 1; x < 8; ++x) v = fma(1.f, f4(from[(out + x) & 7]), v);
#pragma unroll
                for (int o = kPer / 2; o >= 1; o /= 2) {
                    v.lo.x += __shfl_xor_sync(0xffffffffu, v.lo.x, o), v.lo.y += __shfl_xor_sync(0xffffffffu, v.lo.y, o);
                    v.hi.x += __shfl_xor_sync(0xffffffffu, v.hi.x, o), v.hi.y += __shfl_xor_sync(0xffffffffu, v.hi.y, o);
                }
                if (lane % kPer == 0) *reinterpret_cast<float4 *>(&sh.sums[block][m * kT + out_t][out_w][out_state]) = f4(v);
            }
            __syncwarp();
        }
        __syncthreads();  // tile i is done, i + 1 is ready
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (!real[j]) continue;
        const int64_t d = at.d0 + ch + j;
        store4(bp.a_part + ((at.b * p.pieces + piece) * p.channels + d) * N, kS * q, N, da[j]);
        if (bp.dstate_in && piece == 0) store4(bp.dstate_in + (at.b * p.channels + d) * N, kS * q, N, g[j]);
    }
}

// d_b and d_c [batch, seq, groups, N] from the CTAs' sums, in their order.
template <typename TI>
__global__ void __launch_bounds__(256) scan_bwd_bc_kernel(const float *part, int64_t batch, int64_t seq, int64_t groups, int64_t blocks,
                                                          int N, const int32_t *lengths, TI *db, TI *dc) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = 2 * (int64_t)N;
    if (i >= batch * groups * seq * row) return;
    const int64_t in_row = i % row, t = i / row % seq, be = i / (row * seq), b = be / groups, e = be - b * groups;
    float v = 0.f;
    if (t < length_of(lengths, b, seq)) {
        v = vec::sum_lines(part + (be * blocks * seq + t) * row + in_row, 0, blocks, 1, seq * row);
    }
    const int64_t n = in_row % N;
    TI *o = (in_row >= N ? dc : db) + ((b * seq + t) * groups + e) * N + n;
    st(o, v);
}

// The sums over the batch: d_a [channels, N], d_d and d_dt_bias [channels] (either may be null).
__global__ void __launch_bounds__(256) scan_bwd_batch_kernel(const float *a_part, const float *d_part, int64_t batch, int64_t channels, int N,
                                                             float *da, float *dd, float *dbias) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, na = channels * N;
    if (i < na) {
        da[i] = vec::sum_lines(a_part + i, 0, batch, 1, na);
    } else if (i < na + 2 * channels) {
        const int64_t j = i - na;
        const float v = vec::sum_lines(d_part + j, 0, batch, 1, 2 * channels);
        if (j < channels) {
            if (dd) dd[j] = v;
        } else if (dbias) {
            dbias[j - channels] = v;
        }
    }
}

}  // namespace scan
}  // namespace dc
