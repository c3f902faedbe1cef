// selective_scan_bwd.cuh — the backward of the selective scan, tile by tile from the last token back.
//
// With decay_t = exp(step_t a), r_t = dy_t z sigma(z) the gradient of the read-out, and for each state n
//   g_t = c_t r_t + decay_{t+1} g_{t+1}     (g of the final state from the caller)
// the gradients are, per (token, channel):
//   d_step = u sum_n b g + sum_n a w,  w = g decay h_{t-1};   d_u = step sum_n b g + r d;   d_z = dy (sum_n c h + d u) silu'(z)
// summed over the channels of a group: d_b = step u g, d_c = r h;  over tokens: d_a = step w, d_d = r u, d_dt_bias.
//
// The same tiles, segments and registers as the forward (selective_scan.cuh), whose checkpoints hold h at each tile's
// first token: a tile's decays are taken once and serve the states' walk forward and the gradients' walk back; both
// walks run once from zero for the exchange between the segments and once for good.
//
// d_b and d_c sum over channels, which lie across lanes: a token's eight sums of a thread (four states of each) are
// halved lane by lane into one register per token (LaneSum), and a CTA takes up to four blocks of 16 channels one after
// the other through each tile, so that those registers gather 64 channels before they leave for memory: the partial
// sums are then 1/4 of what one block at a time would write and a second kernel read again.
#pragma once

#include "selective_scan.cuh"

namespace dc {
namespace scan {

constexpr int kMaxSub = 4;  // blocks of 16 channels of a CTA

struct BwdParams {
    Params f;
    int32_t nsub;        // blocks of 16 channels per CTA
    int64_t dy_b, dy_t;  // d_y's strides (f.y_dt is its type)
    const void *dy;
    const float *dstate_out;
    void *du, *ddt, *dz;  // [batch, seq, channels]
    float *dstate_in;
    float *bc_part;  // [batch, groups, CTAs of a group, seq, 2, N]
    float *a_part;   // [batch, channels, N]
    float *d_part;   // [batch, 2, channels]: d_d, d_dt_bias
};

template <typename TI, int P>
struct BwdSmem {
    using T = Tile<P>;
    static constexpr int kL = P == 1 ? 16 : 32 / P < 16 ? 32 / P : 16;  // channels whose sums meet in a warp
    static constexpr int kSets = kCh / kL;
    struct RawX {
        TI u[T::kTokens * kCh], dt[T::kTokens * kCh], z[T::kTokens * kCh];
        float dy[T::kTokens * kCh];  // or as many bfloat16
    };
    struct RawBC {
        TI b[T::kTokens * T::kN], c[T::kTokens * T::kN];
    };
    RawX x[2];
    RawBC bc[2];
    float4 step[T::kTokens * kCh];  // (step, step * u, r, -)
    float4 b[T::kTokens * P], c[T::kTokens * P];
    float4 decay[kThreads], end[kThreads], back[kThreads];
    float y[T::kTokens * kCh], gb[T::kTokens * kCh], aw[T::kTokens * kCh];
    float sums[kSets][T::kTokens][2][T::kN];
    // per block of 16 channels, carried from tile to tile
    float4 a2[kMaxSub][kCh * P], g[kMaxSub][kCh * P];
    float4 da[kMaxSub][kThreads], dd[kMaxSub][kThreads];
};

template <typename TI, int P>
__global__ void __launch_bounds__(kThreads, 2) scan_bwd_kernel(const BwdParams bp) {
    using T = Tile<P>;
    using Smem = BwdSmem<TI, P>;
    using ChSum = LaneSum<Smem::kL, P>;
    constexpr int kTok = T::kTokens, kLanes = kCh * P;
    const Params &p = bp.f;
    extern __shared__ __align__(16) unsigned char smem_bytes[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_bytes);
    const int tid = threadIdx.x, seg = tid / kLanes, r = tid % kLanes, ch = r / P, q = r % P;
    const Place at = place_of(blockIdx.x, p, kCh * bp.nsub);
    const int nsub = (at.nch + kCh - 1) / kCh;
    const int64_t len = length_of(p.lengths, at.b, p.seq);
    const int64_t ntiles = (len + kTok - 1) / kTok;
    const int N = p.N;
    const int64_t dy_size = p.y_dt ? 2 : 4;
    const TI *U = static_cast<const TI *>(p.u) + at.b * p.u_b + at.d0, *D = static_cast<const TI *>(p.dt) + at.b * p.dt_b + at.d0;
    const TI *Z = p.z ? static_cast<const TI *>(p.z) + at.b * p.z_b + at.d0 : nullptr;
    const TI *B = static_cast<const TI *>(p.b) + at.b * p.b_b + at.e * N, *C = static_cast<const TI *>(p.c) + at.b * p.c_b + at.e * N;
    const char *DY = static_cast<const char *>(bp.dy) + (at.b * bp.dy_b + at.d0) * dy_size;

    auto load = [&](int64_t it) {
        const int64_t back = it / nsub, t0 = (ntiles - 1 - back) * kTok;
        const int sub = (int)(it - back * nsub), c0 = sub * kCh;
        const int nch = at.nch - c0 < kCh ? at.nch - c0 : kCh;
        const int live = len - t0 < kTok ? (int)(len - t0) : kTok;
        typename Smem::RawX &w = sm.x[it & 1];
        stage_x<kThreads, kCh>(w.u, U + t0 * p.u_t + c0, p.u_t, kTok, live, nch, p.vec_x);
        stage_x<kThreads, kCh>(w.dt, D + t0 * p.dt_t + c0, p.dt_t, kTok, live, nch, p.vec_x);
        if (Z) stage_x<kThreads, kCh>(w.z, Z + t0 * p.z_t + c0, p.z_t, kTok, live, nch, p.vec_x);
        if (p.y_dt)
            stage_x<kThreads, kCh>(reinterpret_cast<__nv_bfloat16 *>(w.dy), reinterpret_cast<const __nv_bfloat16 *>(DY) + t0 * bp.dy_t + c0, bp.dy_t, kTok,
                    live, nch, p.vec_x);
        else
            stage_x<kThreads, kCh>(w.dy, reinterpret_cast<const float *>(DY) + t0 * bp.dy_t + c0, bp.dy_t, kTok, live, nch, p.vec_x);
        if (sub == 0) {
            typename Smem::RawBC &v = sm.bc[back & 1];
            stage_bc<kThreads, T::kN>(v.b, B + t0 * p.b_t, p.b_t, kTok, live, N, p.vec_bc);
            stage_bc<kThreads, T::kN>(v.c, C + t0 * p.c_t, p.c_t, kTok, live, N, p.vec_bc);
        }
        ptx::cp_async_commit();
    };
    auto ld_dy = [&](const typename Smem::RawX &w, int i) {
        return p.y_dt ? ld(reinterpret_cast<const __nv_bfloat16 *>(w.dy) + i) : w.dy[i];
    };

    for (int i = tid; i < kTok * T::kN; i += kThreads)
        if (i % T::kN >= N)
#pragma unroll
            for (int s = 0; s < 2; ++s) st(&sm.bc[s].b[i], 0.f), st(&sm.bc[s].c[i], 0.f);
    for (int sub = 0; sub < nsub; ++sub) {
        sm.da[sub][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
        sm.dd[sub][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (seg == 0) {
            const bool real = sub * kCh + ch < at.nch;
            const int64_t d = at.d0 + (real ? sub * kCh + ch : 0);
            sm.a2[sub][r] = f4(real ? mul(kLog2e, load4(p.a + d * N, kS * q, N)) : zero4());
            sm.g[sub][r] = f4(real && bp.dstate_out ? load4(bp.dstate_out + (at.b * p.channels + d) * N, kS * q, N) : zero4());
        }
    }
    const int oc = 2 * (tid % (kCh / 2));  // the output phase's pair of channels within a block
    float acc[kK][ChSum::kOut];
#pragma unroll
    for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < ChSum::kOut; ++j) acc[k][j] = 0.f;
    const int64_t out0 = at.b * p.seq * p.channels + at.d0;
    auto put = [&](void *o, int64_t t, int c, float v0, float v1) {  // channels c, c + 1 of token t
        TI *w = static_cast<TI *>(o) + out0 + t * p.channels + c;
        if (c + 1 < at.nch && (reinterpret_cast<uintptr_t>(w) % (2 * sizeof(TI))) == 0) {
            if constexpr (sizeof(TI) == 2) *reinterpret_cast<uint32_t *>(w) = vec::pack(v0, v1);
            else *reinterpret_cast<float2 *>(w) = make_float2(v0, v1);
        } else {
            if (c < at.nch) st(w, v0);
            if (c + 1 < at.nch) st(w + 1, v1);
        }
    };

    const int64_t items = ntiles * nsub;
    if (items > 0) load(0);
    for (int64_t it = 0; it < items; ++it) {
        const int64_t back = it / nsub, tile = ntiles - 1 - back, t0 = tile * kTok;
        const int sub = (int)(it - back * nsub), c0 = sub * kCh;
        const int live = len - t0 < kTok ? (int)(len - t0) : kTok;
        const bool real = c0 + ch < at.nch;
        const int64_t d = at.d0 + (real ? c0 + ch : 0);
        ptx::cp_async_wait<0>();
        __syncthreads();  // this item's values have landed, and the last item's shared values are done with
        if (it + 1 < items) load(it + 1);
        const F4 h0 = real ? load4(p.ckpt + ((at.b * p.tiles + tile) * p.channels + d) * N, kS * q, N) : zero4();
        const typename Smem::RawX &w = sm.x[it & 1];
        {
            const int pc = c0 + tid % kCh;
            const float bias = p.dt_bias && pc < at.nch ? p.dt_bias[at.d0 + pc] : 0.f;
            for (int i = tid; i < kTok * kCh; i += kThreads) {
                float v = ld(&w.dt[i]) + bias, g = ld_dy(w, i);
                if (p.softplus) v = softplus(v);
                if (Z) {
                    const float z = ld(&w.z[i]);
                    g *= z * sigmoid(z);
                }
                if (i / kCh >= live) v = 0.f, g = 0.f;
                sm.step[i] = make_float4(v, v * ld(&w.u[i]), g, 0.f);
            }
        }
        if (sub == 0) {
            float *fb = reinterpret_cast<float *>(sm.b), *fc = reinterpret_cast<float *>(sm.c);
            const typename Smem::RawBC &v = sm.bc[back & 1];
            for (int i = tid; i < kTok * T::kN; i += kThreads) fb[i] = ld(&v.b[i]), fc[i] = ld(&v.c[i]);
        }
        __syncthreads();

        const F4 a2 = f4(sm.a2[sub][r]);
        F4 av[kK], hv[kK];  // hv: what is added at each token, then the states
        F4 g_in = f4(sm.g[sub][r]), h_in = h0;
        {
            F4 prod = one4(), h = zero4();
#pragma unroll
            for (int k = 0; k < kK; ++k) {
                const int t = seg * kK + k;
                const float4 sd = sm.step[t * kCh + ch];
                av[k] = ex2(mul(sd.x, a2));
                hv[k] = mul(sd.y, f4(sm.b[t * P + q]));
                if constexpr (T::kSegs > 1) {
                    prod = mul(prod, av[k]);
                    h = fma(av[k], h, hv[k]);
                }
            }
            if constexpr (T::kSegs > 1) {
                F4 g = zero4();
#pragma unroll
                for (int k = kK - 1; k >= 0; --k) {
                    const int t = seg * kK + k;
                    g = mul(av[k], fma(sm.step[t * kCh + ch].z, f4(sm.c[t * P + q]), g));
                }
                sm.decay[tid] = f4(prod);
                sm.end[tid] = f4(h);
                sm.back[tid] = f4(g);
            }
        }
        __syncthreads();
        if constexpr (T::kSegs > 1) {
#pragma unroll
            for (int i = 0; i < T::kSegs - 1; ++i) {
                if (i < seg) h_in = fma(f4(sm.decay[i * kLanes + r]), h_in, f4(sm.end[i * kLanes + r]));
                const int o = T::kSegs - 1 - i;
                if (o > seg) g_in = fma(f4(sm.decay[o * kLanes + r]), g_in, f4(sm.back[o * kLanes + r]));
            }
        }
        float y[kK], gb[kK], aw[kK];
        {
            F4 h = h_in;
#pragma unroll
            for (int k = 0; k < kK; ++k) {
                h = fma(av[k], h, hv[k]);
                hv[k] = h;
                y[k] = dot(h, f4(sm.c[(seg * kK + k) * P + q]));
            }
        }
        F4 da = f4(sm.da[sub][tid]);
        F4 g = g_in;  // decay_{t+1} g_{t+1}
#pragma unroll
        for (int k = kK - 1; k >= 0; --k) {
            const int t = seg * kK + k;
            const float4 sd = sm.step[t * kCh + ch];
            const F4 b = f4(sm.b[t * P + q]), c = f4(sm.c[t * P + q]);
            const F4 dc = mul(sd.z, hv[k]);
            g = fma(sd.z, c, g);
            gb[k] = dot(g, b);
            const F4 db = mul(sd.y, g);
            g = mul(av[k], g);
            const F4 wv = mul(g, k > 0 ? hv[k > 0 ? k - 1 : 0] : h_in);
            aw[k] = dot(wv, a2);
            da = fma(sd.x, wv, da);
            float v[8] = {db.lo.x, db.lo.y, db.hi.x, db.hi.y, dc.lo.x, dc.lo.y, dc.hi.x, dc.hi.y};
            ChSum::run(v, ch % Smem::kL);
#pragma unroll
            for (int j = 0; j < ChSum::kOut; ++j) acc[k][j] += v[j];
        }
        sm.da[sub][tid] = f4(da);
        if (seg == 0) sm.g[sub][r] = f4(g);
        LaneSum<P, 1>::run(gb, q);
        LaneSum<P, 1>::run(aw, q);
        LaneSum<P, 1>::run(y, q);
        const int first = seg * kK + LaneSum<P, 1>::first(q);
#pragma unroll
        for (int k = 0; k < LaneSum<P, 1>::kOut; ++k) {
            const int o = (first + k) * kCh + ch;
            sm.gb[o] = gb[k], sm.aw[o] = aw[k], sm.y[o] = y[k];
        }
        if (sub == nsub - 1) {  // the tile's sums over this CTA's channels
            const int j0 = ChSum::first(ch % Smem::kL), set = ch / Smem::kL;
#pragma unroll
            for (int k = 0; k < kK; ++k)
#pragma unroll
                for (int j = 0; j < ChSum::kOut; ++j) {
                    sm.sums[set][seg * kK + k][(j0 + j) / kS][kS * q + (j0 + j) % kS] = acc[k][j];
                    acc[k][j] = 0.f;
                }
        }
        __syncthreads();
        {
            const int oa = c0 + oc;
            const bool in0 = oa < at.nch, in1 = oa + 1 < at.nch;
            const float dv0 = p.d && in0 ? p.d[at.d0 + oa] : 0.f, dv1 = p.d && in1 ? p.d[at.d0 + oa + 1] : 0.f;
            const float bi0 = p.dt_bias && in0 ? p.dt_bias[at.d0 + oa] : 0.f, bi1 = p.dt_bias && in1 ? p.dt_bias[at.d0 + oa + 1] : 0.f;
            float4 dd = sm.dd[sub][tid];
            for (int i = tid; i < kTok * kCh / 2; i += kThreads) {
                const int t = i / (kCh / 2);
                if (t >= live) continue;
                const int o = t * kCh + oc;
                float du[2], ds[2], dz[2], sum_d[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float4 sd = sm.step[o + j];
                    const float u = ld(&w.u[o + j]), dv = j ? dv1 : dv0;
                    const float gbv = sm.gb[o + j];
                    du[j] = fmaf(gbv, sd.x, sd.z * dv);
                    ds[j] = fmaf(gbv, u, kLn2 * sm.aw[o + j]);
                    if (p.softplus) ds[j] *= sigmoid(ld(&w.dt[o + j]) + (j ? bi1 : bi0));
                    sum_d[j] = sd.z * u;
                    if (Z) {
                        const float z = ld(&w.z[o + j]), sg = sigmoid(z);
                        dz[j] = ld_dy(w, o + j) * fmaf(dv, u, sm.y[o + j]) * sg * fmaf(z, 1.f - sg, 1.f);
                    }
                }
                put(bp.du, t0 + t, oa, du[0], du[1]);
                put(bp.ddt, t0 + t, oa, ds[0], ds[1]);
                if (Z) put(bp.dz, t0 + t, oa, dz[0], dz[1]);
                dd.x += sum_d[0], dd.y += sum_d[1], dd.z += ds[0], dd.w += ds[1];
            }
            sm.dd[sub][tid] = dd;
        }
        if (sub == nsub - 1) {
            const int64_t blocks = (p.per + kCh * bp.nsub - 1) / (kCh * bp.nsub);
            const int64_t blk = (at.d0 - at.e * p.per) / (kCh * bp.nsub);
            float *part = bp.bc_part + (((at.b * p.groups + at.e) * blocks + blk) * p.seq + t0) * 2 * N;
            for (int i = tid; i < live * 2 * T::kN; i += kThreads) {
                const int n = i % T::kN, j = i / T::kN;  // j: (token, which)
                if (n < N) {
                    float v = 0.f;
#pragma unroll
                    for (int q2 = 0; q2 < Smem::kSets; ++q2) v += sm.sums[q2][j >> 1][j & 1][n];
                    part[(int64_t)j * N + n] = v;
                }
            }
        }
    }
    __syncthreads();
    for (int sub = 0; sub < nsub; ++sub) {
        const int c0 = sub * kCh;
        if (seg == 0 && c0 + ch < at.nch) {
            const int64_t row = (at.b * p.channels + at.d0 + c0 + ch) * N;
            F4 v = f4(sm.da[sub][r]);
            for (int i = 1; i < T::kSegs; ++i) {
                const F4 o = f4(sm.da[sub][i * kLanes + r]);
                v = fma(1.f, o, v);
            }
            store4(bp.a_part + row, kS * q, N, v);
            if (bp.dstate_in) store4(bp.dstate_in + row, kS * q, N, f4(sm.g[sub][r]));
        }
        if (tid < kCh && c0 + tid < at.nch) {
            float sd = 0.f, sb = 0.f;
            for (int i = tid / 2; i < kThreads; i += kCh / 2) {
                const float4 v = sm.dd[sub][i];
                sd += tid & 1 ? v.y : v.x;
                sb += tid & 1 ? v.w : v.z;
            }
            float *o = bp.d_part + at.b * 2 * p.channels + at.d0 + c0 + tid;
            o[0] = sd;
            o[p.channels] = sb;
        }
        for (int64_t t = len + tid / (kCh / 2); t < p.seq; t += kThreads / (kCh / 2)) {
            put(bp.du, t, c0 + oc, 0.f, 0.f);
            put(bp.ddt, t, c0 + oc, 0.f, 0.f);
            if (bp.dz) put(bp.dz, t, c0 + oc, 0.f, 0.f);
        }
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
        const float *src = part + (be * blocks * seq + t) * row + in_row;
#pragma unroll 8
        for (int64_t k = 0; k < blocks; ++k) v += src[k * seq * row];
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
        float v = 0.f;
        for (int64_t b = 0; b < batch; ++b) v += a_part[b * na + i];
        da[i] = v;
    } else if (i < na + 2 * channels) {
        const int64_t j = i - na;
        float v = 0.f;
        for (int64_t b = 0; b < batch; ++b) v += d_part[b * 2 * channels + j];
        if (j < channels) {
            if (dd) dd[j] = v;
        } else if (dbias) {
            dbias[j - channels] = v;
        }
    }
}

}  // namespace scan
}  // namespace dc
