// selective_scan_bwd.cu — C entry points of the selective scan's backward (include/deltacore_layers.h).
#include "selective_scan_bwd.cuh"
#include "selective_scan_host.hpp"

namespace {

using namespace dc::host;
namespace sc = dc::scan;

struct Layout {
    int64_t blocks;  // CTAs of a group, for one piece
    int64_t pieces, piece;
    uint64_t bc, a, d, out, step, bytes;
};

// Pieces of the time axis: as many as the card has room for, 256 tokens each at least (1 x 4096 x 1024 x 16, forward and
// backward: 225 us with nine of them, 773 us in one).
Layout layout_of(const dc_selective_scan_args *f) {
    constexpr int64_t kLeast = 256;
    const int lanes = sc::lanes_of(f->state);
    Layout l;
    l.blocks = ceil_div(f->channels / f->groups, sc::bwd_channels(lanes));
    const int64_t ctas = f->batch * f->groups * l.blocks, room = (int64_t)sm_count() * sc::bwd_ctas(lanes);
    const int64_t want = room / ctas, most = f->seq / kLeast, pieces = want < most ? want : most;
    l.pieces = 1, l.piece = f->seq;
    if (pieces > 1) {
        l.piece = ceil_div(ceil_div(f->seq, pieces), sc::kTile) * sc::kTile;
        l.pieces = ceil_div(f->seq, l.piece);
    }
    uint64_t at = 0;
    auto take = [&](int64_t floats) {
        const uint64_t from = at;
        at += ((uint64_t)floats * 4 + 255) & ~(uint64_t)255;
        return from;
    };
    l.bc = take(f->batch * f->groups * l.blocks * f->seq * 2 * f->state);
    l.a = take(f->batch * l.pieces * f->channels * f->state);
    l.d = take(f->batch * l.pieces * 2 * f->channels);
    l.out = take(f->batch * (l.pieces - 1) * f->channels * f->state);
    l.step = take(f->batch * (l.pieces - 1) * f->channels);
    l.bytes = at;
    return l;
}

int validate(const dc_selective_scan_bwd_args *a) {
    const dc_selective_scan_args *f = &a->fwd;
    if (f->channels == 0) return DC_OK;
    if (!a->d_a) return DC_EINVAL_ARG;
    if (f->batch > 0) {
        const int st = sc::validate_inputs(f, f->seq);
        if (st != DC_OK) return st;
        if (f->seq > 0 && (!a->d_y || !a->d_u || !a->d_dt || !a->d_b || !a->d_c || (f->z && !a->d_z) || !f->checkpoints)) return DC_EINVAL_ARG;
        if ((f->seq > 1 && a->d_y_token_stride < f->channels) || (f->seq > 0 && f->batch > 1 && a->d_y_batch_stride < f->channels)) return DC_EINVAL_SHAPE;
    }
    const size_t is = dtype_size(f->in_dtype);
    const void *outs[] = {a->d_u, a->d_dt, a->d_z, a->d_b, a->d_c};
    const void *ins[] = {f->u, f->dt, f->z, f->b, f->c, a->d_y};
    for (const void *o : outs) {
        if (!aligned(o, is)) return DC_EINVAL_ARG;
        for (const void *i : ins)
            if (o && o == i) return DC_EINVAL_ARG;
    }
    // of these, a CTA that runs later would read what another one wrote
    const int64_t row = f->channels * is, states = f->batch * f->channels * f->state * 4, os = dtype_size(f->out_dtype);
    const Rows dy{a->d_y, f->batch, f->seq, a->d_y_batch_stride * os, a->d_y_token_stride * os, f->channels * os};
    for (const void *o : {a->d_u, a->d_dt, a->d_z}) {
        const Rows out{o, f->batch, f->seq, f->seq * row, row, row};
        if (sc::meets_inputs(f, f->seq, out) || rows_meet(dy, out)) return DC_EINVAL_ARG;
    }
    if (overlap(a->d_state_in, states, a->d_state_out, states)) return DC_EINVAL_ARG;
    const void *f32s[] = {a->d_a, a->d_d, a->d_dt_bias, a->d_state_in, a->d_state_out};
    for (const void *o : f32s)
        if (!aligned(o, 4)) return DC_EINVAL_ARG;
    if (!aligned(a->d_y, os)) return DC_EINVAL_ARG;
    return DC_OK;
}

template <typename TI>
struct Launch {
    const sc::BwdParams &p;
    int64_t ctas;  // of one piece
    cudaStream_t s;
    template <int P, bool FULL>
    int go(int64_t n) const {
        constexpr size_t smem = sizeof(sc::BwdSmem<TI, P>);
        static_assert(smem <= 227 * 1024, "shared memory of a CTA");
        if (n > 0x7fffffff) return DC_EUNSUPPORTED;
        const int st = sc::allow_smem(&sc::scan_bwd_kernel<TI, P, FULL>, smem);
        if (st != DC_OK) return st;
        sc::scan_bwd_kernel<TI, P, FULL><<<(unsigned)n, sc::BwdShape<P>::kNT, smem, s>>>(p);
        return launched();
    }
    template <int P>
    int operator()() const {
        const int st = p.f.pieces > 1 ? go<P, false>(ctas * (p.f.pieces - 1)) : DC_OK;
        return st == DC_OK ? go<P, true>(ctas * p.f.pieces) : st;
    }
};

template <typename TI>
int run(const dc_selective_scan_bwd_args *a, const sc::BwdParams &p, int64_t blocks, cudaStream_t s) {
    const dc_selective_scan_args *f = &a->fwd;
    if (f->batch > 0) {
        const int64_t ctas = f->batch * f->groups * blocks;
        const int64_t bc = ceil_div(f->batch * f->groups * f->seq * 2 * f->state, 256);
        if (bc > 0x7fffffff) return DC_EUNSUPPORTED;
        int st = sc::for_lanes(f->state, Launch<TI>{p, ctas, s});
        if (st != DC_OK) return st;
        if (bc > 0) {
            sc::scan_bwd_bc_kernel<TI><<<(unsigned)bc, 256, 0, s>>>(p.bc_part, f->batch, f->seq, f->groups, blocks, (int)f->state, f->lengths,
                                                                    static_cast<TI *>(a->d_b), static_cast<TI *>(a->d_c));
            st = launched();
            if (st != DC_OK) return st;
        }
    }
    const int64_t n = f->channels * (f->state + 2);
    sc::scan_bwd_batch_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(p.a_part, p.d_part, f->batch * p.f.pieces, f->channels, (int)f->state, a->d_a, a->d_d,
                                                                        a->d_dt_bias);
    return launched();
}

}  // namespace

extern "C" {

uint64_t dc_selective_scan_bwd_workspace_size(const dc_selective_scan_bwd_args *a) {
    if (!a || sc::validate_dims(&a->fwd) != DC_OK || a->fwd.batch == 0 || a->fwd.channels == 0) return 0;
    return layout_of(&a->fwd).bytes;
}

int dc_selective_scan_bwd(const dc_selective_scan_bwd_args *a, dc_stream_t stream) {
    if (!a) return DC_EINVAL_ARG;
    int st = sc::validate_dims(&a->fwd);
    if (st == DC_OK) st = validate(a);
    if (st != DC_OK) return st;
    if (a->fwd.channels == 0) return DC_OK;
    Layout l{};
    l.pieces = 1;
    if (a->fwd.batch > 0) {
        l = layout_of(&a->fwd);
        if (a->workspace_bytes < l.bytes) return DC_EWORKSPACE;
        if (!a->workspace || !aligned(a->workspace, 16)) return DC_EINVAL_ARG;
    }
    st = check_device();
    if (st != DC_OK) return st;
    sc::BwdParams p{};
    p.f = sc::params_of(&a->fwd);
    p.dy_b = a->d_y_batch_stride, p.dy_t = a->d_y_token_stride;
    const int64_t dy_bytes = p.dy_t * (int64_t)dtype_size(a->fwd.out_dtype);
    if (dy_bytes % 16) p.f.vec_x = dy_bytes % 4 ? sc::kScalar : p.f.vec_x < sc::kWords ? p.f.vec_x : sc::kWords;
    p.dy = a->d_y, p.dstate_out = a->d_state_out;
    p.du = a->d_u, p.ddt = a->d_dt, p.dz = a->fwd.z ? a->d_z : nullptr, p.dstate_in = a->d_state_in;
    char *ws = static_cast<char *>(a->workspace);
    p.bc_part = reinterpret_cast<float *>(ws + l.bc), p.a_part = reinterpret_cast<float *>(ws + l.a), p.d_part = reinterpret_cast<float *>(ws + l.d);
    p.piece_out = reinterpret_cast<float *>(ws + l.out), p.piece_step = reinterpret_cast<float *>(ws + l.step);
    p.f.pieces = (int32_t)l.pieces, p.f.piece = l.piece;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return a->fwd.in_dtype == DC_BF16 ? run<__nv_bfloat16>(a, p, l.blocks, s) : run<float>(a, p, l.blocks, s);
}

}  // extern "C"
