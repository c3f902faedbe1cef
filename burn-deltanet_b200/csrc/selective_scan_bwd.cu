// selective_scan_bwd.cu — C entry points of the selective scan's backward (include/deltacore_layers.h).
#include "selective_scan_bwd.cuh"
#include "selective_scan_host.hpp"

namespace {

using namespace dc::host;
namespace sc = dc::scan;

struct Layout {
    int64_t blocks;  // CTAs of a group
    uint64_t bc, a, d, bytes;
};

Layout layout_of(const dc_selective_scan_args *f) {
    Layout l;
    const uint64_t al = 255;
    l.blocks = ceil_div(f->channels / f->groups, sc::bwd_channels(sc::lanes_of(f->state)));
    l.bc = 0;
    l.a = ((uint64_t)f->batch * f->groups * l.blocks * f->seq * 2 * f->state * 4 + al) & ~al;
    l.d = l.a + (((uint64_t)f->batch * f->channels * f->state * 4 + al) & ~al);
    l.bytes = l.d + (uint64_t)f->batch * 2 * f->channels * 4;
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
    const void *f32s[] = {a->d_a, a->d_d, a->d_dt_bias, a->d_state_in, a->d_state_out};
    for (const void *o : f32s)
        if (!aligned(o, 4)) return DC_EINVAL_ARG;
    if (!aligned(a->d_y, dtype_size(f->out_dtype)) || (a->d_state_in && a->d_state_in == a->d_state_out)) return DC_EINVAL_ARG;
    return DC_OK;
}

template <typename TI>
struct Launch {
    const sc::BwdParams &p;
    unsigned ctas;
    cudaStream_t s;
    template <int P>
    int operator()() const {
        constexpr size_t smem = sizeof(sc::BwdSmem<TI, P>);
        static_assert(smem <= 227 * 1024, "shared memory of a CTA");
        const int st = sc::allow_smem(&sc::scan_bwd_kernel<TI, P>, smem);
        if (st != DC_OK) return st;
        sc::scan_bwd_kernel<TI, P><<<ctas, sc::BwdShape<P>::kNT, smem, s>>>(p);
        return launched();
    }
};

template <typename TI>
int run(const dc_selective_scan_bwd_args *a, const sc::BwdParams &p, int64_t blocks, cudaStream_t s) {
    const dc_selective_scan_args *f = &a->fwd;
    if (f->batch > 0) {
        const int64_t ctas = f->batch * f->groups * blocks;
        const int64_t bc = ceil_div(f->batch * f->groups * f->seq * 2 * f->state, 256);
        if (ctas > 0x7fffffff || bc > 0x7fffffff) return DC_EUNSUPPORTED;
        int st = sc::for_lanes(f->state, Launch<TI>{p, (unsigned)ctas, s});
        if (st != DC_OK) return st;
        if (bc > 0) {
            sc::scan_bwd_bc_kernel<TI><<<(unsigned)bc, 256, 0, s>>>(p.bc_part, f->batch, f->seq, f->groups, blocks, (int)f->state, f->lengths,
                                                                    static_cast<TI *>(a->d_b), static_cast<TI *>(a->d_c));
            st = launched();
            if (st != DC_OK) return st;
        }
    }
    const int64_t n = f->channels * (f->state + 2);
    sc::scan_bwd_batch_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(p.a_part, p.d_part, f->batch, f->channels, (int)f->state, a->d_a, a->d_d,
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
    const Layout l = layout_of(&a->fwd);
    if (a->fwd.batch > 0) {
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
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return a->fwd.in_dtype == DC_BF16 ? run<__nv_bfloat16>(a, p, l.blocks, s) : run<float>(a, p, l.blocks, s);
}

}  // extern "C"
