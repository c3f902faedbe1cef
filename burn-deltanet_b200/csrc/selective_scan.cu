// selective_scan.cu — C entry points of the selective scan and its decode tick (include/deltacore_layers.h).
#include "selective_scan_host.hpp"

namespace {

using namespace dc::host;
namespace sc = dc::scan;

static_assert(DC_SCAN_MAX_STATE == 16 * sc::kS, "the header's limit is the kernels'");

int validate_output(const dc_selective_scan_args *a, int64_t seq) {
    const int64_t os = dtype_size(a->out_dtype), is = dtype_size(a->in_dtype), c = a->channels;
    if (seq == 0) return DC_OK;
    if (!a->y || !aligned(a->y, os)) return DC_EINVAL_ARG;
    if ((seq > 1 && a->y_token_stride < c) || (a->batch > 1 && a->y_batch_stride < c)) return DC_EINVAL_SHAPE;
    // y over an input would be read by a CTA that runs later; interleaved slices of one buffer start elsewhere
    const void *ins[] = {a->u, a->dt, a->z, a->b, a->c};
    for (const void *q : ins)
        if (q && q == a->y) return DC_EINVAL_ARG;
    (void)is;
    return DC_OK;
}

template <typename TI>
struct Launch {
    const sc::Params &p;
    cudaStream_t s;
    template <int P>
    int operator()() const {
        const int64_t ctas = p.batch * p.groups * p.blocks;
        if (ctas > 0x7fffffff) return DC_EUNSUPPORTED;
        constexpr size_t smem = sizeof(sc::FwdSmem<TI, P>);
        const int st = sc::allow_smem(&sc::scan_kernel<TI, P>, smem);
        if (st != DC_OK) return st;
        sc::scan_kernel<TI, P><<<(unsigned)ctas, sc::kThreads, smem, s>>>(p);
        return launched();
    }
};

template <typename TI>
struct LaunchStep {
    const sc::Params &p;
    cudaStream_t s;
    template <int P>
    int operator()() const {
        const int64_t ctas = ceil_div(p.batch * p.channels, sc::kThreads / P);
        if (ctas > 0x7fffffff) return DC_EUNSUPPORTED;
        sc::scan_step_kernel<TI, P><<<(unsigned)ctas, sc::kThreads, 0, s>>>(p);
        return launched();
    }
};

}  // namespace

extern "C" {

uint64_t dc_selective_scan_checkpoint_size(const dc_selective_scan_args *a) {
    if (sc::validate_dims(a) != DC_OK) return 0;
    return (uint64_t)a->batch * (uint64_t)ceil_div(a->seq, sc::tile_tokens(a->state)) * (uint64_t)a->channels * (uint64_t)a->state * 4;
}

uint64_t dc_selective_scan_workspace_size(const dc_selective_scan_args *) { return 0; }

int dc_selective_scan(const dc_selective_scan_args *a, dc_stream_t stream) {
    int st = sc::validate_dims(a);
    if (st != DC_OK) return st;
    if (a->batch == 0 || a->channels == 0) return DC_OK;
    st = sc::validate_inputs(a, a->seq);
    if (st == DC_OK) st = validate_output(a, a->seq);
    if (st == DC_OK) st = check_device();
    if (st != DC_OK) return st;
    sc::Params p = sc::params_of(a);
    p.blocks = (int32_t)ceil_div(p.per, sc::kCh);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a->in_dtype == DC_BF16) return sc::for_lanes(a->state, Launch<__nv_bfloat16>{p, s});
    return sc::for_lanes(a->state, Launch<float>{p, s});
}

int dc_selective_scan_step(const dc_selective_scan_args *a, dc_stream_t stream) {
    int st = sc::validate_dims(a);
    if (st != DC_OK) return st;
    if (a->seq != 1) return DC_EINVAL_SHAPE;
    if (a->batch == 0 || a->channels == 0) return DC_OK;
    st = sc::validate_inputs(a, 1);
    if (st == DC_OK) st = validate_output(a, 1);
    if (st == DC_OK) st = check_device();
    if (st != DC_OK) return st;
    const sc::Params p = sc::params_of(a);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a->in_dtype == DC_BF16) return sc::for_lanes(a->state, LaunchStep<__nv_bfloat16>{p, s});
    return sc::for_lanes(a->state, LaunchStep<float>{p, s});
}

}  // extern "C"
