// selective_scan.cu — C entry points of the selective scan and its decode tick (include/deltacore_layers.h).
#include "selective_scan_host.hpp"

namespace {

using namespace dc::host;
namespace sc = dc::scan;

static_assert(DC_SCAN_MAX_STATE == 16 * sc::kS, "the header's limit is the kernels'");

int validate_output(const dc_selective_scan_args *a, int64_t seq) {
    const int64_t os = dtype_size(a->out_dtype), c = a->channels, states = a->batch * c * a->state * 4;
    // in place, or apart: a CTA that runs later would read what another one wrote
    if (a->state_out != a->state_in && overlap(a->state_out, states, a->state_in, states)) return DC_EINVAL_ARG;
    if (seq == 0) return DC_OK;
    if (!a->y || !aligned(a->y, os)) return DC_EINVAL_ARG;
    if ((seq > 1 && a->y_token_stride < c) || (a->batch > 1 && a->y_batch_stride < c)) return DC_EINVAL_SHAPE;
    const Rows y{a->y, a->batch, seq, a->y_batch_stride * os, a->y_token_stride * os, c * os};
    if (rows_fold(y)) return DC_EINVAL_SHAPE;
    if (sc::meets_inputs(a, seq, y) || rows_meet(a->a, c * a->state * 4, y) || rows_meet(a->d, c * 4, y) || rows_meet(a->dt_bias, c * 4, y) ||
        rows_meet(a->state_in, states, y) || rows_meet(a->state_out, states, y))
        return DC_EINVAL_ARG;
    return DC_OK;
}

// How a prompt is cut (selective_scan.cuh): segments side by side, or a walk of `pieces` pieces of `piece` tokens.
struct Cut {
    bool segments;
    int64_t pieces, piece;
};

// By the CTAs that the walk would give and those that the card holds (`room`).  Measured, state 16, bfloat16, microseconds:
//   8 x 4096 x 2048 (1024 CTAs): walk 463, segments 1067      4 x 2048 x 2048 (512): walk 151, segments 311
//   2 x 4096 x 2048 (256): walk 254, segments 310, 4 pieces 213
//   1 x 4096 x 2048 (128): walk 223, segments 159, 8 pieces 116
//   1 x 16384 x 1024 (64): walk 872, segments 478, 16 pieces 220
// So: the walk from a third of the room on; below that as many pieces as fill the room, each 128 tokens at least, if
// that makes three or more of them; else segments.
Cut cut_of(const dc_selective_scan_args *a, bool workspace) {
    constexpr int64_t kLeast = 128;
    const int lanes = sc::lanes_of(a->state);
    const int64_t ctas = a->batch * a->groups * ceil_div(a->channels / a->groups, sc::walk_channels(lanes));
    const int64_t room = (int64_t)sm_count() * sc::walk_ctas(lanes, dtype_size(a->in_dtype));
    Cut c{false, 1, a->seq};
    if (3 * ctas > room) return c;
    const int64_t want = room / ctas, most = a->seq / kLeast, pieces = want < most ? want : most;
    if (workspace && pieces >= 3) {
        c.piece = ceil_div(ceil_div(a->seq, pieces), sc::kTile) * sc::kTile;  // (still three or more: seq >= 3 kLeast)
        c.pieces = ceil_div(a->seq, c.piece);
    } else {
        c.segments = true;
    }
    return c;
}

// Floats of the pieces' end states, then of their sums of steps.
int64_t piece_floats(const dc_selective_scan_args *a, const Cut &c) {
    return c.pieces > 1 ? a->batch * a->channels * (c.pieces * a->state + c.pieces - 1) : 0;
}

template <typename Smem, typename K>
int launch(K *kernel, const sc::Params &p, int64_t ctas, int threads, cudaStream_t s) {
    if (ctas > 0x7fffffff) return DC_EUNSUPPORTED;
    if (sizeof(Smem) > 48 * 1024) {
        const int st = sc::allow_smem(kernel, sizeof(Smem));
        if (st != DC_OK) return st;
    }
    kernel<<<(unsigned)ctas, threads, sizeof(Smem), s>>>(p);
    return launched();
}

template <typename TI>
struct Launch {
    const sc::Params &p;
    const Cut &c;
    cudaStream_t s;
    template <int P>
    int operator()() const {
        using Walk = sc::WalkShape<P>;
        using Seg = sc::SegShape<P>;
        const int64_t seqs = p.batch * p.groups;
        if (c.segments)
            return launch<sc::SegSmem<TI, P>>(&sc::scan_segments_kernel<TI, P>, p, seqs * ceil_div(p.per, Seg::kCh), Seg::kNT, s);
        const int64_t blocks = seqs * ceil_div(p.per, Walk::kCh);
        if (c.pieces > 1) {
            const int st = launch<sc::WalkSmem<TI, P>>(&sc::scan_walk_kernel<TI, P, false>, p, blocks * (c.pieces - 1), Walk::kNT, s);
            if (st != DC_OK) return st;
        }
        return launch<sc::WalkSmem<TI, P>>(&sc::scan_walk_kernel<TI, P, true>, p, blocks * c.pieces, Walk::kNT, s);
    }
};

template <typename TI>
struct LaunchStep {
    const sc::Params &p;
    cudaStream_t s;
    template <int P>
    int operator()() const {
        // several sequences per thread where that still leaves two CTAs for every SM
        const int64_t blocks = ceil_div(p.channels, sc::kThreads / P), seqs = ceil_div(p.batch, sc::kStepSeqs);
        const bool many = blocks * seqs >= 2 * (int64_t)sm_count();
        const int64_t rows = many ? seqs : p.batch;
        if (blocks > 0x7fffffff) return DC_EUNSUPPORTED;
        constexpr int64_t kRows = 65535;  // of a grid's second axis
        const dim3 grid((unsigned)blocks, (unsigned)(rows < kRows ? rows : kRows), (unsigned)ceil_div(rows, kRows));
        // every group of four states whole and aligned
        const int64_t four = 4 * (int64_t)sizeof(TI);
        const bool whole = p.N == 4 * P && aligned(p.a, 16) && aligned(p.state_in, 16) && aligned(p.state_out, 16) && aligned(p.b, four) &&
                           aligned(p.c, four) && (p.batch == 1 || (p.b_b % 4 == 0 && p.c_b % 4 == 0));
        if (many && whole) sc::scan_step_kernel<TI, P, sc::kStepSeqs, true><<<grid, sc::kThreads, 0, s>>>(p);
        else if (many) sc::scan_step_kernel<TI, P, sc::kStepSeqs, false><<<grid, sc::kThreads, 0, s>>>(p);
        else if (whole) sc::scan_step_kernel<TI, P, 1, true><<<grid, sc::kThreads, 0, s>>>(p);
        else sc::scan_step_kernel<TI, P, 1, false><<<grid, sc::kThreads, 0, s>>>(p);
        return launched();
    }
};

}  // namespace

extern "C" {

uint64_t dc_selective_scan_checkpoint_size(const dc_selective_scan_args *a) {
    if (sc::validate_dims(a) != DC_OK) return 0;
    return (uint64_t)a->batch * (uint64_t)ceil_div(a->seq, sc::kTile) * (uint64_t)a->channels * (uint64_t)a->state * 4;
}

uint64_t dc_selective_scan_workspace_size(const dc_selective_scan_args *a) {
    if (sc::validate_dims(a) != DC_OK || a->batch == 0 || a->channels == 0) return 0;
    return (uint64_t)piece_floats(a, cut_of(a, true)) * 4;
}

int dc_selective_scan(const dc_selective_scan_args *a, dc_stream_t stream) {
    int st = sc::validate_dims(a);
    if (st != DC_OK) return st;
    if (a->batch == 0 || a->channels == 0) return DC_OK;
    st = sc::validate_inputs(a, a->seq);
    if (st == DC_OK) st = validate_output(a, a->seq);
    if (st == DC_OK) st = check_device();
    if (st != DC_OK) return st;
    const Cut c = cut_of(a, a->workspace != nullptr);
    if (c.pieces > 1) {
        if (a->workspace_bytes < (uint64_t)piece_floats(a, c) * 4) return DC_EWORKSPACE;
        if (!aligned(a->workspace, 16)) return DC_EINVAL_ARG;
    }
    sc::Params p = sc::params_of(a);
    p.pieces = (int32_t)c.pieces;
    p.piece = c.piece;
    p.piece_end = static_cast<float *>(a->workspace);
    p.piece_step = p.piece_end + a->batch * a->channels * c.pieces * a->state;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a->in_dtype == DC_BF16) return sc::for_lanes(a->state, Launch<__nv_bfloat16>{p, c, s});
    return sc::for_lanes(a->state, Launch<float>{p, c, s});
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
