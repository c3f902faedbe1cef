// causal_conv.cu — C entry points of the causal depthwise convolution (include/deltacore_layers.h): checks and
// launch shapes.
#include "../../include/deltacore_layers.h"
#include "causal_conv.cuh"
#include "host.hpp"
#include "rows.hpp"

namespace {

using namespace dc::host;
namespace cv = dc::conv;

static_assert(DC_CONV_MAX_TAPS == cv::kMaxTaps, "the header's limit is the kernels'");

bool valid_strides(int64_t batch, int64_t seq, int64_t channels, int64_t bs, int64_t ts) {
    return (seq <= 1 || ts >= channels) && (batch <= 1 || bs >= 0);
}

int validate_dims(int64_t batch, int64_t seq, int64_t channels, int32_t taps, int32_t in_dt, int32_t out_dt, uint32_t flags) {
    if (batch < 0 || seq < 0 || channels < 0) return DC_EINVAL_SHAPE;
    if (taps < 1) return DC_EINVAL_ARG;
    if (!valid_dtype(in_dt) || !valid_dtype(out_dt)) return DC_EUNSUPPORTED_DTYPE;
    if (flags & ~DC_CONV_SILU) return DC_EINVAL_ARG;
    if (taps > DC_CONV_MAX_TAPS || channels > (int64_t)65535 * 32 || batch > 0x7fffffff || seq > 0x7fffffff) return DC_EUNSUPPORTED;
    return DC_OK;
}

// Whether every row of a tensor starts on a boundary of `n` elements.
bool vectors(const void *p, int64_t bs, int64_t ts, int64_t elem, int64_t n) {
    return aligned(p, (size_t)(elem * n)) && bs % n == 0 && ts % n == 0;
}

// Tokens per thread: halved from `most` until there are 24 warps for every SM, or `least` is reached.  Each run reads K - 1
// tokens of its neighbour again (5 % at 64 tokens and 4 taps).  24 is what the forward holds on an SM (the backward holds 16);
// halving may give up to twice that.  Chosen at one shape: ragged 6 x 2049 x 1536 forward takes 19 us at 24 warps, 23 at 16; with
// 48 the runs of its backward get too short.
int run_length(int64_t batch, int64_t seq, int64_t groups, int least, int most) {
    int run = most;
    while (run > least && batch * ceil_div(seq, run) * groups < (int64_t)sm_count() * 24) run /= 2;
    return run;
}

int validate_conv(const dc_causal_conv_args *a) {
    if (!a) return DC_EINVAL_ARG;
    const int st = validate_dims(a->batch, a->seq, a->channels, a->taps, a->in_dtype, a->out_dtype, a->flags);
    if (st != DC_OK) return st;
    if (a->batch == 0 || a->channels == 0) return DC_OK;
    if (!a->weight || (a->seq > 0 && (!a->x || !a->y))) return DC_EINVAL_ARG;
    const int64_t is = dtype_size(a->in_dtype), os = dtype_size(a->out_dtype);
    if (!aligned(a->x, is) || !aligned(a->y, os) || !aligned(a->weight, 4) || !aligned(a->bias, 4) || !aligned(a->window_in, 4) ||
        !aligned(a->window_out, 4) || !aligned(a->lengths, 4))
        return DC_EINVAL_ARG;
    if (!valid_strides(a->batch, a->seq, a->channels, a->x_batch_stride, a->x_token_stride) ||
        !valid_strides(a->batch, a->seq, a->channels, a->y_batch_stride, a->y_token_stride))
        return DC_EINVAL_SHAPE;
    const int64_t wb = a->batch * a->channels * a->taps * 4;
    if (overlap(a->window_in, wb, a->window_out, wb) && !(a->seq == 1 && a->window_in == a->window_out)) return DC_EINVAL_ARG;
    const Rows x{a->x, a->batch, a->seq, a->x_batch_stride * is, a->x_token_stride * is, a->channels * is};
    const Rows y{a->y, a->batch, a->seq, a->y_batch_stride * os, a->y_token_stride * os, a->channels * os};
    if (rows_fold(y)) return DC_EINVAL_SHAPE;
    if (rows_meet(x, y)) return DC_EINVAL_ARG;
    return DC_OK;
}

template <typename TI, typename TO, bool STAGED>
int launch_conv(const cv::Params &p, dim3 grid, cudaStream_t s) {
    const size_t smem = STAGED ? sizeof(typename cv::FwdRing<TI>::Buffer) * (cv::kThreads / 32) : 0;
    auto go = [&](auto *kernel) {
        if (smem > 48 * 1024) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return cuda_fail(e);
        }
        kernel<<<grid, cv::kThreads, smem, s>>>(p);
        return launched();
    };
    switch (p.K) {
        case 2: return go(&cv::conv_kernel<TI, TO, STAGED, 2>);
        case 3: return go(&cv::conv_kernel<TI, TO, STAGED, 3>);
        case 4: return go(&cv::conv_kernel<TI, TO, STAGED, 4>);
        default: return go(&cv::conv_kernel<TI, TO, STAGED, cv::kMaxTaps>);
    }
}

template <typename TI>
int run_conv(const dc_causal_conv_args *a, cv::Params p, cudaStream_t s) {
    if (a->seq == 1) {
        cv::conv_step_kernel<TI><<<(unsigned)ceil_div(a->batch * a->channels, 256), 256, 0, s>>>(p);
        return launched();
    }
    const int64_t el = 16 / (int64_t)sizeof(TI);
    const bool staged = a->channels % el == 0 && vectors(a->x, p.x_b, p.x_t, sizeof(TI), el);
    p.y_pair = vectors(a->y, p.y_b, p.y_t, dtype_size(a->out_dtype), cv::kVec);
    const int64_t groups = ceil_div(a->channels, cv::kRow);
    p.run = run_length(a->batch, a->seq, groups, cv::kStageTokens, 128);
    p.runs = (int32_t)(a->seq > 0 ? ceil_div(a->seq, p.run) : 1);
    const int64_t ctas = ceil_div(a->batch * p.runs, cv::kThreads / 32);
    if (ctas > 0x7fffffff) return DC_EUNSUPPORTED;
    const dim3 grid((unsigned)ctas, (unsigned)groups);
    if (a->out_dtype == DC_BF16)
        return staged ? launch_conv<TI, __nv_bfloat16, true>(p, grid, s) : launch_conv<TI, __nv_bfloat16, false>(p, grid, s);
    return staged ? launch_conv<TI, float, true>(p, grid, s) : launch_conv<TI, float, false>(p, grid, s);
}

// ---------------------------------------------------------------------------------------------- backward
int validate_bwd_dims(const dc_causal_conv_bwd_args *a) {
    if (!a) return DC_EINVAL_ARG;
    return validate_dims(a->batch, a->seq, a->channels, a->taps, a->in_dtype, a->out_dtype, a->flags);
}

int validate_bwd(const dc_causal_conv_bwd_args *a) {
    if (a->channels == 0) return DC_OK;
    if (!a->weight || !a->d_weight) return DC_EINVAL_ARG;
    if (a->batch == 0) return DC_OK;
    if (a->seq > 0 && (!a->x || !a->d_y || !a->d_x)) return DC_EINVAL_ARG;
    const int64_t is = dtype_size(a->in_dtype), os = dtype_size(a->out_dtype);
    const void *f32s[] = {a->weight, a->bias, a->window_in, a->lengths, a->d_window_out, a->d_weight, a->d_bias, a->d_window_in};
    for (const void *q : f32s)
        if (!aligned(q, 4)) return DC_EINVAL_ARG;
    if (!aligned(a->x, is) || !aligned(a->d_x, is) || !aligned(a->d_y, os)) return DC_EINVAL_ARG;
    if (!valid_strides(a->batch, a->seq, a->channels, a->x_batch_stride, a->x_token_stride) ||
        !valid_strides(a->batch, a->seq, a->channels, a->d_y_batch_stride, a->d_y_token_stride) ||
        !valid_strides(a->batch, a->seq, a->channels, a->d_x_batch_stride, a->d_x_token_stride))
        return DC_EINVAL_SHAPE;
    const Rows x{a->x, a->batch, a->seq, a->x_batch_stride * is, a->x_token_stride * is, a->channels * is};
    const Rows dy{a->d_y, a->batch, a->seq, a->d_y_batch_stride * os, a->d_y_token_stride * os, a->channels * os};
    const Rows dx{a->d_x, a->batch, a->seq, a->d_x_batch_stride * is, a->d_x_token_stride * is, a->channels * is};
    if (rows_fold(dx)) return DC_EINVAL_SHAPE;
    // a run's neighbour still reads what the run would overwrite
    if (rows_meet(x, dx) || rows_meet(dy, dx)) return DC_EINVAL_ARG;
    const int64_t wb = a->batch * a->channels * a->taps * 4;
    if (overlap(a->d_window_in, wb, a->d_window_out, wb) || overlap(a->d_window_in, wb, a->window_in, wb)) return DC_EINVAL_ARG;
    return DC_OK;
}

struct BwdShape {
    bool staged, pair;  // x and d_y through rings; pairs of d_x's channels aligned
    int run;
    int64_t runs, groups, ctas;
};

BwdShape bwd_shape(const dc_causal_conv_bwd_args *a) {
    const int64_t is = dtype_size(a->in_dtype), os = dtype_size(a->out_dtype);
    BwdShape b;
    b.staged = a->channels % (16 / is) == 0 && vectors(a->x, a->x_batch_stride, a->x_token_stride, is, 16 / is) &&
               a->channels % (16 / os) == 0 && vectors(a->d_y, a->d_y_batch_stride, a->d_y_token_stride, os, 16 / os);
    b.pair = vectors(a->d_x, a->d_x_batch_stride, a->d_x_token_stride, is, cv::kVec);
    b.groups = ceil_div(a->channels, cv::kRow);
    b.run = run_length(a->batch, a->seq, b.groups, 16, 64);
    b.runs = a->seq > 0 ? ceil_div(a->seq, b.run) : 1;
    b.ctas = ceil_div(a->batch * b.runs, cv::kBwdThreads / 32);
    return b;
}

template <typename TI, typename TO, bool STAGED>
int launch_bwd(const cv::BwdParams &p, dim3 grid, cudaStream_t s) {
    const size_t smem = STAGED ? sizeof(cv::BwdRings<TI, TO>) * (cv::kBwdThreads / 32) : 0;
    auto go = [&](auto *kernel) {
        if (smem + sizeof(float2) * cv::kBwdThreads > 48 * 1024) {  // with the kernel's sums, which lie beside the rings
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return cuda_fail(e);
        }
        kernel<<<grid, cv::kBwdThreads, smem, s>>>(p);
        return launched();
    };
    switch (p.K) {
        case 2: return go(&cv::conv_bwd_kernel<TI, TO, STAGED, 2>);
        case 3: return go(&cv::conv_bwd_kernel<TI, TO, STAGED, 3>);
        case 4: return go(&cv::conv_bwd_kernel<TI, TO, STAGED, 4>);
        default: return go(&cv::conv_bwd_kernel<TI, TO, STAGED, cv::kMaxTaps>);
    }
}

template <typename TI>
int launch_bwd_as(bool staged, const cv::BwdParams &p, dim3 grid, cudaStream_t s) {
    if (p.y_dt) return staged ? launch_bwd<TI, __nv_bfloat16, true>(p, grid, s) : launch_bwd<TI, __nv_bfloat16, false>(p, grid, s);
    return staged ? launch_bwd<TI, float, true>(p, grid, s) : launch_bwd<TI, float, false>(p, grid, s);
}

}  // namespace

extern "C" {

int dc_causal_conv(const dc_causal_conv_args *a, dc_stream_t stream) {
    int st = validate_conv(a);
    if (st != DC_OK) return st;
    if (a->batch == 0 || a->channels == 0) return DC_OK;
    st = check_device();
    if (st != DC_OK) return st;
    cv::Params p{};
    p.batch = a->batch, p.seq = a->seq, p.channels = a->channels;
    p.x_b = a->x_batch_stride, p.x_t = a->x_token_stride, p.y_b = a->y_batch_stride, p.y_t = a->y_token_stride;
    p.K = a->taps;
    p.silu = (a->flags & DC_CONV_SILU) ? 1 : 0;
    p.y_dt = a->out_dtype;
    p.x = a->x, p.weight = a->weight, p.bias = a->bias, p.window_in = a->window_in, p.lengths = a->lengths;
    p.y = a->y, p.window_out = a->window_out;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return a->in_dtype == DC_BF16 ? run_conv<__nv_bfloat16>(a, p, s) : run_conv<float>(a, p, s);
}

uint64_t dc_causal_conv_bwd_workspace_size(const dc_causal_conv_bwd_args *a) {
    if (validate_bwd_dims(a) != DC_OK || a->batch == 0 || a->channels == 0) return 0;
    return (uint64_t)bwd_shape(a).ctas * (uint64_t)(a->taps + 1) * (uint64_t)a->channels * 4;
}

int dc_causal_conv_bwd(const dc_causal_conv_bwd_args *a, dc_stream_t stream) {
    int st = validate_bwd_dims(a);
    if (st == DC_OK) st = validate_bwd(a);
    if (st != DC_OK) return st;
    if (a->channels == 0) return DC_OK;
    if (a->batch > 0) {
        if (a->workspace_bytes < dc_causal_conv_bwd_workspace_size(a)) return DC_EWORKSPACE;
        if (!a->workspace || !aligned(a->workspace, 16)) return DC_EINVAL_ARG;
    }
    st = check_device();
    if (st != DC_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int64_t ctas = 0;  // no sequence: the sums are zero
    cv::BwdParams p{};
    if (a->batch > 0) {
        const BwdShape b = bwd_shape(a);
        if (b.ctas > 0x7fffffff) return DC_EUNSUPPORTED;
        ctas = b.ctas;
        p.batch = a->batch, p.seq = a->seq, p.channels = a->channels;
        p.x_b = a->x_batch_stride, p.x_t = a->x_token_stride, p.dy_b = a->d_y_batch_stride, p.dy_t = a->d_y_token_stride;
        p.dx_b = a->d_x_batch_stride, p.dx_t = a->d_x_token_stride;
        p.K = a->taps;
        p.silu = (a->flags & DC_CONV_SILU) ? 1 : 0;
        p.run = b.run, p.runs = (int32_t)b.runs, p.dx_pair = b.pair;
        p.y_dt = a->out_dtype;
        p.dy = a->d_y, p.x = a->x, p.dwin_out = a->d_window_out, p.weight = a->weight, p.bias = a->bias, p.window_in = a->window_in;
        p.lengths = a->lengths;
        p.dx = a->d_x, p.dwin_in = a->d_window_in;
        p.part = static_cast<float *>(a->workspace);
        const dim3 grid((unsigned)b.ctas, (unsigned)b.groups);
        st = a->in_dtype == DC_BF16 ? launch_bwd_as<__nv_bfloat16>(b.staged, p, grid, s) : launch_bwd_as<float>(b.staged, p, grid, s);
        if (st != DC_OK) return st;
    }
    cv::conv_bwd_sum_kernel<<<dim3((unsigned)ceil_div(a->channels, 32), (unsigned)(a->taps + 1)), 256, 0, s>>>(
        static_cast<const float *>(a->workspace), ctas, a->channels, a->taps, a->d_weight, a->d_bias);
    return launched();
}

}  // extern "C"
