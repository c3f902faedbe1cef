// rms_norm.cu — C entry points of the residual add + RMS norm (include/deltacore_layers.h): checks, launch shapes.
#include <math.h>

#include "../../include/deltacore_layers.h"
#include "host.hpp"
#include "rms_norm.cuh"
#include "rows.hpp"

namespace {

using namespace dc::host;

constexpr int kThreads = 256, kMaxThreads = 512;

bool valid_stride(int64_t stride, int64_t width, int64_t rows) { return rows <= 1 || stride >= width; }

Rows rows_of(const void *p, int64_t rows, int64_t stride, int64_t width, int64_t elem) { return {p, 1, rows, 0, stride * elem, width * elem}; }

// Whether every row of a tensor starts on a 16-byte boundary (8 for one-byte elements).
bool rows_aligned(const void *p, int64_t stride, int64_t elem, int64_t rows) {
    if (!p) return true;
    const int64_t a = elem == 1 ? 8 : 16;
    return aligned(p, (size_t)a) && (rows <= 1 || (stride * elem) % a == 0);
}

struct Shape {
    int tpr, vpt, threads;
};

// Threads per row for `accesses` of eight columns per thread (the others are in flight with the first) where there are
// rows enough to fill the card, and one where there are few rows and a row's own latency is all that counts.
Shape shape_of(int64_t rows, int64_t width, int accesses) {
    const int64_t vecs = ceil_div(width, dc::rms::kVec);
    const int want = rows <= 2 * (int64_t)sm_count() ? 1 : accesses;
    Shape s;
    s.tpr = 32;
    while (s.tpr < kMaxThreads && (int64_t)s.tpr * want < vecs) s.tpr *= 2;
    s.vpt = (int)ceil_div(vecs, s.tpr);
    s.vpt = s.vpt <= 1 ? 1 : s.vpt <= 2 ? 2 : 4;
    s.threads = s.tpr > kThreads ? s.tpr : kThreads;
    return s;
}

// Two accesses; four for wide rows of 16-bit values, whose CTAs would otherwise be 512 threads (8192 x 8192 in bfloat16:
// 86 us, 100 with two; with a float32 residual four no longer fit the registers).
Shape fwd_shape(const dc_rms_norm_args *a) {
    const bool narrow = a->x_dtype == DC_BF16 && (!a->residual_in || a->residual_dtype == DC_BF16);
    return shape_of(a->rows, a->width, narrow && a->width > 4096 ? 4 : 2);
}
Shape bwd_shape(const dc_rms_norm_bwd_args *a) { return shape_of(a->rows, a->width, 2); }

int validate_norm(const dc_rms_norm_args *a) {
    if (!a) return DC_EINVAL_ARG;
    if (a->rows < 0 || a->width < 1) return DC_EINVAL_SHAPE;
    if (a->width > DC_RMS_MAX_WIDTH) return DC_EUNSUPPORTED;
    const bool f8 = a->out_dtype == DC_E4M3, res = a->residual_in || a->residual_out;
    if (!valid_dtype(a->x_dtype) || (!f8 && !valid_dtype(a->out_dtype)) || (res && !valid_dtype(a->residual_dtype)))
        return DC_EUNSUPPORTED_DTYPE;
    if (!(a->eps >= 0.f) || !isfinite(a->eps)) return DC_EINVAL_ARG;
    if (f8) {
        if (a->group != 0 && a->group != 32 && a->group != 64 && a->group != 128 && a->group != 256) return DC_EINVAL_WIDTH;
        if (a->group && a->width % a->group) return DC_EINVAL_SHAPE;
    } else if (a->group) {
        return DC_EINVAL_ARG;
    }
    if (!valid_stride(a->x_stride, a->width, a->rows) || !valid_stride(a->y_stride, a->width, a->rows)) return DC_EINVAL_SHAPE;
    if (a->residual_in && !valid_stride(a->residual_in_stride, a->width, a->rows)) return DC_EINVAL_SHAPE;
    if (a->residual_out && !valid_stride(a->residual_out_stride, a->width, a->rows)) return DC_EINVAL_SHAPE;
    if (a->rows == 0) return DC_OK;
    if (!a->x || !a->weight || !a->y || (f8 && !a->scale)) return DC_EINVAL_ARG;
    if (!aligned(a->x, dtype_size(a->x_dtype)) || !aligned(a->weight, 4) || (!f8 && !aligned(a->y, dtype_size(a->out_dtype))) ||
        (f8 && !aligned(a->scale, 4)))
        return DC_EINVAL_ARG;
    if (res && (!aligned(a->residual_in, dtype_size(a->residual_dtype)) || !aligned(a->residual_out, dtype_size(a->residual_dtype))))
        return DC_EINVAL_ARG;
    // in place only over the very same rows
    if (a->y == a->x && (a->out_dtype != a->x_dtype || a->y_stride != a->x_stride)) return DC_EINVAL_ARG;
    if (a->residual_out && a->residual_out == a->residual_in && a->residual_out_stride != a->residual_in_stride) return DC_EINVAL_ARG;
    if (a->residual_out && a->residual_out == a->y) return DC_EINVAL_ARG;
    if (a->residual_in && a->y == a->residual_in && (a->out_dtype != a->residual_dtype || a->y_stride != a->residual_in_stride))
        return DC_EINVAL_ARG;
    if (a->residual_out && a->residual_out == a->x && (a->residual_dtype != a->x_dtype || a->residual_out_stride != a->x_stride))
        return DC_EINVAL_ARG;
    const int64_t xs = dtype_size(a->x_dtype), rs = res ? dtype_size(a->residual_dtype) : 0, ys = f8 ? 1 : dtype_size(a->out_dtype);
    const Rows x = rows_of(a->x, a->rows, a->x_stride, a->width, xs), rin = rows_of(a->residual_in, a->rows, a->residual_in_stride, a->width, rs);
    const Rows y = rows_of(a->y, a->rows, a->y_stride, a->width, ys), rout = rows_of(a->residual_out, a->rows, a->residual_out_stride, a->width, rs);
    for (const Rows *out : {&y, &rout}) {
        if (rows_meet(a->weight, a->width * 4, *out)) return DC_EINVAL_ARG;
        for (const Rows *in : {&x, &rin})
            if (out->p != in->p && rows_meet(*in, *out)) return DC_EINVAL_ARG;
    }
    if (rows_meet(y, rout)) return DC_EINVAL_ARG;
    if (f8) {
        const int64_t scales = a->rows * (a->group ? a->width / a->group : 1) * 4;
        if (rows_meet(a->scale, scales, x) || rows_meet(a->scale, scales, rin) || rows_meet(a->scale, scales, y) || rows_meet(a->scale, scales, rout))
            return DC_EINVAL_ARG;
    }
    return DC_OK;
}

template <int VPT, bool F8>
void launch_norm(bool vec, unsigned grid, const Shape &sh, const dc::rms::Params &p, cudaStream_t s) {
    using bf16 = __nv_bfloat16;
    constexpr auto kAny = F8 ? dc::rms::Lay::kSide : dc::rms::Lay::kApart;  // the scales' groups are neighbouring columns
    if (!vec) dc::rms::rms_norm_kernel<VPT, F8, kAny><<<grid, sh.threads, 0, s>>>(p, sh.tpr);
    else if (p.x_dt && p.r_dt) dc::rms::rms_norm_vec_kernel<bf16, bf16, VPT, F8><<<grid, sh.threads, 0, s>>>(p, sh.tpr);
    else if (p.x_dt) dc::rms::rms_norm_vec_kernel<bf16, float, VPT, F8><<<grid, sh.threads, 0, s>>>(p, sh.tpr);
    else if (p.r_dt) dc::rms::rms_norm_vec_kernel<float, bf16, VPT, F8><<<grid, sh.threads, 0, s>>>(p, sh.tpr);
    else dc::rms::rms_norm_vec_kernel<float, float, VPT, F8><<<grid, sh.threads, 0, s>>>(p, sh.tpr);
}

// CTAs that stay: `per_sm` for every SM, never more than the rows give.
unsigned grid_of(int64_t rows, const Shape &sh, int per_sm) {
    const int64_t ctas = ceil_div(rows, sh.threads / sh.tpr), cap = (int64_t)sm_count() * per_sm;
    return (unsigned)(ctas < cap ? ctas : cap);
}

// ---------------------------------------------------------------------------------------------- backward
int validate_norm_bwd(const dc_rms_norm_bwd_args *a) {
    if (!a) return DC_EINVAL_ARG;
    if (a->rows < 0 || a->width < 1) return DC_EINVAL_SHAPE;
    if (a->width > DC_RMS_MAX_WIDTH) return DC_EUNSUPPORTED;
    if (!valid_dtype(a->y_dtype) || !valid_dtype(a->r_dtype) || (a->d_x && !valid_dtype(a->x_dtype))) return DC_EUNSUPPORTED_DTYPE;
    if (!(a->eps >= 0.f) || !isfinite(a->eps)) return DC_EINVAL_ARG;
    const int64_t w = a->width, n = a->rows;
    if (!valid_stride(a->d_y_stride, w, n) || !valid_stride(a->r_stride, w, n) || (a->d_r && !valid_stride(a->d_r_stride, w, n)) ||
        (a->d_x && !valid_stride(a->d_x_stride, w, n)) || (a->d_residual && !valid_stride(a->d_residual_stride, w, n)))
        return DC_EINVAL_SHAPE;
    return DC_OK;
}

int validate_norm_bwd_buffers(const dc_rms_norm_bwd_args *a) {
    if (a->rows == 0) return a->d_weight && !aligned(a->d_weight, 4) ? DC_EINVAL_ARG : DC_OK;
    const size_t ys = dtype_size(a->y_dtype), rs = dtype_size(a->r_dtype);
    if (!a->d_y || !a->r || !a->weight) return DC_EINVAL_ARG;
    if (!aligned(a->d_y, ys) || !aligned(a->r, rs) || !aligned(a->d_r, rs) || !aligned(a->d_residual, rs) || !aligned(a->weight, 4) ||
        !aligned(a->d_weight, 4) || !aligned(a->d_x, dtype_size(a->x_dtype)))
        return DC_EINVAL_ARG;
    if (a->d_x && (a->d_x == a->d_residual || (a->d_x == a->d_y && (a->x_dtype != a->y_dtype || a->d_x_stride != a->d_y_stride)) ||
                   (a->d_x == a->d_r && (a->x_dtype != a->r_dtype || a->d_x_stride != a->d_r_stride)) || a->d_x == a->r))
        return DC_EINVAL_ARG;
    if (a->d_residual && ((a->d_residual == a->d_r && a->d_residual_stride != a->d_r_stride) || a->d_residual == a->r ||
                          a->d_residual == a->d_y))
        return DC_EINVAL_ARG;
    const int64_t w = a->width, xs = a->d_x ? dtype_size(a->x_dtype) : 0;
    const Rows dy = rows_of(a->d_y, a->rows, a->d_y_stride, w, ys), dr = rows_of(a->d_r, a->rows, a->d_r_stride, w, rs);
    const Rows r = rows_of(a->r, a->rows, a->r_stride, w, rs), dx = rows_of(a->d_x, a->rows, a->d_x_stride, w, xs);
    const Rows dres = rows_of(a->d_residual, a->rows, a->d_residual_stride, w, rs);
    for (const Rows *out : {&dx, &dres}) {
        if (rows_meet(a->weight, w * 4, *out)) return DC_EINVAL_ARG;
        for (const Rows *in : {&dy, &dr, &r})
            if (out->p != in->p && rows_meet(*in, *out)) return DC_EINVAL_ARG;
    }
    if (rows_meet(dx, dres)) return DC_EINVAL_ARG;
    return DC_OK;
}

unsigned bwd_grid(const dc_rms_norm_bwd_args *a, const Shape &sh) { return grid_of(a->rows, sh, 512 / sh.threads); }

template <int VPT>
void launch_bwd(bool vec, unsigned grid, size_t smem, const Shape &sh, const dc::rms::BwdParams &p, cudaStream_t s) {
    using bf16 = __nv_bfloat16;
    if (!vec) {
        dc::rms::rms_norm_bwd_kernel<VPT, dc::rms::Lay::kApart><<<grid, sh.threads, smem, s>>>(p, sh.tpr);
    } else if constexpr (VPT == 4) {
        dc::rms::rms_norm_bwd_kernel<VPT, dc::rms::Lay::kAligned><<<grid, sh.threads, smem, s>>>(p, sh.tpr);
    } else {
        if (p.y_dt && p.r_dt) dc::rms::rms_norm_bwd_vec_kernel<bf16, bf16, VPT><<<grid, sh.threads, smem, s>>>(p, sh.tpr);
        else if (p.y_dt) dc::rms::rms_norm_bwd_vec_kernel<bf16, float, VPT><<<grid, sh.threads, smem, s>>>(p, sh.tpr);
        else if (p.r_dt) dc::rms::rms_norm_bwd_vec_kernel<float, bf16, VPT><<<grid, sh.threads, smem, s>>>(p, sh.tpr);
        else dc::rms::rms_norm_bwd_vec_kernel<float, float, VPT><<<grid, sh.threads, smem, s>>>(p, sh.tpr);
    }
}

}  // namespace

extern "C" {

int dc_rms_norm(const dc_rms_norm_args *a, dc_stream_t stream) {
    int st = validate_norm(a);
    if (st != DC_OK) return st;
    if (a->rows == 0) return DC_OK;
    st = check_device();
    if (st != DC_OK) return st;
    const bool f8 = a->out_dtype == DC_E4M3;
    dc::rms::Params p{};
    p.rows = a->rows;
    p.width = (int32_t)a->width;
    p.group = a->group;
    p.groups = a->group ? (int32_t)(a->width / a->group) : 1;
    while (a->group && (dc::rms::kVec << p.group_shift) < a->group) ++p.group_shift;
    p.x_stride = a->x_stride, p.rin_stride = a->residual_in_stride, p.rout_stride = a->residual_out_stride, p.y_stride = a->y_stride;
    p.x_dt = a->x_dtype, p.r_dt = a->residual_dtype, p.y_dt = f8 ? 0 : a->out_dtype;
    p.eps = a->eps;
    p.x = a->x, p.rin = a->residual_in, p.weight = a->weight;
    p.rout = a->residual_out, p.y = a->y, p.scale = a->scale;
    const int64_t xs = dtype_size(a->x_dtype), rs = dtype_size(a->residual_dtype), ys = f8 ? 1 : dtype_size(a->out_dtype);
    const bool vec = a->width % dc::rms::kVec == 0 && rows_aligned(a->x, a->x_stride, xs, a->rows) &&
                     rows_aligned(a->residual_in, a->residual_in_stride, rs, a->rows) &&
                     rows_aligned(a->residual_out, a->residual_out_stride, rs, a->rows) &&
                     rows_aligned(a->y, a->y_stride, ys, a->rows) && aligned(a->weight, 16);
    const Shape sh = fwd_shape(a);
    const unsigned grid = grid_of(a->rows, sh, 2048 / sh.threads);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    switch (sh.vpt * 2 + (f8 ? 1 : 0)) {
        case 2: launch_norm<1, false>(vec, grid, sh, p, s); break;
        case 3: launch_norm<1, true>(vec, grid, sh, p, s); break;
        case 4: launch_norm<2, false>(vec, grid, sh, p, s); break;
        case 5: launch_norm<2, true>(vec, grid, sh, p, s); break;
        case 8: launch_norm<4, false>(vec, grid, sh, p, s); break;
        default: launch_norm<4, true>(vec, grid, sh, p, s); break;
    }
    return launched();
}

uint64_t dc_rms_norm_bwd_workspace_size(const dc_rms_norm_bwd_args *a) {
    if (validate_norm_bwd(a) != DC_OK || !a->d_weight || a->rows == 0) return 0;
    return (uint64_t)bwd_grid(a, bwd_shape(a)) * (uint64_t)a->width * 4;
}

int dc_rms_norm_bwd(const dc_rms_norm_bwd_args *a, dc_stream_t stream) {
    int st = validate_norm_bwd(a);
    if (st == DC_OK) st = validate_norm_bwd_buffers(a);
    if (st != DC_OK) return st;
    if (a->d_weight && a->rows > 0) {
        if (a->workspace_bytes < dc_rms_norm_bwd_workspace_size(a)) return DC_EWORKSPACE;
        if (!a->workspace || !aligned(a->workspace, 16)) return DC_EINVAL_ARG;
    }
    st = check_device();
    if (st != DC_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a->rows == 0) {
        if (!a->d_weight) return DC_OK;
        const cudaError_t e = cudaMemsetAsync(a->d_weight, 0, (size_t)a->width * 4, s);
        return e == cudaSuccess ? DC_OK : cuda_fail(e);
    }
    dc::rms::BwdParams p{};
    p.rows = a->rows;
    p.width = (int32_t)a->width;
    p.dy_stride = a->d_y_stride, p.dr_stride = a->d_r_stride, p.r_stride = a->r_stride, p.dx_stride = a->d_x_stride;
    p.dres_stride = a->d_residual_stride;
    p.y_dt = a->y_dtype, p.r_dt = a->r_dtype, p.x_dt = a->x_dtype;
    p.eps = a->eps;
    p.dy = a->d_y, p.dr = a->d_r, p.r = a->r, p.weight = a->weight, p.dx = a->d_x, p.dres = a->d_residual;
    p.part = a->d_weight ? static_cast<float *>(a->workspace) : nullptr;
    const int64_t ys = dtype_size(a->y_dtype), rs = dtype_size(a->r_dtype), xs = dtype_size(a->x_dtype);
    const bool vec = a->width % dc::rms::kVec == 0 && rows_aligned(a->d_y, a->d_y_stride, ys, a->rows) &&
                     rows_aligned(a->d_r, a->d_r_stride, rs, a->rows) && rows_aligned(a->r, a->r_stride, rs, a->rows) &&
                     rows_aligned(a->d_x, a->d_x_stride, xs, a->rows) && rows_aligned(a->d_residual, a->d_residual_stride, rs, a->rows) &&
                     aligned(a->weight, 16);
    const Shape sh = bwd_shape(a);
    const unsigned grid = bwd_grid(a, sh);
    const size_t smem = (size_t)(sh.threads / sh.tpr - 1) * (size_t)a->width * 4;
    switch (sh.vpt) {
        case 1: launch_bwd<1>(vec, grid, smem, sh, p, s); break;
        case 2: launch_bwd<2>(vec, grid, smem, sh, p, s); break;
        default: launch_bwd<4>(vec, grid, smem, sh, p, s); break;
    }
    st = launched();
    if (st != DC_OK || !a->d_weight) return st;
    dc::column_sum_kernel<<<(unsigned)ceil_div(a->width, 32), dc::kColThreads, 0, s>>>(p.part, grid, a->width, a->width, a->d_weight);
    return launched();
}

}  // extern "C"
