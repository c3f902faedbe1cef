// selective_scan_host.hpp — the argument checks and kernel parameters that the selective scan's forward and backward
// entry points share.
#pragma once

#include "../../include/deltacore_layers.h"
#include "host.hpp"
#include "rows.hpp"
#include "selective_scan.cuh"

namespace dc {
namespace scan {

// Threads per channel: four states each, rounded up to a power of two.
inline int lanes_of(int64_t state) {
    int p = 1;
    while (p * kS < state) p *= 2;
    return p;
}
inline int validate_dims(const dc_selective_scan_args *a) {
    if (!a) return DC_EINVAL_ARG;
    if (a->batch < 0 || a->seq < 0 || a->channels < 0 || a->state < 1 || a->groups < 1) return DC_EINVAL_SHAPE;
    if (a->channels % a->groups) return DC_EINVAL_SHAPE;
    if (!host::valid_dtype(a->in_dtype) || !host::valid_dtype(a->out_dtype)) return DC_EUNSUPPORTED_DTYPE;
    if (a->flags & ~DC_SCAN_SOFTPLUS) return DC_EINVAL_ARG;
    if (a->state > DC_SCAN_MAX_STATE || a->batch > 0x7fffffff || a->seq > 0x7fffffff || a->channels > 0x7fffffff) return DC_EUNSUPPORTED;
    return DC_OK;
}

// The inputs of a call with `seq` tokens (1 in the step), after validate_dims.
inline int validate_inputs(const dc_selective_scan_args *a, int64_t seq) {
    using namespace host;
    const size_t is = dtype_size(a->in_dtype);
    if (!a->a || (seq > 0 && (!a->u || !a->dt || !a->b || !a->c))) return DC_EINVAL_ARG;
    const void *ins[] = {a->u, a->dt, a->z, a->b, a->c};
    for (const void *q : ins)
        if (!aligned(q, is)) return DC_EINVAL_ARG;
    const void *f32s[] = {a->a, a->d, a->dt_bias, a->state_in, a->state_out, a->lengths, a->checkpoints};
    for (const void *q : f32s)
        if (!aligned(q, 4)) return DC_EINVAL_ARG;
    const int64_t c = a->channels, n = a->groups * a->state;
    const int64_t strides[][3] = {{a->u_batch_stride, a->u_token_stride, c}, {a->dt_batch_stride, a->dt_token_stride, c},
                                  {a->z_batch_stride, a->z_token_stride, a->z ? c : 0}, {a->b_batch_stride, a->b_token_stride, n},
                                  {a->c_batch_stride, a->c_token_stride, n}};
    for (const auto &s : strides)
        if (s[2] && ((seq > 1 && s[1] < s[2]) || (seq > 0 && a->batch > 1 && s[0] < s[2]))) return DC_EINVAL_SHAPE;
    return DC_OK;
}

// Whether rows that a call writes meet what it reads token by token (with `seq` tokens).
inline bool meets_inputs(const dc_selective_scan_args *a, int64_t seq, const host::Rows &out) {
    const int64_t is = host::dtype_size(a->in_dtype), c = a->channels * is, n = a->groups * a->state * is;
    const host::Rows ins[] = {{a->u, a->batch, seq, a->u_batch_stride * is, a->u_token_stride * is, c},
                              {a->dt, a->batch, seq, a->dt_batch_stride * is, a->dt_token_stride * is, c},
                              {a->z, a->batch, seq, a->z_batch_stride * is, a->z_token_stride * is, c},
                              {a->b, a->batch, seq, a->b_batch_stride * is, a->b_token_stride * is, n},
                              {a->c, a->batch, seq, a->c_batch_stride * is, a->c_token_stride * is, n}};
    for (const host::Rows &in : ins)
        if (host::rows_meet(in, out)) return true;
    return false;
}

inline Params params_of(const dc_selective_scan_args *a) {
    Params p{};
    p.batch = a->batch, p.seq = a->seq, p.channels = a->channels, p.groups = a->groups, p.per = a->channels / a->groups;
    p.N = (int32_t)a->state;
    p.u_b = a->u_batch_stride, p.u_t = a->u_token_stride, p.dt_b = a->dt_batch_stride, p.dt_t = a->dt_token_stride;
    p.z_b = a->z_batch_stride, p.z_t = a->z_token_stride, p.b_b = a->b_batch_stride, p.b_t = a->b_token_stride;
    p.c_b = a->c_batch_stride, p.c_t = a->c_token_stride, p.y_b = a->y_batch_stride, p.y_t = a->y_token_stride;
    p.softplus = (a->flags & DC_SCAN_SOFTPLUS) ? 1 : 0;
    p.y_dt = a->out_dtype;
    const int64_t is = host::dtype_size(a->in_dtype);
    auto how = [](int64_t bytes) { return bytes % 16 == 0 ? kVectors : bytes % 4 == 0 ? kWords : kScalar; };
    auto least = [](int a, int b) { return a < b ? a : b; };
    p.vec_x = least(least(how(p.u_t * is), how(p.dt_t * is)), a->z ? how(p.z_t * is) : kVectors);
    p.vec_bc = least(how(p.b_t * is), how(p.c_t * is));
    p.tiles = (int32_t)host::ceil_div(a->seq, kTile);
    p.u = a->u, p.dt = a->dt, p.z = a->z, p.b = a->b, p.c = a->c;
    p.a = a->a, p.d = a->d, p.dt_bias = a->dt_bias, p.state_in = a->state_in, p.lengths = a->lengths;
    p.y = a->y, p.state_out = a->state_out, p.ckpt = a->checkpoints;
    return p;
}

// A kernel's dynamic shared memory above the default 48 KB has to be allowed once per device.
template <typename K>
int allow_smem(K *kernel, size_t bytes) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == cudaSuccess ? DC_OK : host::cuda_fail(e);
}

// f.template operator()<P>() for the P = lanes_of(state).
template <typename F>
int for_lanes(int64_t state, F &&f) {
    switch (lanes_of(state)) {
        case 1: return f.template operator()<1>();
        case 2: return f.template operator()<2>();
        case 4: return f.template operator()<4>();
        case 8: return f.template operator()<8>();
        default: return f.template operator()<16>();
    }
}

}  // namespace scan
}  // namespace dc
