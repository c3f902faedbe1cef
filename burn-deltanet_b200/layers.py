"""The operators around the token mixers of a block stack, over the C ABI of include/deltacore_layers.h.

* :func:`add_rms_norm`, :func:`add_rms_norm_f8`, :func:`add_rms_norm_backward` — the residual stream's addition and the RMS
  norm of the sum, in float32 / bfloat16 or in 8 bits (e4m3) with scales;
* :func:`causal_conv`, :func:`causal_conv_step`, :func:`causal_conv_backward` — the short causal depthwise convolution;
* :func:`selective_scan`, :func:`selective_scan_step`, :func:`selective_scan_backward` — the selective state space scan;
* :class:`AddRmsNormFunction`, :class:`CausalConvFunction`, :class:`SelectiveScanFunction` — their autograd nodes, once
  differentiable (a second derivative is an error).  The functions above are no nodes: their outputs carry no gradient.

They have no counterpart in burn-deltanet (the norm in front of a block is a Burn module there, and the selective scan is the
diagonal relative of the delta rule that hybrid stacks interleave with it).  The manner is :mod:`.core`'s: CUDA tensors only,
errors as :class:`~.core.DeltaCoreError` / :class:`~.core.DeltaShapeError`, work on the tensors' device and its current
stream, outputs as new tensors unless given.  Inputs may be column slices of a projection where the text says so: the last
axis contiguous, one stride per token.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _abi
from .core import DeltaCoreError, DeltaShapeError, _raise

# Counts a buffer of the caller's that a call wrote as changed, so that autograd refuses a backward which saved its old values.
_wrote = torch.autograd.graph.increment_version

_CODES = {torch.float32: _abi.DC_F32, torch.bfloat16: _abi.DC_BF16}


def _code(dtype: torch.dtype, what: str) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise DeltaCoreError(_abi.DC_EUNSUPPORTED_DTYPE, f"{what} has dtype {dtype}")
    return code


def _cuda(t: torch.Tensor, what: str, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if not t.is_cuda:
        raise DeltaCoreError(_abi.DC_EDEVICE, f"{what} is on {t.device}: the delta-rule core runs on CUDA only")
    if device is not None and t.device != device:
        raise DeltaCoreError(_abi.DC_EDEVICE, f"{what} is on {t.device}, the other tensors on {device}")


def _whole(t: Optional[torch.Tensor], what: str, shape, dtype: torch.dtype, device: torch.device) -> None:
    """Refuse what is not a contiguous tensor of this shape and dtype (or None)."""
    if t is None:
        return
    _cuda(t, what, device)
    if t.dtype != dtype:
        raise DeltaCoreError(_abi.DC_EUNSUPPORTED_DTYPE, f"{what} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"{what} has shape {tuple(t.shape)}, want {tuple(shape)}")
    if not t.is_contiguous():
        raise DeltaCoreError(_abi.DC_EINVAL_ARG, f"{what} must be contiguous")


def _row_stride(t: torch.Tensor, what: str) -> int:
    """The one stride between the rows (all axes but the last) of `t`."""
    width = t.shape[-1]
    if t.is_contiguous():
        return width
    if t.stride(-1) != 1 and width > 1:
        raise DeltaCoreError(_abi.DC_EINVAL_ARG, f"{what} must have a contiguous last axis")
    stride, span = width, None
    for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if span is None:
            stride = st
        elif st != span:
            raise DeltaCoreError(_abi.DC_EINVAL_ARG, f"{what} must have one stride between its rows")
        span = st * size
    return stride


def _strides(t: torch.Tensor, what: str, shape, dtype: torch.dtype, device: torch.device):
    """(sequence stride, token stride) of a [batch, seq, channels] tensor with contiguous channels."""
    _cuda(t, what, device)
    if t.dtype != dtype:
        raise DeltaCoreError(_abi.DC_EUNSUPPORTED_DTYPE, f"{what} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"{what} has shape {tuple(t.shape)}, want {shape}")
    if t.stride(2) != 1 and shape[2] > 1:
        raise DeltaCoreError(_abi.DC_EINVAL_ARG, f"{what} must have contiguous channels")
    return t.stride(0), t.stride(1)


# What a call's shapes, strides, dtypes and device decide (the checks, the C arguments without their addresses, the size of the
# workspace) is worked out once and kept by those: a decode tick would otherwise spend three times its kernel's time on it.
_PLANS: dict = {}
_MOST_PLANS = 1024


def _sig(t):
    if t is None:
        return None
    try:
        return t.shape, t.stride(), t.dtype, t.device
    except AttributeError:
        raise TypeError(f"a torch.Tensor is wanted, got {type(t).__name__}") from None


def _planned(build, *key):
    """build(), or what it returned for the same key before.  An error is not kept."""
    plan = _PLANS.get(key)
    if plan is None:
        plan = build()
        if len(_PLANS) >= _MOST_PLANS:
            _PLANS.clear()
        _PLANS[key] = plan
    return plan


def _on(device: torch.device, fn, *args):
    """fn(*args) with `device` current."""
    if torch.cuda.current_device() == device.index:
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


def _call(fn, args, device: torch.device, what: str) -> None:
    """Run a C entry point on `device`'s current stream."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)  # current_stream(device).cuda_stream without the object around it
    if torch._C._cuda_getDevice() == device.index:
        status = fn(args, stream)
    else:
        with torch.cuda.device(device):
            status = fn(args, stream)
    if status:
        _raise(status, what)


def _workspace(need: int, args, workspace: Optional[torch.Tensor], device: torch.device):
    """Point `args` at a workspace of `need` bytes, or the caller's; returns the tensor, to be kept until the launch."""
    if workspace is None:
        if need == 0:
            return None
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    else:
        _cuda(workspace, "workspace", device)
        if not workspace.is_contiguous():
            raise DeltaCoreError(_abi.DC_EINVAL_ARG, "workspace must be contiguous")
    args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return workspace


def _ptr(t):
    return None if t is None else t.data_ptr()


def _new(like: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A contiguous tensor of `like`'s shape (empty_like takes a third of empty's time, and a decode tick is short)."""
    if like.dtype == dtype and like.is_contiguous():
        return torch.empty_like(like)
    return torch.empty(like.shape, device=like.device, dtype=dtype)


class _Gradients(torch.autograd.Function):
    """`count` gradients as they are, depending on the tensors behind them; to differentiate them is an error."""

    @staticmethod
    def forward(ctx, count, *tensors):
        return tuple(t.detach() for t in tensors[:count])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("this operator can be differentiated once: its backward has no derivative")


def _once(backward):
    """A node's backward whose gradients refuse a second derivative, also where only a part of it would pass through them (torch's
    own once_differentiable leaves that part out where the derivative is asked for by torch.autograd.grad)."""

    @functools.wraps(backward)
    def once(ctx, *d_outputs):
        with torch.no_grad():
            grads = backward(ctx, *d_outputs)
        if not torch.is_grad_enabled():
            return grads
        behind = [t for t in (*d_outputs, *ctx.saved_tensors) if t is not None and t.requires_grad]
        given = [i for i, g in enumerate(grads) if g is not None]
        if not behind:
            return grads
        grads = list(grads)
        for i, g in zip(given, _Gradients.apply(len(given), *(grads[i] for i in given), *behind)):
            grads[i] = g
        return tuple(grads)

    return once


# ------------------------------------------------------------------------------------------------ residual add + norm
def _norm_plan(x, weight, residual, eps, out_dtype, residual_dtype, y_out, residual_out, group):
    """(C arguments without addresses, dtype of y, dtype of the sum or None where it is x itself); group: None, or of the e4m3 form."""
    _cuda(x, "x")
    if x.dim() < 1:
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, "x must have at least one axis")
    width, dev = x.shape[-1], x.device
    a = _abi.RmsNormArgs()
    a.rows, a.width = x.numel() // width if width else 0, width
    a.eps = eps
    _cuda(weight, "weight")
    _whole(weight, "weight", (width,), torch.float32, dev)
    a.x_dtype, a.x_stride = _code(x.dtype, "x"), _row_stride(x, "x")
    r_dtype = residual_dtype or (residual.dtype if residual is not None else residual_out.dtype if residual_out is not None else x.dtype)
    a.residual_dtype = _code(r_dtype, "residual")
    for t, what in ((residual, "residual"), (residual_out, "residual_out")):
        if t is not None:
            _cuda(t, what, dev)
            if t.shape != x.shape:
                raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"{what} has shape {tuple(t.shape)}, want {tuple(x.shape)}")
            if t.dtype != r_dtype:
                raise DeltaCoreError(_abi.DC_EUNSUPPORTED_DTYPE, f"{what} must be {r_dtype}, got {t.dtype}")
    if residual is not None:
        a.residual_in_stride = _row_stride(residual, "residual")
    a.residual_out_stride = width if residual_out is None else _row_stride(residual_out, "residual_out")
    if residual is None and residual_out is None and r_dtype == x.dtype:
        r_dtype = None
    if group is None:
        y_dtype = y_out.dtype if y_out is not None else out_dtype or x.dtype
        a.out_dtype, a.y_stride = _code(y_dtype, "y"), width
        if y_out is not None:
            _cuda(y_out, "y_out", dev)
            if y_out.shape != x.shape or (out_dtype is not None and y_out.dtype != out_dtype):
                raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, "y_out must be shaped like x, in out_dtype")
            a.y_stride = _row_stride(y_out, "y_out")
    else:
        if group not in (0, 32, 64, 128, 256):
            raise DeltaShapeError(_abi.DC_EINVAL_WIDTH, f"group must be 0, 32, 64, 128 or 256, got {group}")
        if group and width % group:
            raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"group {group} does not divide the width {width}")
        y_dtype = torch.float8_e4m3fn
        a.out_dtype, a.y_stride, a.group = _abi.DC_E4M3, width, group
    return a, y_dtype, r_dtype


def _norm(x, weight, residual, eps, out_dtype, residual_dtype, y_out, residual_out, group):
    """add_rms_norm's and add_rms_norm_f8's call: (y, scale, r)."""
    eps = float(eps)
    proto, y_dtype, r_dtype = _planned(
        lambda: _norm_plan(x, weight, residual, eps, out_dtype, residual_dtype, y_out, residual_out, group),
        "norm", _sig(x), _sig(weight), _sig(residual), eps, out_dtype, residual_dtype, _sig(y_out), _sig(residual_out), group)
    a = _abi.RmsNormArgs.from_buffer_copy(proto)
    dev = x.device
    y = _new(x, y_dtype) if y_out is None else y_out
    scale = None
    if group is not None:
        scale = torch.empty((*x.shape[:-1], x.shape[-1] // group if group else 1), device=dev, dtype=torch.float32)
        a.scale = scale.data_ptr()
    r = x
    if r_dtype is not None:
        r = _new(x if residual is None else residual, r_dtype) if residual_out is None else residual_out
        a.residual_out = r.data_ptr()
    a.x, a.weight, a.y = x.data_ptr(), weight.data_ptr(), y.data_ptr()
    if residual is not None:
        a.residual_in = residual.data_ptr()
    _call(_abi.lib().dc_rms_norm, a, dev, "dc_rms_norm")
    if y_out is not None:
        _wrote(y_out)
    if residual_out is not None:
        _wrote(residual_out)
    return y, scale, r


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-5, *,
                 out_dtype: Optional[torch.dtype] = None, residual_dtype: Optional[torch.dtype] = None,
                 y_out: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None):
    """The residual stream's addition and the RMS norm of the sum (``dc_rms_norm``) over the last axis of ``x``:
    ``s = x + residual``, ``y = s / sqrt(mean(s^2) + eps) * weight``.

    ``x`` and ``residual`` (the same shape; ``None``: zero) are float32 or bfloat16 each; their rows may be column slices with
    one stride.  ``weight`` is float32 ``[width]``.  Returns ``(y, r)``: ``y`` in ``out_dtype`` (default: ``x``'s), ``r`` the
    sum in ``residual_dtype`` (default: ``residual``'s), the next layer's ``residual``; without a residual ``r`` is ``x``.
    ``y`` is made from the sum before ``r``'s rounding.  ``residual_out`` may be ``residual`` and ``y_out`` may be ``x``.
    """
    y, _, r = _norm(x, weight, residual, eps, out_dtype, residual_dtype, y_out, residual_out, None)
    return y, r


def add_rms_norm_f8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-5, *,
                    group: int = 0, residual_dtype: Optional[torch.dtype] = None, residual_out: Optional[torch.Tensor] = None):
    """:func:`add_rms_norm` with ``y`` in 8 bits: returns ``(q, scale, r)``, ``y = q * scale`` with ``q`` float8_e4m3fn shaped
    like ``x`` and one float32 scale, ``max|y| / 448``, per ``group`` consecutive columns (32, 64, 128 or 256 dividing the
    width; 0: per row).  ``scale`` is ``x``'s shape with the last axis ``width / group`` (1 per row)."""
    return _norm(x, weight, residual, eps, None, residual_dtype, None, residual_out, int(group))


def _norm_bwd_plan(d_y, d_r, r, weight, eps, x_dtype):
    """(C arguments without addresses, dtype of d_x or None where d_residual is it, bytes of workspace)."""
    _cuda(r, "r")
    dev, width = r.device, r.shape[-1]
    _cuda(d_y, "d_y", dev)
    if d_y.shape != r.shape or (d_r is not None and d_r.shape != r.shape):
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, "d_y and d_r must be shaped like r")
    a = _abi.RmsNormBwdArgs()
    a.rows, a.width, a.eps = r.numel() // width if width else 0, width, eps
    _cuda(weight, "weight")
    _whole(weight, "weight", (width,), torch.float32, dev)
    a.r_dtype, a.r_stride = _code(r.dtype, "r"), _row_stride(r, "r")
    a.y_dtype, a.d_y_stride = _code(d_y.dtype, "d_y"), _row_stride(d_y, "d_y")
    if d_r is not None:
        _cuda(d_r, "d_r", dev)
        if d_r.dtype != r.dtype:
            raise DeltaCoreError(_abi.DC_EUNSUPPORTED_DTYPE, f"d_r must be {r.dtype}, got {d_r.dtype}")
        a.d_r_stride = _row_stride(d_r, "d_r")
    a.d_residual_stride = width
    other = x_dtype is not None and x_dtype != r.dtype
    if other:
        a.d_x_stride, a.x_dtype = width, _code(x_dtype, "x_dtype")
    a.d_weight = 16  # stands for the buffer in the query
    need = int(_on(dev, _abi.lib().dc_rms_norm_bwd_workspace_size, a))
    return a, x_dtype if other else None, need


def add_rms_norm_backward(d_y: torch.Tensor, d_r: Optional[torch.Tensor], r: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *,
                          x_dtype: Optional[torch.dtype] = None, workspace: Optional[torch.Tensor] = None):
    """The backward of :func:`add_rms_norm` (``dc_rms_norm_bwd``) from its ``r``: returns ``(d_x, d_residual, d_weight)``,
    ``d_x`` in ``x_dtype`` (default: ``r``'s), ``d_residual`` in ``r``'s dtype (the same tensor where the dtypes are equal: the
    two gradients are), ``d_weight`` float32.  ``d_r`` is the gradient of the returned sum, in ``r``'s dtype (``None``: zero)."""
    eps = float(eps)
    proto, other, need = _planned(lambda: _norm_bwd_plan(d_y, d_r, r, weight, eps, x_dtype),
                                  "norm_bwd", _sig(d_y), _sig(d_r), _sig(r), _sig(weight), eps, x_dtype)
    a = _abi.RmsNormBwdArgs.from_buffer_copy(proto)
    dev = r.device
    d_x = d_residual = _new(r, r.dtype)
    if other is not None:
        d_x = _new(d_y, other)
        a.d_x = d_x.data_ptr()
    d_weight = _new(weight, torch.float32)
    a.d_y, a.d_r, a.r, a.weight = d_y.data_ptr(), _ptr(d_r), r.data_ptr(), weight.data_ptr()
    a.d_residual, a.d_weight = d_residual.data_ptr(), d_weight.data_ptr()
    keep = _workspace(need, a, workspace, dev)
    _call(_abi.lib().dc_rms_norm_bwd, a, dev, "dc_rms_norm_bwd")
    del keep
    return d_x, d_residual, d_weight


class AddRmsNormFunction(torch.autograd.Function):
    """``y, r = AddRmsNormFunction.apply(x, weight, residual, eps)`` (only ``y`` without a residual): :func:`add_rms_norm` as an
    autograd node.  It keeps the sum and the weight."""

    @staticmethod
    def forward(ctx, x, weight, residual=None, eps=1e-5):
        y, r = add_rms_norm(x, weight, residual, eps)
        ctx.save_for_backward(r, weight)
        ctx.cfg = (eps, x.dtype, residual is not None)
        return y if residual is None else (y, r)

    @staticmethod
    @_once
    def backward(ctx, d_y, d_r=None):
        r, weight = ctx.saved_tensors
        eps, x_dtype, has_residual = ctx.cfg
        d_x, d_residual, d_weight = add_rms_norm_backward(d_y.contiguous(), None if d_r is None else d_r.contiguous(), r, weight, eps,
                                                          x_dtype=x_dtype)
        return d_x, d_weight, d_residual if has_residual else None, None


# ------------------------------------------------------------------------------------------------ causal convolution
def _conv_dims(a, x, weight, bias, window, silu, lengths):
    """The forward's and the backward's common checks and fields, for x [batch, seq, channels]."""
    _cuda(x, "x")
    if x.dim() != 3:
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"x must be [batch, seq, channels], got {tuple(x.shape)}")
    b, s, c = x.shape
    dev = x.device
    if weight is None or weight.dim() != 2:
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"weight must be [{c}, taps]")
    k = weight.shape[1]
    a.batch, a.seq, a.channels, a.taps = b, s, c, k
    a.in_dtype = _code(x.dtype, "x")
    a.flags = _abi.DC_CONV_SILU if silu else 0
    a.x_batch_stride, a.x_token_stride = _strides(x, "x", (b, s, c), x.dtype, dev)
    _whole(weight, "weight", (c, k), torch.float32, dev)
    _whole(bias, "bias", (c,), torch.float32, dev)
    _whole(window, "window", (b, c, k), torch.float32, dev)
    _whole(lengths, "lengths", (b,), torch.int32, dev)


def _conv_plan(x, weight, bias, window, silu, lengths, out_dtype, y_out, window_out, step):
    """(C arguments without addresses, dtype of y)."""
    if step:
        if x is None or x.dim() != 2:
            raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, "x must be [batch, channels]")
        x, y_out = x.unsqueeze(1), None if y_out is None else y_out.unsqueeze(1)
    a = _abi.CausalConvArgs()
    _conv_dims(a, x, weight, bias, window, silu, lengths)
    b, s, c = x.shape
    dtype = y_out.dtype if y_out is not None else out_dtype or x.dtype
    if out_dtype is not None and dtype != out_dtype:
        raise DeltaCoreError(_abi.DC_EUNSUPPORTED_DTYPE, f"y_out must be {out_dtype}")
    a.y_batch_stride, a.y_token_stride = (s * c, c) if y_out is None else _strides(y_out, "y_out", (b, s, c), dtype, x.device)
    a.out_dtype = _code(dtype, "y")
    _whole(window_out, "window_out", (b, c, weight.shape[1]), torch.float32, x.device)
    return a, dtype


def _conv(x, weight, bias, window, silu, lengths, out_dtype, y_out, window_out, step):
    """causal_conv's and causal_conv_step's call."""
    proto, dtype = _planned(lambda: _conv_plan(x, weight, bias, window, silu, lengths, out_dtype, y_out, window_out, step),
                            "conv", step, _sig(x), _sig(weight), _sig(bias), _sig(window), bool(silu), _sig(lengths), out_dtype,
                            _sig(y_out), _sig(window_out))
    a = _abi.CausalConvArgs.from_buffer_copy(proto)
    dev = x.device
    y = _new(x, dtype) if y_out is None else y_out
    nxt = window_out
    if nxt is None:
        nxt = torch.empty((a.batch, a.channels, a.taps), device=dev, dtype=torch.float32) if window is None else _new(window, torch.float32)
    a.x, a.weight, a.y, a.window_out = x.data_ptr(), weight.data_ptr(), y.data_ptr(), nxt.data_ptr()
    if bias is not None:
        a.bias = bias.data_ptr()
    if window is not None:
        a.window_in = window.data_ptr()
    if lengths is not None:
        a.lengths = lengths.data_ptr()
    _call(_abi.lib().dc_causal_conv, a, dev, "dc_causal_conv")
    if y_out is not None:
        _wrote(y_out)
    if window_out is not None:
        _wrote(window_out)
    return y, nxt


def causal_conv(x_bsc: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, window: Optional[torch.Tensor] = None, *,
                silu: bool = True, lengths: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                y_out: Optional[torch.Tensor] = None, window_out: Optional[torch.Tensor] = None):
    """The causal depthwise convolution of ``x [batch, seq, channels]`` (``dc_causal_conv``) with ``weight [channels, taps]``
    (up to 8 taps) and ``bias``, then SiLU (``silu``): ``y_t = silu(bias + sum_j weight[:, j] x_{t - taps + 1 + j})``.

    ``window [batch, channels, taps]`` (float32, ``None``: zeros) holds the tokens before the first in its last ``taps - 1``
    columns, as :func:`~.core.qkv_prologue`'s does.  ``lengths`` (int32 ``[batch]``) ends each sequence early: the padding is
    not read and its ``y`` is zero.  ``x`` may be a column slice.  Returns ``(y, next window)``.
    """
    return _conv(x_bsc, weight, bias, window, silu, lengths, out_dtype, y_out, window_out, False)


def causal_conv_step(x_bc: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, window: Optional[torch.Tensor] = None, *,
                     silu: bool = True, out_dtype: Optional[torch.dtype] = None, y_out: Optional[torch.Tensor] = None,
                     window_out: Optional[torch.Tensor] = None):
    """:func:`causal_conv` for one token per sequence: ``x [batch, channels]`` to ``(y [batch, channels], next window)``; pass
    ``window_out=window`` to roll the window in place."""
    return _conv(x_bc, weight, bias, window, silu, None, out_dtype, y_out, window_out, True)


def _conv_bwd_plan(d_y, d_window_out, x, weight, bias, window, silu, lengths):
    """(C arguments without addresses, bytes of workspace)."""
    a = _abi.CausalConvBwdArgs()
    _conv_dims(a, x, weight, bias, window, silu, lengths)
    b, s, c = x.shape
    _cuda(d_y, "d_y", x.device)
    a.out_dtype = _code(d_y.dtype, "d_y")
    a.d_y_batch_stride, a.d_y_token_stride = _strides(d_y, "d_y", (b, s, c), d_y.dtype, x.device)
    _whole(d_window_out, "d_window_out", (b, c, weight.shape[1]), torch.float32, x.device)
    a.d_x_batch_stride, a.d_x_token_stride = s * c, c
    return a, int(_on(x.device, _abi.lib().dc_causal_conv_bwd_workspace_size, a))


def causal_conv_backward(d_y: torch.Tensor, d_window_out: Optional[torch.Tensor], x_bsc: torch.Tensor, weight: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, window: Optional[torch.Tensor] = None, *, silu: bool = True,
                         lengths: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """The backward of :func:`causal_conv` (``dc_causal_conv_bwd``), given ``d_y`` and the gradient of the returned window
    (``None``: zero): returns ``(d_x, d_weight, d_bias, d_window)``, ``d_x`` in ``x``'s dtype, the others float32; ``d_bias`` and
    ``d_window`` are ``None`` where ``bias`` and ``window`` are."""
    proto, need = _planned(lambda: _conv_bwd_plan(d_y, d_window_out, x_bsc, weight, bias, window, silu, lengths),
                           "conv_bwd", _sig(d_y), _sig(d_window_out), _sig(x_bsc), _sig(weight), _sig(bias), _sig(window), bool(silu),
                           _sig(lengths))
    a = _abi.CausalConvBwdArgs.from_buffer_copy(proto)
    dev = x_bsc.device
    d_x, d_weight = _new(x_bsc, x_bsc.dtype), _new(weight, torch.float32)
    d_bias = None if bias is None else _new(bias, torch.float32)
    d_window = None if window is None else _new(window, torch.float32)
    a.d_y, a.d_window_out, a.x, a.weight, a.bias = d_y.data_ptr(), _ptr(d_window_out), x_bsc.data_ptr(), weight.data_ptr(), _ptr(bias)
    a.window_in, a.lengths = _ptr(window), _ptr(lengths)
    a.d_x, a.d_weight, a.d_bias, a.d_window_in = d_x.data_ptr(), d_weight.data_ptr(), _ptr(d_bias), _ptr(d_window)
    keep = _workspace(need, a, workspace, dev)
    _call(_abi.lib().dc_causal_conv_bwd, a, dev, "dc_causal_conv_bwd")
    del keep
    return d_x, d_weight, d_bias, d_window


class CausalConvFunction(torch.autograd.Function):
    """``y, next_window = CausalConvFunction.apply(x, weight, bias, window, silu, lengths)``: :func:`causal_conv` as an autograd
    node that keeps its inputs and recomputes the convolution in the backward."""

    @staticmethod
    def forward(ctx, x, weight, bias=None, window=None, silu=True, lengths=None):
        y, nxt = causal_conv(x, weight, bias, window, silu=silu, lengths=lengths)
        ctx.save_for_backward(x, weight, bias, window, lengths)
        ctx.silu = silu
        return y, nxt

    @staticmethod
    @_once
    def backward(ctx, d_y, d_next):
        x, weight, bias, window, lengths = ctx.saved_tensors
        d_x, d_weight, d_bias, d_window = causal_conv_backward(d_y.contiguous(), d_next.contiguous(), x, weight, bias, window,
                                                               silu=ctx.silu, lengths=lengths)
        return d_x, d_weight, d_bias, d_window, None, None


# ------------------------------------------------------------------------------------------------ selective scan
def _bc(t, what, b, s, dtype, dev):
    """(groups, state, sequence stride, token stride) of b or c: [batch, seq, groups, state] or [batch, seq, state]."""
    _cuda(t, what, dev)
    if t.dtype != dtype:
        raise DeltaCoreError(_abi.DC_EUNSUPPORTED_DTYPE, f"{what} must be {dtype}, got {t.dtype}")
    if t.dim() not in (3, 4) or t.shape[0] != b or t.shape[1] != s:
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"{what} has shape {tuple(t.shape)}, want [{b}, {s}, groups, state]")
    g, n = (1, t.shape[2]) if t.dim() == 3 else t.shape[2:]
    if (n > 1 and t.stride(-1) != 1) or (t.dim() == 4 and g > 1 and t.stride(2) != n):
        raise DeltaCoreError(_abi.DC_EINVAL_ARG, f"{what} must have contiguous [groups, state]")
    return g, n, t.stride(0), t.stride(1)


def _scan_dims(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths):
    """dc_selective_scan_args without addresses and outputs, for u [batch, seq, channels]."""
    _cuda(u, "u")
    if u.dim() != 3:
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"u must be [batch, seq, channels], got {tuple(u.shape)}")
    bs, s, ch = u.shape
    dev, dtype = u.device, u.dtype
    g = _abi.SelectiveScanArgs()
    g.in_dtype = _code(dtype, "u")
    groups, n, g.b_batch_stride, g.b_token_stride = _bc(b, "b", bs, s, dtype, dev)
    groups_c, n_c, g.c_batch_stride, g.c_token_stride = _bc(c, "c", bs, s, dtype, dev)
    if (groups_c, n_c) != (groups, n):
        raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, f"c has [groups, state] {(groups_c, n_c)}, b {(groups, n)}")
    g.batch, g.seq, g.channels, g.state, g.groups = bs, s, ch, n, groups
    g.u_batch_stride, g.u_token_stride = _strides(u, "u", (bs, s, ch), dtype, dev)
    g.dt_batch_stride, g.dt_token_stride = _strides(dt, "dt", (bs, s, ch), dtype, dev)
    if z is not None:
        g.z_batch_stride, g.z_token_stride = _strides(z, "z", (bs, s, ch), dtype, dev)
    g.flags = _abi.DC_SCAN_SOFTPLUS if softplus else 0
    _cuda(a, "a")
    _whole(a, "a", (ch, n), torch.float32, dev)
    _whole(d, "d", (ch,), torch.float32, dev)
    _whole(dt_bias, "dt_bias", (ch,), torch.float32, dev)
    _whole(state, "state", (bs, ch, n), torch.float32, dev)
    _whole(lengths, "lengths", (bs,), torch.int32, dev)
    return g


def _scan_plan(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, out_dtype, y_out, state_out, step):
    """(C arguments without addresses, dtype of y, bytes of checkpoints, bytes of workspace)."""
    if step:
        if u is None or u.dim() != 2:
            raise DeltaShapeError(_abi.DC_EINVAL_SHAPE, "u must be [batch, channels]")
        one = lambda t: None if t is None else t.unsqueeze(1)
        u, dt, b, c, z, y_out = one(u), one(dt), one(b), one(c), one(z), one(y_out)
    g = _scan_dims(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths)
    dev, shape = u.device, (g.batch, g.seq, g.channels)
    dtype = y_out.dtype if y_out is not None else out_dtype or u.dtype
    if out_dtype is not None and dtype != out_dtype:
        raise DeltaCoreError(_abi.DC_EUNSUPPORTED_DTYPE, f"y_out must be {out_dtype}")
    strides = (g.seq * g.channels, g.channels) if y_out is None else _strides(y_out, "y_out", shape, dtype, dev)
    g.y_batch_stride, g.y_token_stride = strides
    g.out_dtype = _code(dtype, "y")
    _whole(state_out, "state_out", (g.batch, g.channels, g.state), torch.float32, dev)
    L = _abi.lib()
    return g, dtype, int(L.dc_selective_scan_checkpoint_size(g)), 0 if step else int(_on(dev, L.dc_selective_scan_workspace_size, g))


def _scan(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, out_dtype, y_out, state_out, step, checkpoints, workspace):
    """selective_scan's and selective_scan_step's call: (y, final state, checkpoints or None)."""
    proto, dtype, saves, need = _planned(
        lambda: _scan_plan(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, out_dtype, y_out, state_out, step),
        "scan", step, _sig(u), _sig(dt), _sig(a), _sig(b), _sig(c), _sig(d), _sig(z), _sig(dt_bias), _sig(state), bool(softplus),
        _sig(lengths), out_dtype, _sig(y_out), _sig(state_out))
    g = _abi.SelectiveScanArgs.from_buffer_copy(proto)
    dev = u.device
    y = _new(u, dtype) if y_out is None else y_out
    h = state_out
    if h is None:
        h = torch.empty((g.batch, g.channels, g.state), device=dev, dtype=torch.float32) if state is None else _new(state, torch.float32)
    _scan_inputs(g, u, dt, a, b, c, d, z, dt_bias, state, lengths)
    g.y, g.state_out = y.data_ptr(), h.data_ptr()
    saved = keep = None
    if checkpoints:
        saved = torch.empty(saves // 4, device=dev, dtype=torch.float32)
        g.checkpoints = saved.data_ptr()
    if step:
        _call(_abi.lib().dc_selective_scan_step, g, dev, "dc_selective_scan_step")
    else:
        keep = _workspace(need, g, workspace, dev)
        _call(_abi.lib().dc_selective_scan, g, dev, "dc_selective_scan")
    if y_out is not None:
        _wrote(y_out)
    if state_out is not None:
        _wrote(state_out)
    del keep
    return y, h, saved


def _scan_inputs(g, u, dt, a, b, c, d, z, dt_bias, state, lengths):
    g.u, g.dt, g.a, g.b, g.c = u.data_ptr(), dt.data_ptr(), a.data_ptr(), b.data_ptr(), c.data_ptr()
    if d is not None:
        g.d = d.data_ptr()
    if z is not None:
        g.z = z.data_ptr()
    if dt_bias is not None:
        g.dt_bias = dt_bias.data_ptr()
    if state is not None:
        g.state_in = state.data_ptr()
    if lengths is not None:
        g.lengths = lengths.data_ptr()


def selective_scan(u: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, d: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None, *,
                   softplus: bool = True, lengths: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                   checkpoints: bool = False, y_out: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None):
    """The selective state space scan over a prompt (``dc_selective_scan``).  Per sequence and channel, with a state ``h`` of
    ``state`` values::

        step = softplus(dt + dt_bias)
        h    = exp(step * a) * h + step * u * b
        y    = (c . h + d * u) * silu(z)

    ``u``, ``dt`` and ``z`` are ``[batch, seq, channels]``, ``b`` and ``c`` ``[batch, seq, groups, state]`` (or ``[batch, seq,
    state]``; channel ``i`` reads group ``i // (channels / groups)``), all of one dtype, float32 or bfloat16, and any of them may
    be a column slice.  ``a [channels, state]``, ``d``, ``dt_bias [channels]`` and ``state [batch, channels, state]`` are float32;
    ``d``, ``z``, ``dt_bias`` and ``state`` may be ``None``.  ``lengths`` (int32 ``[batch]``) ends each sequence early.  Returns
    ``(y, final state)``, with ``checkpoints=True`` also what :func:`selective_scan_backward` starts from.  ``state_out`` may be
    ``state``; ``softplus=False`` takes ``dt + dt_bias`` as it is.
    """
    y, h, saved = _scan(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, out_dtype, y_out, state_out, False, checkpoints, workspace)
    return (y, h, saved) if checkpoints else (y, h)


def selective_scan_step(u: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, d: Optional[torch.Tensor] = None,
                        z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None, *,
                        softplus: bool = True, out_dtype: Optional[torch.dtype] = None, y_out: Optional[torch.Tensor] = None,
                        state_out: Optional[torch.Tensor] = None):
    """:func:`selective_scan` for one token per sequence (``dc_selective_scan_step``): ``u``, ``dt``, ``z [batch, channels]``, ``b``,
    ``c [batch, groups, state]`` or ``[batch, state]``; returns ``(y [batch, channels], next state)``.  Pass ``state_out=state`` to
    update the state in place."""
    y, h, _ = _scan(u, dt, a, b, c, d, z, dt_bias, state, softplus, None, out_dtype, y_out, state_out, True, False, None)
    return y, h


def _scan_bwd_plan(d_y, d_state, u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, checkpoints):
    """(C arguments without addresses, bytes of workspace)."""
    g = _scan_dims(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths)
    dev, shape = u.device, (g.batch, g.seq, g.channels)
    L = _abi.lib()
    _whole(checkpoints, "checkpoints", (int(L.dc_selective_scan_checkpoint_size(g)) // 4,), torch.float32, dev)
    _cuda(d_y, "d_y", dev)
    g.out_dtype = _code(d_y.dtype, "d_y")
    w = _abi.SelectiveScanBwdArgs()
    w.d_y_batch_stride, w.d_y_token_stride = _strides(d_y, "d_y", shape, d_y.dtype, dev)
    _whole(d_state, "d_state", (g.batch, g.channels, g.state), torch.float32, dev)
    w.fwd = g
    return w, int(_on(dev, L.dc_selective_scan_bwd_workspace_size, w))


def selective_scan_backward(d_y: torch.Tensor, d_state: Optional[torch.Tensor], u: torch.Tensor, dt: torch.Tensor, a: torch.Tensor,
                            b: torch.Tensor, c: torch.Tensor, d: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                            dt_bias: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None, *, softplus: bool = True,
                            lengths: Optional[torch.Tensor] = None, checkpoints: Optional[torch.Tensor] = None,
                            workspace: Optional[torch.Tensor] = None):
    """The backward of :func:`selective_scan` (``dc_selective_scan_bwd``), given ``d_y`` and the gradient of the final state
    (``None``: zero), on the forward's inputs and its ``checkpoints`` (``None``: the forward is run again for them).  Returns
    ``(d_u, d_dt, d_a, d_b, d_c, d_d, d_z, d_dt_bias, d_state)``: those of ``u``, ``dt``, ``b``, ``c``, ``z`` in their dtype, the others
    float32, ``None`` where the input is."""
    if checkpoints is None:
        checkpoints = selective_scan(u, dt, a, b, c, d, z, dt_bias, state, softplus=softplus, lengths=lengths, checkpoints=True)[2]
    proto, need = _planned(
        lambda: _scan_bwd_plan(d_y, d_state, u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, checkpoints),
        "scan_bwd", _sig(d_y), _sig(d_state), _sig(u), _sig(dt), _sig(a), _sig(b), _sig(c), _sig(d), _sig(z), _sig(dt_bias), _sig(state),
        bool(softplus), _sig(lengths), _sig(checkpoints))
    w = _abi.SelectiveScanBwdArgs.from_buffer_copy(proto)
    _scan_inputs(w.fwd, u, dt, a, b, c, d, z, dt_bias, state, lengths)
    w.fwd.checkpoints = checkpoints.data_ptr()
    dev, dtype = u.device, u.dtype
    like = lambda t, dtype=torch.float32: None if t is None else _new(t, dtype)
    d_u, d_dt, d_z, d_b, d_c = like(u, dtype), like(dt, dtype), like(z, dtype), like(b, dtype), like(c, dtype)
    d_a, d_d, d_dt_bias, d_state_in = like(a), like(d), like(dt_bias), like(state)
    w.d_y, w.d_state_out = d_y.data_ptr(), _ptr(d_state)
    w.d_u, w.d_dt, w.d_a, w.d_b, w.d_c, w.d_d = d_u.data_ptr(), d_dt.data_ptr(), d_a.data_ptr(), d_b.data_ptr(), d_c.data_ptr(), _ptr(d_d)
    w.d_z, w.d_dt_bias, w.d_state_in = _ptr(d_z), _ptr(d_dt_bias), _ptr(d_state_in)
    keep = _workspace(need, w, workspace, dev)
    _call(_abi.lib().dc_selective_scan_bwd, w, dev, "dc_selective_scan_bwd")
    del keep
    return d_u, d_dt, d_a, d_b, d_c, d_d, d_z, d_dt_bias, d_state_in


class SelectiveScanFunction(torch.autograd.Function):
    """``y, final_state = SelectiveScanFunction.apply(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths)``:
    :func:`selective_scan` as an autograd node.  It keeps its inputs and the checkpoints (the state at the first token of every
    tile), and the backward recomputes the states between them."""

    @staticmethod
    def forward(ctx, u, dt, a, b, c, d=None, z=None, dt_bias=None, state=None, softplus=True, lengths=None):
        y, h, saved = selective_scan(u, dt, a, b, c, d, z, dt_bias, state, softplus=softplus, lengths=lengths, checkpoints=True)
        ctx.save_for_backward(u, dt, a, b, c, d, z, dt_bias, state, lengths, saved)
        ctx.softplus = softplus
        return y, h

    @staticmethod
    @_once
    def backward(ctx, d_y, d_h):
        *args, lengths, saved = ctx.saved_tensors
        grads = selective_scan_backward(d_y.contiguous(), d_h.contiguous(), *args, softplus=ctx.softplus, lengths=lengths, checkpoints=saved)
        return (*grads, None, None)
