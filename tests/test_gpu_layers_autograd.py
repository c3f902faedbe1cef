"""What autograd knows of the block-level operators on the GPU: buffers that a call writes count as changed, so that a backward
which still needs their old values is refused, and a second derivative is refused, not left out."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
dn = importlib.import_module("burn-deltanet_b200")


def rand(*shape, grad=False, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).requires_grad_(grad)


def scan_args(b=2, s=6, c=8, n=4):
    return [rand(b, s, c, seed=1, grad=True), rand(b, s, c, seed=2), -rand(c, n, seed=3).abs(), rand(b, s, 1, n, seed=4), rand(b, s, 1, n, seed=5),
            rand(c, seed=6), rand(b, s, c, seed=7), rand(c, seed=8), rand(b, c, n, seed=9)]


def one(args):
    return [t[:, 0].detach() if i in (0, 1, 3, 4, 6) else t for i, t in enumerate(args)]


def changed(t, call):
    before = t._version
    call()
    assert t._version > before


def test_buffers_that_a_call_writes_count_as_changed():
    x, w, buffer = rand(4, 64), rand(64, seed=1), rand(4, 64, seed=2)
    changed(buffer, lambda: dn.add_rms_norm(x, w, buffer, residual_out=buffer))
    changed(buffer, lambda: dn.add_rms_norm(x, w, y_out=buffer))
    changed(buffer, lambda: dn.add_rms_norm_f8(x, w, buffer, residual_out=buffer))
    x, cw, window = rand(2, 6, 8), rand(8, 4, seed=1), rand(2, 8, 4, seed=2)
    out = torch.empty_like(x)
    changed(out, lambda: dn.causal_conv(x, cw, y_out=out))
    changed(window, lambda: dn.causal_conv(x, cw, window_out=window))
    changed(window, lambda: dn.causal_conv_step(x[:, 0], cw, None, window, window_out=window))
    args = [t.detach() for t in scan_args()]
    out, state = torch.empty_like(args[0]), args[-1]
    changed(out, lambda: dn.selective_scan(*args, y_out=out))
    changed(state, lambda: dn.selective_scan(*args, state_out=state))
    changed(state, lambda: dn.selective_scan_step(*one(args), state_out=state))
    row = out[:, 0].contiguous()
    changed(row, lambda: dn.selective_scan_step(*one(args), y_out=row))
    versions = [t._version for t in (x, cw, *args)]
    dn.causal_conv(x, cw)
    dn.selective_scan(*args)
    assert versions == [t._version for t in (x, cw, *args)]  # inputs do not


def test_a_backward_that_needs_an_overwritten_buffer_is_refused():
    args = scan_args()
    y, _ = dn.SelectiveScanFunction.apply(*args)
    dn.selective_scan_step(*one(args), state_out=args[-1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    x, w, window = rand(2, 6, 8, grad=True), rand(8, 4, seed=1), rand(2, 8, 4, seed=2)
    y, _ = dn.CausalConvFunction.apply(x, w, None, window)
    dn.causal_conv_step(x[:, 0].detach(), w, None, window, window_out=window)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    x, w, res = rand(4, 64, grad=True), rand(64, seed=1), rand(4, 64, seed=2)
    y, r = dn.AddRmsNormFunction.apply(x, w, res)
    dn.add_rms_norm(x.detach(), w, r.detach(), residual_out=r.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_in_inference_mode():
    """Tensors without a version are written all the same."""
    with torch.inference_mode():
        args = [t.detach() * 1 for t in scan_args()]
        want = dn.selective_scan_step(*one(args))
        got = dn.selective_scan_step(*one(args), state_out=args[-1])
        assert torch.equal(got[0], want[0]) and torch.equal(args[-1], want[1])
    dn.selective_scan_step(*one([t.clone() for t in args[:-1]]), args[-1], state_out=args[-1])


def test_a_second_derivative_is_refused():
    """By backward and by torch.autograd.grad, also where another part of it exists; the first derivative is there."""
    x, w, res = rand(4, 64, grad=True), rand(64, seed=1, grad=True), rand(4, 64, seed=2, grad=True)
    cx, cw = rand(2, 6, 8, grad=True), rand(8, 4, seed=1, grad=True)
    for apply, arg in ((lambda: dn.AddRmsNormFunction.apply(x, w, res)[0], x), (lambda: dn.AddRmsNormFunction.apply(x, w), x),
                       (lambda: dn.AddRmsNormFunction.apply(x, w, res)[1] + dn.AddRmsNormFunction.apply(x, w), w),
                       (lambda: dn.CausalConvFunction.apply(cx, cw)[0], cx), (lambda: dn.CausalConvFunction.apply(cx, cw)[1], cw),
                       (lambda: dn.SelectiveScanFunction.apply(*([cx] + [t.detach() for t in scan_args()[1:]]))[0], cx)):
        for head in (lambda y: y.square().sum(), lambda y: y.sum()):
            plain, = torch.autograd.grad(head(apply()), arg)
            grad, = torch.autograd.grad(head(apply()), arg, create_graph=True)
            assert torch.equal(grad.detach(), plain)
            with pytest.raises(RuntimeError, match="differentiated once"):
                torch.autograd.grad((grad * arg).sum(), arg)
            grad, = torch.autograd.grad(head(apply()), arg, create_graph=True)
            with pytest.raises(RuntimeError, match="differentiated once"):
                (grad.square().sum() + arg.sum()).backward()
        x.grad = w.grad = res.grad = cx.grad = cw.grad = None
