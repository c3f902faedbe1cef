"""The residual add + RMS norm (dc_rms_norm, dc_rms_norm_bwd) on the GPU against the float64 oracle.

Tolerances, per element: the kernel's y is a product of the float32 sum s (half an ulp), the inverse root (the mean of
`width` squares: each thread adds 8 to 32 of them in order and ten shuffles follow, at most 42 roundings of 2^-24, halved by
the root) and the weight (two roundings): under 30 * 2^-24 = 1.8e-6 of |y|, taken as 4e-6.  A bfloat16 value adds half its
ulp.  An e4m3 value is off by at most half its step: 2^-4 of it, or 2^-10 of the scale below the normal range.
The backward's mean(w dy r) sums with both signs, so its share is measured against the same sum of magnitudes."""
import importlib

import numpy as np
import pytest
import torch

from oracle import layers as ol

pytestmark = pytest.mark.gpu
dn = importlib.import_module("burn-deltanet_b200")
BF, F32 = torch.bfloat16, torch.float32
REL = 4e-6


def half_ulp(ref, dtype):
    """Half the distance between the bfloat16 values around ref (float32's is in the other terms)."""
    return np.exp2(np.floor(np.log2(np.maximum(np.abs(ref), 1e-38))) - 8) if dtype == BF else 0.0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def f64(t):
    return None if t is None else t.double().cpu().numpy()


def close(got, ref, dtype, size=None):
    err = np.abs(f64(got) - ref)
    off = REL * np.abs(ref) + (REL * size if size is not None else 0)
    bound = off + half_ulp(np.abs(ref) + off, dtype) + 1e-37
    assert (err <= bound).all(), float((err / bound).max())


WIDTHS = [1, 7, 8, 40, 100, 128, 520, 1000, 2048, 4104, 8192, 16384]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("types", [(BF, BF, BF), (BF, F32, BF), (F32, F32, F32), (F32, BF, BF), (BF, None, F32)])
@pytest.mark.parametrize("rows", [1, 3, 700])
def test_forward(width, types, rows):
    xd, rd, od = types
    g = gen(width + rows)
    x, w = rand(g, rows, width, dtype=xd), rand(g, width) + 1
    res = None if rd is None else rand(g, rows, width, dtype=rd, scale=3)
    y, r = dn.add_rms_norm(x, w, res, 1e-5, out_dtype=od)
    assert y.dtype == od and r.dtype == (rd or xd)
    ry, rr = ol.rms_norm(f64(x), f64(res), f64(w), 1e-5)
    close(y, ry, od)
    close(r, rr, r.dtype)
    if res is None:
        assert r.data_ptr() == x.data_ptr()


@pytest.mark.parametrize("width,group", [(32, 32), (96, 32), (128, 64), (2048, 128), (4096, 256), (1280, 256), (13, 0), (8, 0), (2048, 0), (5001, 0), (16384, 128)])
@pytest.mark.parametrize("rows", [1, 5, 600])
@pytest.mark.parametrize("xd", [BF, F32])
def test_f8(width, group, rows, xd):
    g = gen(width)
    x, res, w = rand(g, rows, width, dtype=xd), rand(g, rows, width), rand(g, width)
    if width >= 2 * group > 0:
        w[:group] = 0  # a group of zeros
    q, scale, r = dn.add_rms_norm_f8(x, w, res, 1e-5, group=group)
    ry, rr = ol.rms_norm(f64(x), f64(res), f64(w), 1e-5)
    parts = ry.reshape(rows, -1, group or width)
    amax = np.abs(parts).max(-1)
    want = np.where(amax > 0, amax / 448, 1)
    assert scale.shape == want.shape
    assert (np.abs(f64(scale) - want) <= 2 * REL * want).all()
    s = np.repeat(f64(scale), group or width, axis=1)
    got = f64(q)
    step = np.maximum(np.abs(ry / s) * 2.0 ** -4, 2.0 ** -10)
    assert (np.abs(got - ry / s) <= step * (1 + 1e-4) + 4 * REL * np.abs(ry / s)).all()
    # and it is the nearest value wherever the float32 quotient is not near a tie
    near = ol.to_e4m3(ry / s)
    assert (got != near).mean() < 1e-3
    close(r, rr, F32)


def test_rows_of_slices_and_in_place():
    """Column slices of a wider buffer with odd and aligned offsets; the sum into the residual, y into x."""
    g = gen(1)
    for width, off in ((64, 8), (64, 3), (37, 5)):
        base, rbase = rand(g, 4, 9, 2 * width + 8, dtype=BF), rand(g, 4, 9, 3 * width + 16)
        x, res = base[..., off:off + width], rbase[..., 2 * off:2 * off + width]
        w = rand(g, width)
        ry, rr = ol.rms_norm(f64(x), f64(res), f64(w), 1e-6)
        outside = base.clone(), rbase.clone()
        y, r = dn.add_rms_norm(x, w, res, 1e-6, y_out=x, residual_out=res)
        assert y.data_ptr() == x.data_ptr() and r.data_ptr() == res.data_ptr()
        close(y, ry, BF)
        close(r, rr, F32)
        outside[0][..., off:off + width], outside[1][..., 2 * off:2 * off + width] = x, res
        assert torch.equal(outside[0], base) and torch.equal(outside[1], rbase)  # nothing beside the slices changed


def test_rows_far_apart():
    """Offsets past 32 bits: 2300 rows 2^20 elements apart."""
    base = torch.empty(2300, 1 << 20, device="cuda", dtype=BF)
    x = base[:, :72]
    x.copy_(rand(gen(2), 2300, 72))
    w = rand(gen(3), 72)
    y, _ = dn.add_rms_norm(x, w)
    close(y, ol.rms_norm(f64(x), None, f64(w), 1e-5)[0], BF)
    dx, _, dw = dn.add_rms_norm_backward(y, None, x, w)
    rd, rdw = ol.rms_norm_backward(f64(y), None, f64(x), f64(w), 1e-5)
    assert np.abs(f64(dx) - rd).max() <= 2.0 ** -8 * np.abs(rd).max()


def test_zero_rows_nan_and_infinity():
    g = gen(4)
    x, w = rand(g, 6, 256), rand(g, 256)
    x[0] = 0
    x[1, 17] = float("nan")
    x[2, 3] = float("inf")
    y, _ = dn.add_rms_norm(x, w)
    q, scale, _ = dn.add_rms_norm_f8(x, w, group=64)
    ref = (x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)) * w
    assert (y[0] == 0).all() and (q[0].float() == 0).all() and (scale[0] == 1).all()
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(torch.isnan(q.float()), torch.isnan(ref))
    assert (scale[1] == 1).all()
    close(y[3:], f64(ref[3:]) * 0 + ol.rms_norm(f64(x[3:]), None, f64(w), 1e-5)[0], F32)
    # scales below the smallest normal float32 stay usable
    tiny = torch.full((2, 64), 1e-30, device="cuda")
    q, scale, _ = dn.add_rms_norm_f8(tiny, torch.full((64,), 1e-12, device="cuda"), eps=1.0)
    assert (scale == 2.0 ** -126).all() and torch.isfinite(q.float()).all()
    assert dn.add_rms_norm(torch.empty(0, 16, device="cuda"), rand(g, 16))[0].shape == (0, 16)


@pytest.mark.parametrize("width", [1, 7, 40, 128, 520, 1000, 2048, 4104, 8192, 16384])
@pytest.mark.parametrize("types", [(BF, BF, BF), (BF, F32, BF), (F32, F32, F32), (BF, F32, F32)])
@pytest.mark.parametrize("rows", [1, 5, 1203])
def test_backward(width, types, rows):
    yd, rd, xd = types
    g = gen(width * rows)
    dy, dr, r, w = rand(g, rows, width, dtype=yd), rand(g, rows, width, dtype=rd), rand(g, rows, width, dtype=rd), rand(g, width)
    dx, dres, dw = dn.add_rms_norm_backward(dy, dr, r, w, 1e-5, x_dtype=xd)
    ref, ref_w = ol.rms_norm_backward(f64(dy), f64(dr), f64(r), f64(w), 1e-5)
    inv = 1 / np.sqrt((f64(r) ** 2).mean(-1, keepdims=True) + 1e-5)
    m = np.abs(f64(dy) * f64(w))
    size = inv * m + np.abs(f64(r)) * inv ** 3 * (m * np.abs(f64(r))).mean(-1, keepdims=True) + np.abs(f64(dr))
    assert dx.dtype == xd and dres.dtype == rd and (dx.data_ptr() == dres.data_ptr()) == (xd == rd)
    close(dx, ref, xd, size)
    close(dres, ref, rd, size)
    # d_weight: up to rows / 296 + 12 products added in order, against the sum of their magnitudes
    size_w = (np.abs(f64(dy) * f64(r)) * inv).sum(0)
    assert (np.abs(f64(dw) - ref_w) <= (REL + (rows / 100 + 20) * 2.0 ** -24) * size_w).all()
    again = dn.add_rms_norm_backward(dy, dr, r, w, 1e-5, x_dtype=xd)
    assert all(torch.equal(a, b) for a, b in zip((dx, dres, dw), again))


def test_autograd_against_differences():
    g = gen(11)
    x, res, w = rand(g, 5, 48), rand(g, 5, 48), rand(g, 48) + 1
    gy, gr = rand(g, 5, 48).double(), rand(g, 5, 48).double()
    args = [t.clone().requires_grad_() for t in (x, w, res)]
    y, r = dn.AddRmsNormFunction.apply(*args, 1e-5)
    (y.double() * gy).sum().add((r.double() * gr).sum()).backward()

    def f(x, w, res):
        y, r = dn.add_rms_norm(x, w, res)
        return float((y.double() * gy).sum() + (r.double() * gr).sum())

    eps = 2.0 ** -7  # differences of a smooth function: eps^2 of its third derivative (order 1 per element) and 2^-23 / eps
    for i in range(3):
        v = rand(g, *args[i].shape)
        plus, minus = ([t + s * eps * v if j == i else t for j, t in enumerate((x, w, res))] for s in (1, -1))
        want = float((args[i].grad.double() * v.double()).sum())
        size = float((args[i].grad.double() * v.double()).abs().sum())
        assert abs((f(*plus) - f(*minus)) / (2 * eps) - want) < 2e-3 * size
    x2 = x.clone().requires_grad_()
    dn.AddRmsNormFunction.apply(x2, w).backward(gy.float())
    assert np.abs(f64(x2.grad) - ol.rms_norm_backward(f64(gy), None, f64(x), f64(w), 1e-5)[0]).max() < 1e-4


def test_on_a_side_stream():
    g = gen(12)
    x, res, w = rand(g, 4096, 2048, dtype=BF), rand(g, 4096, 2048, dtype=BF), rand(g, 2048)
    want = dn.add_rms_norm(x, w, res)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = x * 1
        got = dn.add_rms_norm(late, w, res)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(dn.DeltaShapeError):
        dn.add_rms_norm(x, torch.ones(63, device="cuda"))
    with pytest.raises(dn.DeltaShapeError):
        dn.add_rms_norm(x, w, torch.zeros(4, 65, device="cuda"))
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm(x.half(), w)
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm(x.cpu(), w)
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm(x, w.cpu())
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm(x.t(), torch.ones(4, device="cuda"))
    with pytest.raises(dn.DeltaShapeError):
        dn.add_rms_norm_f8(x, w, group=48)
    with pytest.raises(dn.DeltaShapeError):
        dn.add_rms_norm_f8(x, w, group=128)
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm(torch.zeros(1, 16385, device="cuda"), torch.ones(16385, device="cuda"))
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm(x[:1].expand(4, 64), w)  # rows on top of each other
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm(x, w, eps=float("nan"))
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm(x, w, y_out=torch.empty(4, 64, device="cuda"), residual=x.to(BF), residual_dtype=F32)
    with pytest.raises(dn.DeltaCoreError):
        dn.add_rms_norm_backward(x, None, x, w, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
