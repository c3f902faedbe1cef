"""The residual add + RMS norm on the GPU with more rows than the card holds at once, so that CTAs go on to further rows with the
next row's loads under way and the last pass is partly empty; and rows far from 1 in size.

Tolerances are test_gpu_layers_norm's.  The longest chain of additions behind a row's mean is 32 values of a thread, 5 shuffles
and the 15 other warps of the widest rows: 52 roundings of 2^-24, halved by the root, and four more make 1.8e-6 of REL's 4e-6."""
import importlib

import numpy as np
import pytest
import torch

from oracle import layers as ol
from test_gpu_layers_norm import BF, F32, REL, close, f64, gen, rand

pytestmark = pytest.mark.gpu
dn = importlib.import_module("burn-deltanet_b200")

# the grid has 8 CTAs of 256 threads for every SM at most: 1184 rows at a time where a row takes a CTA, 9472 where it takes a warp
MANY = [(2371, 2048), (2999, 1560), (9601, 40), (9601, 128), (9601, 129), (20011, 264), (2371, 2047), (1301, 4104), (1187, 5001), (600, 16384)]


def slices(g, rows, width, off, *dtypes):
    return [None if d is None else rand(g, rows, width + 16, dtype=d)[:, off:off + width] for d in dtypes]


@pytest.mark.parametrize("rows,width", MANY)
@pytest.mark.parametrize("types", [(BF, BF, BF), (BF, F32, BF), (F32, F32, F32), (F32, BF, BF), (BF, None, F32)])
@pytest.mark.parametrize("off", [0, 3])
def test_forward(rows, width, types, off):
    xd, rd, od = types
    g = gen(width + rows)
    x, res = slices(g, rows, width, off, xd, rd)
    w = rand(g, width) + 1
    y, r = dn.add_rms_norm(x, w, res, 1e-5, out_dtype=od)
    ry, rr = ol.rms_norm(f64(x), f64(res), f64(w), 1e-5)
    close(y, ry, od)
    close(r, rr, r.dtype)
    if rd is not None:  # in place, the next rows' loads under way
        y2, r2 = dn.add_rms_norm(x, w, res, 1e-5, out_dtype=od, y_out=x if od == xd else None, residual_out=res)
        assert r2.data_ptr() == res.data_ptr() and torch.equal(r2, r) and torch.equal(y2, y)


@pytest.mark.parametrize("rows,width,group", [(2371, 2048, 128), (2371, 2048, 0), (9601, 128, 32), (9601, 40, 0), (9601, 96, 32), (2371, 2047, 0), (1301, 8192, 256)])
@pytest.mark.parametrize("types", [(BF, F32), (F32, F32), (BF, BF)])
@pytest.mark.parametrize("off", [0, 3])
def test_f8(rows, width, group, types, off):
    g = gen(width)
    x, res = slices(g, rows, width, off, *types)
    w = rand(g, width)
    q, scale, r = dn.add_rms_norm_f8(x, w, res, 1e-5, group=group)
    ry, rr = ol.rms_norm(f64(x), f64(res), f64(w), 1e-5)
    want = np.abs(ry.reshape(rows, -1, group or width)).max(-1) / 448
    assert (np.abs(f64(scale) - want) <= 2 * REL * want).all()
    v = ry / np.repeat(f64(scale), group or width, axis=1)
    step = np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10)
    assert (np.abs(f64(q) - v) <= step * (1 + 1e-4) + 4 * REL * np.abs(v)).all()
    assert (f64(q) != ol.to_e4m3(v)).mean() < 1e-3
    close(r, rr, types[1])


@pytest.mark.parametrize("rows,width", [(2371, 2048), (9601, 40), (9601, 129), (2371, 2047), (1301, 4104), (300, 16384)])
@pytest.mark.parametrize("types", [(BF, BF, BF), (BF, F32, BF), (F32, F32, F32), (F32, BF, F32)])
@pytest.mark.parametrize("off", [0, 3])
def test_backward(rows, width, types, off):
    yd, rd, xd = types
    g = gen(width * rows)
    dy, dr, r = slices(g, rows, width, off, yd, rd, rd)
    w = rand(g, width)
    dx, dres, dw = dn.add_rms_norm_backward(dy, dr, r, w, 1e-5, x_dtype=xd)
    ref, ref_w = ol.rms_norm_backward(f64(dy), f64(dr), f64(r), f64(w), 1e-5)
    inv = 1 / np.sqrt((f64(r) ** 2).mean(-1, keepdims=True) + 1e-5)
    m = np.abs(f64(dy) * f64(w))
    size = inv * m + np.abs(f64(r)) * inv ** 3 * (m * np.abs(f64(r))).mean(-1, keepdims=True) + np.abs(f64(dr))
    close(dx, ref, xd, size)
    close(dres, ref, rd, size)
    size_w = (np.abs(f64(dy) * f64(r)) * inv).sum(0)
    assert (np.abs(f64(dw) - ref_w) <= (REL + (rows / 100 + 20) * 2.0 ** -24) * size_w).all()


@pytest.mark.parametrize("width", [64, 37, 2048, 8192])
@pytest.mark.parametrize("scale", [1e-16, 1e-13, 1e-9, 1e9, 1e13, 1e16])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_small_and_large_rows(width, scale, dtype):
    """Rows whose squares float32 holds, without an eps: the inverse root's cube is past its range on either side."""
    g = gen(width)
    r, dy, w = rand(g, 9, width, dtype=dtype, scale=scale), rand(g, 9, width, dtype=dtype), rand(g, width) + 1
    y, _ = dn.add_rms_norm(r, w, None, 0.0, out_dtype=F32)
    close(y, ol.rms_norm(f64(r), None, f64(w), 0.0)[0], F32)
    dx, _, dw = dn.add_rms_norm_backward(dy, None, r, w, 0.0)
    ref, ref_w = ol.rms_norm_backward(f64(dy), None, f64(r), f64(w), 0.0)
    inv = 1 / np.sqrt((f64(r) ** 2).mean(-1, keepdims=True))
    m = np.abs(f64(dy) * f64(w))
    close(dx, ref, dtype, inv * m + np.abs(f64(r)) * inv ** 3 * (m * np.abs(f64(r))).mean(-1, keepdims=True))
    assert (np.abs(f64(dw) - ref_w) <= (REL + 20 * 2.0 ** -24) * (np.abs(f64(dy) * f64(r)) * inv).sum(0)).all()


def test_slices_of_one_buffer():
    """Inputs and outputs as neighbouring columns or rows of one buffer, and y over the residual while the sum goes elsewhere."""
    g = gen(5)
    w = rand(g, 64)
    base = rand(g, 50, 4 * 64)
    x, res, y_out, r_out = base.split(64, 1)
    want = dn.add_rms_norm(x.clone(), w, res.clone())
    got = dn.add_rms_norm(x, w, res, y_out=y_out, residual_out=r_out)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    lines = rand(g, 100, 64)
    want = dn.add_rms_norm(lines[:50].clone(), w)
    assert torch.equal(dn.add_rms_norm(lines[:50], w, y_out=lines[50:])[0], want[0])
    lines = rand(g, 100, 64)
    want = dn.add_rms_norm(lines[::2].clone(), w)
    assert torch.equal(dn.add_rms_norm(lines[::2], w, y_out=lines[1::2])[0], want[0])
    x, res = rand(g, 50, 64), rand(g, 50, 64)
    want = dn.add_rms_norm(x, w, res)
    got = dn.add_rms_norm(x, w, res, y_out=res, residual_out=torch.empty_like(res))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
