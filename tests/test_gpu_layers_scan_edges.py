"""The selective scan on the GPU with decay rates at the end of float32's range and steps that vanish.

Tolerances are test_gpu_layers_scan's; many channels are compared on the first 40 (the scan is per channel)."""
import importlib

import numpy as np
import pytest
import torch

from oracle import layers as ol
from test_gpu_layers_scan import NAMES, clean, close, f64, gen, inputs, int32, magnitudes, rand

pytestmark = pytest.mark.gpu
dn = importlib.import_module("burn-deltanet_b200")
BF, F32 = torch.bfloat16, torch.float32
LOWEST, INF = torch.finfo(F32).min, float("inf")


def switched_off(t, rate):
    """The rates `rate` in one state of every channel and in all states of channel 1; steps that vanish (softplus(-200)) in a
    stretch of tokens.  Returns the inputs with the rates for the float64 reference: e^(step a) is 0 for every step that is
    not 0 and 1 for those, as at -1e30."""
    t["a"][:, t["a"].shape[1] // 2] = rate
    t["a"][1] = rate
    s = t["dt"].shape[1]
    t["dt"][:, s // 8:s // 2] = -200.0
    if t["dt_bias"] is not None:
        t["dt_bias"].zero_()
    return dict(t, a=t["a"].clamp_min(-1e30))


@pytest.mark.parametrize("rate", [LOWEST, -INF, -2.4e38, -1e37])
@pytest.mark.parametrize("b,s,c,n", [(2, 37, 40, 16), (2, 1, 24, 4), (3, 16, 24, 7), (1, 1000, 24, 16), (1, 700, 20, 64), (24, 21, 1000, 24), (24, 40, 1000, 4)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_lowest_rates(rate, b, s, c, n, dtype):
    """In segments, pieces and the walk; whole and with lengths."""
    t = inputs(b, s, c, n, dtype=dtype, seed=n + s)
    ref = switched_off(t, rate)
    at = list(range(min(c, 40)))
    some = lambda t: {k: v if v is None else v[at] if k in ("a", "d", "dt_bias") else v[:, at] if k == "state" else v if k in ("b", "c") else v[..., at]
                      for k, v in t.items()}
    for lens in (None, [(s, s // 2, 1, 0, s - 1)[i % 5] for i in range(b)]):
        y, h = dn.selective_scan(*(t[k] for k in NAMES), lengths=int32(lens))
        assert torch.isfinite(y).all() and torch.isfinite(h).all()
        x = clean(some(ref), lens)
        ry, rh = ol.selective_scan(**x, lengths=lens)
        sy, sh = ol.selective_scan(**magnitudes(x), lengths=lens)
        close("y", y[..., at], ry, np.abs(sy), 3e-7 * s + 4e-6)
        close("state", h[:, at], rh, np.abs(sh), 3e-7 * s + 4e-6)


@pytest.mark.parametrize("rate", [LOWEST, -INF])
@pytest.mark.parametrize("n", [4, 7, 16, 64])
def test_lowest_rates_in_a_step(rate, n):
    for raw in (0.0, -200.0):
        t = inputs(5, 1, 48, n, seed=n)
        ref = switched_off(t, rate)
        t["dt"].fill_(raw)
        one = {k: v[:, 0] if k in ("u", "dt", "b", "c", "z") else v for k, v in t.items()}
        y, h = dn.selective_scan_step(*(one[k] for k in NAMES))
        x = clean(dict(ref, dt=t["dt"]), None)
        ry, rh = ol.selective_scan(**x)
        sy, sh = ol.selective_scan(**magnitudes(x))
        close("y", y, ry[:, 0], np.abs(sy[:, 0]), 5e-6)
        close("state", h, rh, np.abs(sh), 5e-6)


@pytest.mark.parametrize("rate", [LOWEST, -INF, -2.4e38])
@pytest.mark.parametrize("b,s,c,n", [(2, 37, 40, 16), (2, 1, 24, 4), (3, 16, 24, 7), (1, 900, 24, 16), (1, 600, 20, 64)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_lowest_rates_backward(rate, b, s, c, n, dtype):
    t = inputs(b, s, c, n, dtype=dtype, seed=n + s)
    ref = switched_off(t, rate)
    for lens in (None, [(s // 2, s, 1)[i % 3] for i in range(b)]):
        g = gen(100)
        gy, gs = rand(g, b, s, c, dtype=dtype), rand(g, b, c, n)
        got = dn.selective_scan_backward(gy, gs, *(t[k] for k in NAMES), lengths=int32(lens))
        assert all(torch.isfinite(v).all() for v in got)
        x = clean(dict(ref, d_y=gy), lens)
        x["d_state"] = f64(gs)
        want = ol.selective_scan_backward(**x, lengths=lens)
        size = ol.selective_scan_backward(**magnitudes(x), lengths=lens, sizes=True)
        for name, v in zip(NAMES, got):
            close("d_" + name, v, want[name], np.abs(size[name]), 9e-7 * s + 2e-5)


def test_a_nan_rate_is_not_hidden():
    t = inputs(2, 20, 8, 4, seed=1)
    t["a"][3, 2] = float("nan")
    y, h = dn.selective_scan(*(t[k] for k in NAMES))
    assert torch.isnan(y[:, :, 3]).all() and torch.isnan(h[:, 3, 2]).all() and torch.isfinite(y[:, :, :3]).all()


@pytest.mark.parametrize("s", [384, 385, 400, 511, 513, 1023, 1025])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_lengths_around_the_pieces(s, dtype):
    """Pieces of 128 to 192 tokens, the last one short; checkpoints in each of them."""
    t = inputs(2, s, 24, 16, dtype=dtype, seed=s)
    lens = [s, s // 3 + 1]
    y, h, saved = dn.selective_scan(*(t[k] for k in NAMES), lengths=int32(lens), checkpoints=True)
    x = clean(t, lens)
    ry, rh, before, _ = ol.selective_scan(**x, lengths=lens, keep=True)
    sy, sh, size, _ = ol.selective_scan(**magnitudes(x), lengths=lens, keep=True)
    close("y", y, ry, np.abs(sy), 3e-7 * s + 4e-6)
    close("state", h, rh, np.abs(sh), 3e-7 * s + 4e-6)
    saved = saved.view(2, -(-s // 16), 24, 16)
    for b, n in enumerate(lens):
        for i in range(-(-n // 16)):
            close("checkpoint", saved[b, i], before[16 * i][b], np.abs(size[16 * i][b]), 3e-7 * s + 4e-6)
