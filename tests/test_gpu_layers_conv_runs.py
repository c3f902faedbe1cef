"""The causal convolution on the GPU where its runs are longer than one stage of its rings, in the types and layouts that
test_gpu_layers_conv leaves out: runs of 16 to 128 tokens, whose rings of four stages (16 tokens forward, 8 backward) turn over,
lengths that end inside a stage, and d_y of another type than x.

Tolerances and references are test_gpu_layers_conv's; long cases are compared on a few channels (the convolution is per channel)."""
import importlib

import numpy as np
import pytest
import torch

from oracle import layers as ol
from test_gpu_layers_conv import REL, f64, half_ulp, inputs, int32, magnitude, rand, gen

pytestmark = pytest.mark.gpu
dn = importlib.import_module("burn-deltanet_b200")
abi = importlib.import_module("burn-deltanet_b200._abi")
layers = importlib.import_module("burn-deltanet_b200.layers")
BF, F32 = torch.bfloat16, torch.float32


def some_channels(c):
    return sorted({0, 1, c // 2, c // 2 + 1, 63 % c, 64 % c, c - 2, c - 1})


def backward_run(gy, x, w, bias, win, lens):
    """Tokens per run of the backward, from its workspace: a line of taps + 1 sums per channel for every four runs."""
    _, need = layers._conv_bwd_plan(gy, None, x, w, bias, win, True, lens)
    ctas = need // ((w.shape[1] + 1) * w.shape[0] * 4)
    b, s, _ = x.shape
    return [r for r in (16, 32, 64) if -(-b * -(-s // r) // 4) == ctas]


def compare(got, ref, off, what):
    err = np.abs(f64(got) - ref)
    bound = off + half_ulp(np.abs(ref) + off, got.dtype) + 1e-30
    assert (err <= bound).all(), (what, float((err / bound).max()))


# (batch, tokens, channels) and the run of the forward (as many as leave 24 warps for every SM) and of the backward
SHAPES = [(7, 1025, 4096, 128, 64), (4, 901, 4096, 64, 64), (2, 897, 4088, 32, 32), (2, 600, 1496, 16, 16), (1, 7201, 4104, 128, 64)]
# taps, types of x and y, lengths, elements off a 16-byte boundary (no rings)
FORMS = [(4, BF, BF, True, 0), (4, F32, F32, True, 0), (3, BF, BF, False, 0), (2, F32, F32, True, 0), (8, BF, BF, True, 0), (8, F32, BF, False, 0),
         (1, BF, F32, True, 0), (7, BF, BF, True, 0), (3, F32, BF, True, 0), (4, BF, F32, True, 1), (8, F32, F32, True, 1), (4, BF, BF, False, 1)]


@pytest.mark.parametrize("b,s,c,fwd_run,bwd_run", SHAPES)
@pytest.mark.parametrize("k,it,ot,ragged,odd", FORMS)
def test_long_runs(b, s, c, fwd_run, bwd_run, k, it, ot, ragged, odd):
    """Forward and backward at every length of run."""
    groups = -(-c // 64)
    run = 128
    while run > 16 and b * -(-s // run) * groups < torch.cuda.get_device_properties(0).multi_processor_count * 24:
        run //= 2
    assert run == fwd_run
    g = gen(s + k)
    at = some_channels(c)
    x = torch.empty(b, s, c + 8, device="cuda", dtype=it)[..., odd:odd + c]
    gy = torch.empty(b, s, c + 8, device="cuda", dtype=ot)[..., odd:odd + c]
    x.copy_(rand(g, b, s, c, dtype=it))
    gy.copy_(rand(g, b, s, c, dtype=ot))
    w, bias, win, gn = rand(g, c, k, scale=k ** -0.5), rand(g, c), rand(g, b, c, k), rand(g, b, c, k)
    # the whole sequence, the end of a run, one token into a stage, in its middle, just behind a stage and a run
    lens = [(s, s // fwd_run * fwd_run, 3 * 16 + 1, s // 2 // 16 * 16 + 7, s // 3 // 8 * 8, 2 * fwd_run + 1, s - 1, 5, 0)[i % 9] for i in range(b)] if ragged else None
    if ragged:
        for i, n in enumerate(lens):
            x[i, n:], gy[i, n:] = float("nan"), float("nan")
    assert [bwd_run] == backward_run(gy, x, w, bias, win, int32(lens))
    y, nxt = dn.causal_conv(x, w, bias, win, lengths=int32(lens), out_dtype=ot)
    got = dn.causal_conv_backward(gy, gn, x, w, bias, win, lengths=int32(lens))
    # on a few channels
    cut = lambda t: torch.nan_to_num(t[..., at]) if ragged else t[..., at]
    xs, gs, ws, bs, wins, gns = cut(x), cut(gy), w[at], bias[at], win[:, at], gn[:, at]
    ry, rn = ol.causal_conv(f64(xs), f64(ws), f64(bs), f64(wins), True, lens)
    mag = magnitude(xs, ws, bs, wins, lens)
    compare(y[..., at], ry, REL * (1 + mag) * mag, "y")
    assert np.array_equal(f64(nxt[:, at]), rn.astype(np.float32).astype(np.float64))
    if ragged:
        assert all((y[i, n:] == 0).all() and (got[0][i, n:] == 0).all() for i, n in enumerate(lens))
    assert torch.isfinite(y).all() and all(torch.isfinite(t).all() for t in got)
    args = (f64(gs), f64(gns), f64(xs), f64(ws), f64(bs), f64(wins))
    ref = ol.causal_conv_backward(*args, lengths=lens)
    ge = 1.1 * np.abs(args[0]) * REL * (1 + mag) * mag
    size = ol.causal_conv_backward(1.1 * np.abs(args[0]) + 0 * mag, np.abs(args[1]), *map(np.abs, args[2:4]), None, np.abs(args[5]), False, lens)
    err = ol.causal_conv_backward(ge, None, *map(np.abs, args[2:4]), None, np.abs(args[5]), False, lens)
    adds = (s * b / 16 + 80) * 2.0 ** -24
    mine = (got[0][..., at], got[1][at], got[2][at], got[3][:, at])
    for name, t, r, m, e in zip(("d_x", "d_weight", "d_bias", "d_window"), mine, ref, size, err):
        compare(t, r, e + (adds + REL) * m, name)


@pytest.mark.parametrize("types", [(BF, F32), (F32, BF), (BF, BF)])
@pytest.mark.parametrize("k", [2, 4, 6])
@pytest.mark.parametrize("c", [40, 135])
def test_backward_types_and_lengths(types, k, c):
    """d_y of another type than x, and ragged batches of bfloat16, every channel against the oracle."""
    lens = [0, 1, 3, k, 63, 64, 100]
    b, s = len(lens), 100
    x, w, bias, win = inputs(b, s, c, k, types[0], seed=k + c)
    g = gen(c)
    gy, gn = rand(g, b, s, c, dtype=types[1]), rand(g, b, c, k)
    for i, n in enumerate(lens):
        x[i, n:], gy[i, n:] = float("nan"), float("nan")
    got = dn.causal_conv_backward(gy, gn, x, w, bias, win, lengths=int32(lens))
    xs, gs = torch.nan_to_num(x), torch.nan_to_num(gy)
    mag = magnitude(xs, w, bias, win, lens)
    args = (f64(gs), f64(gn), f64(xs), f64(w), f64(bias), f64(win))
    ref = ol.causal_conv_backward(*args, lengths=lens)
    ge = 1.1 * np.abs(args[0]) * REL * (1 + mag) * mag
    size = ol.causal_conv_backward(1.1 * np.abs(args[0]) + 0 * mag, np.abs(args[1]), *map(np.abs, args[2:4]), None, np.abs(args[5]), False, lens)
    err = ol.causal_conv_backward(ge, None, *map(np.abs, args[2:4]), None, np.abs(args[5]), False, lens)
    adds = (s * b / 16 + 80) * 2.0 ** -24
    assert got[0].dtype == types[0]
    for name, t, r, m, e in zip(("d_x", "d_weight", "d_bias", "d_window"), got, ref, size, err):
        compare(t, r, e + (adds + REL) * m, name)
