"""The selective scan on the GPU in the forms that test_gpu_layers_scan leaves out: the walk in one piece, single tokens of many
sequences, and single tokens on column slices.

Tolerances are test_gpu_layers_scan's; many channels are compared on a few of them (the scan is per channel)."""
import importlib

import numpy as np
import pytest
import torch

from oracle import layers as ol
from test_gpu_layers_scan import NAMES, check_backward, clean, close, gen, inputs, int32, magnitudes, rand

pytestmark = pytest.mark.gpu
dn = importlib.import_module("burn-deltanet_b200")
abi = importlib.import_module("burn-deltanet_b200._abi")
layers = importlib.import_module("burn-deltanet_b200.layers")
BF, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------------ the walk in one piece
def few(t, at, groups):
    """The inputs of channels `at` (the same ones of every group), as many groups."""
    c = t["u"].shape[-1]
    idx = [e * (c // groups) + i for e in range(groups) for i in at]
    cut = {}
    for k, v in t.items():
        if v is None or k in ("b", "c"):
            cut[k] = v
        else:
            cut[k] = v[idx] if k in ("a", "d", "dt_bias") else v[:, idx] if k == "state" else v[..., idx]
    return cut, idx


@pytest.mark.parametrize("n", [1, 4, 6, 8, 16, 20, 24, 32, 40, 64])
@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_walk_in_one_piece(n, groups, dtype):
    """Enough sequences and channels that the card is a third full: y, state, lengths that end inside a tile, the state in place."""
    b, s, c = 24, 45, 1000
    t = inputs(b, s, c, n, groups, dtype, seed=n)
    lens = [(45, 44, 33, 32, 31, 16, 15, 1, 0)[i % 9] for i in range(b)]
    g = layers._scan_dims(*(t[k] for k in NAMES), True, None)
    assert abi.lib().dc_selective_scan_workspace_size(g) == 0  # one launch
    for lengths in (None, lens):
        if lengths is not None:
            for i, m in enumerate(lens):
                for k in ("u", "dt", "b", "c", "z"):
                    t[k][i, m:] = float("nan")
        args = [t[k].clone() if k == "state" else t[k] for k in NAMES]
        y, h = dn.selective_scan(*args, lengths=int32(lengths), state_out=args[-1])
        assert h.data_ptr() == args[-1].data_ptr() and torch.isfinite(y).all() and torch.isfinite(h).all()
        cut, idx = few(t, [0, 1, 15, 16, 17, 250, 498, 499], groups)
        x = clean(cut, lengths)
        ry, rh = ol.selective_scan(**x, lengths=lengths)
        sy, sh = ol.selective_scan(**magnitudes(x), lengths=lengths)
        close("y", y[..., idx], ry, np.abs(sy), 3e-7 * s + 4e-6)
        close("state", h[:, idx], rh, np.abs(sh), 3e-7 * s + 4e-6)
    if n in (4, 16, 24):  # without the gate and the other options (no 16-byte staging), and off 16-byte boundaries
        t = inputs(b, s, c, n, groups, dtype, seed=n, without=("d", "z", "dt_bias", "state"))
        y, h = dn.selective_scan(*(t[k] for k in NAMES))
        cut, idx = few(t, [0, 16, 499], groups)
        ry, rh = ol.selective_scan(**clean(cut, None))
        sy, sh = ol.selective_scan(**magnitudes(clean(cut, None)))
        close("y", y[..., idx], ry, np.abs(sy), 3e-7 * s + 4e-6)
        close("state", h[:, idx], rh, np.abs(sh), 3e-7 * s + 4e-6)


@pytest.mark.parametrize("n,dtype", [(8, BF), (16, BF), (64, BF), (24, F32)])
def test_backward_of_the_walk(n, dtype):
    check_backward(inputs(9, 35, 1220, n, dtype=dtype, seed=n), lens=[0, 1, 3, 34, 35, 16, 17, 32, 33])


# ------------------------------------------------------------------------------------------------ one token, many sequences
def check_step(t, out, idx_at, groups, state_out=None):
    """t: the step's inputs ([batch, channels] and so on) against the oracle on channels idx_at of each group."""
    y, h = out
    long = {k: v if v is None or k in ("a", "d", "dt_bias", "state") else v[:, None] for k, v in t.items()}
    cut, idx = few(long, idx_at, groups)
    x = clean(cut, None)
    ry, rh = ol.selective_scan(**x)
    sy, sh = ol.selective_scan(**magnitudes(x))
    close("y", y[:, idx], ry[:, 0], np.abs(sy[:, 0]), 5e-6)
    close("state", h[:, idx], rh, np.abs(sh), 5e-6)


@pytest.mark.parametrize("batch", [255, 256])
@pytest.mark.parametrize("n", [1, 4, 7, 8, 16, 24, 32, 64])
@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_step_of_many_sequences(batch, n, groups, dtype):
    """Two sequences per thread (an odd batch leaves one alone), whole blocks of channels and a last one that is not, in place."""
    for c in (2048, 1206):
        t = inputs(batch, 1, c, n, groups, dtype, seed=n)
        t = {k: v[:, 0] if k in ("u", "dt", "b", "c", "z") else v for k, v in t.items()}
        at = [0, 1, 2, 63, 64, 255, 256, c // groups - 1]
        y, h = dn.selective_scan_step(*(t[k] for k in NAMES))
        check_step(t, (y, h), at, groups)
        state = t["state"].clone()
        y2, h2 = dn.selective_scan_step(*(t[k] for k in NAMES[:-1]), state, state_out=state)
        assert h2.data_ptr() == state.data_ptr() and torch.equal(y2, y) and torch.equal(h2, h)
    t.update(d=None, z=None, dt_bias=None, state=None)
    check_step(t, dn.selective_scan_step(*(t[k] for k in NAMES)), [0, 5, 300], groups)


@pytest.mark.parametrize("batch,c", [(5, 48), (255, 2048), (256, 1206)])
@pytest.mark.parametrize("off", [0, 8, 3, 1])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_step_on_column_slices(batch, c, off, dtype):
    """u, dt, z, b and c as slices of wider rows (of which a decode loop's projections are made), y into one."""
    n, groups = 16, 2
    t = inputs(batch, 1, c, n, groups, dtype, seed=c)
    t = {k: v[:, 0] if k in ("u", "dt", "b", "c", "z") else v for k, v in t.items()}
    cut = dict(t)
    for k in ("u", "dt", "z", "b", "c"):
        m = t[k][0].numel()
        wide = rand(gen(off), batch, m + 24, dtype=dtype)
        wide[:, off:off + m] = t[k].reshape(batch, m)
        cut[k] = wide[:, off:off + m].unflatten(-1, t[k].shape[1:])
    out = torch.zeros(batch, c + 24, device="cuda", dtype=dtype)
    y, h = dn.selective_scan_step(*(cut[k] for k in NAMES), y_out=out[:, off:off + c])
    want = dn.selective_scan_step(*(t[k] for k in NAMES))
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    assert (out[:, :off] == 0).all() and (out[:, off + c:] == 0).all()
    check_step(t, (y, h), [0, 1, c // groups - 1], groups)


@pytest.mark.parametrize("n,dtype", [(4, BF), (16, F32)])
def test_step_of_very_many_sequences(n, dtype):
    """More pairs of sequences than one axis of a grid holds."""
    b, c = 140001, 12
    t = inputs(b, 1, c, n, dtype=dtype, seed=n)
    t = {k: v[:, 0] if k in ("u", "dt", "b", "c", "z") else v for k, v in t.items()}
    y, h = dn.selective_scan_step(*(t[k] for k in NAMES))
    for part in (slice(0, 300), slice(130900, 131300), slice(139800, None)):
        cut = {k: v if k in ("a", "d", "dt_bias") else v[part] for k, v in t.items()}
        check_step(cut, (y[part], h[part]), range(c), 1)
