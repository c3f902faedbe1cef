"""The block-level operators on the GPU with outputs and inputs in one buffer: slices that do not touch are computed as if they were
apart, the others are refused (the refusals at given addresses are in test_layers_rows)."""
import importlib

import pytest
import torch

from test_gpu_layers_conv import gen, inputs, rand

pytestmark = pytest.mark.gpu
dn = importlib.import_module("burn-deltanet_b200")
BF, F32 = torch.bfloat16, torch.float32


def test_conv_outputs_beside_inputs():
    """y in the other half of x's rows, in the other half of its tokens, and for a single token: slices that do not touch."""
    g = gen(3)
    b, s, c = 3, 40, 24
    _, w, bias, win = inputs(b, 1, c, 4, BF, seed=3)
    rows, tokens = rand(g, b, s, 2 * c, dtype=BF), rand(g, b, 2 * s, c, dtype=BF)
    for x, out in ((rows[..., :c], rows[..., c:]), (rows[..., c:], rows[..., :c]), (tokens[:, :s], tokens[:, s:]), (tokens[:, s:], tokens[:, :s]),
                   (tokens[:, ::2], tokens[:, 1::2])):
        want = dn.causal_conv(x.clone(), w, bias, win)
        got = dn.causal_conv(x, w, bias, win, y_out=out)
        assert got[0].data_ptr() == out.data_ptr() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = rand(g, b, 2 * c, dtype=BF)
    want = dn.causal_conv_step(one[:, :c].clone(), w, bias, win)
    got = dn.causal_conv_step(one[:, :c], w, bias, win, y_out=one[:, c:])
    assert torch.equal(one[:, c:], want[0]) and torch.equal(got[1], want[1])


def test_conv_outputs_that_fold_are_refused():
    x, w, bias, win = inputs(2, 6, 32, 4, F32, seed=0)
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv(x, w, bias, win, y_out=torch.empty(1, 6, 32, device="cuda").expand(2, 6, 32))
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv_step(x[:, 0], w, bias, win, y_out=torch.empty(1, 32, device="cuda").expand(2, 32))
    # an input may: every sequence starts with the same tokens
    one = x[:1].expand(2, 6, 32)
    assert torch.equal(dn.causal_conv(one, w, bias, win)[0], dn.causal_conv(one.contiguous(), w, bias, win)[0])


def test_scan_outputs_beside_inputs():
    """y in a projection's free columns, in the other half of u's tokens, in every other token, and for single tokens."""
    from test_gpu_layers_scan import NAMES, inputs as scan_inputs

    b, s, c = 3, 40, 24
    t = scan_inputs(b, s, c, 16, dtype=BF, seed=3)
    want = dn.selective_scan(*(t[k] for k in NAMES))
    g = gen(4)
    rows, tokens = rand(g, b, s, 3 * c, dtype=BF), rand(g, b, 2 * s, c, dtype=BF)
    for u, out in ((rows[..., :c], rows[..., c:2 * c]), (rows[..., 2 * c:], rows[..., c:2 * c]), (tokens[:, :s], tokens[:, s:]),
                   (tokens[:, s:], tokens[:, :s]), (tokens[:, ::2], tokens[:, 1::2])):
        u.copy_(t["u"])
        y, h = dn.selective_scan(u, *(t[k] for k in NAMES[1:]), y_out=out)
        assert y.data_ptr() == out.data_ptr() and torch.equal(y, want[0]) and torch.equal(h, want[1]) and torch.equal(u, t["u"])
    one = {k: v[:, 0] if k in ("u", "dt", "b", "c", "z") else v for k, v in t.items()}
    want = dn.selective_scan_step(*(one[k] for k in NAMES))
    row = rand(g, b, 2 * c, dtype=BF)
    row[:, :c] = one["u"]
    y, h = dn.selective_scan_step(row[:, :c], *(one[k] for k in NAMES[1:]), y_out=row[:, c:])
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])


def test_scan_outputs_over_inputs_are_refused():
    from test_gpu_layers_scan import NAMES, inputs as scan_inputs

    t = scan_inputs(2, 12, 16, 4, seed=1)
    wide = torch.zeros(2, 12, 40, device="cuda")
    wide[..., :16] = t["u"]
    for out in (wide[..., 1:17], wide[..., 15:31]):
        with pytest.raises(dn.DeltaCoreError):
            dn.selective_scan(wide[..., :16], *(t[k] for k in NAMES[1:]), y_out=out)
    with pytest.raises(dn.DeltaCoreError):
        dn.selective_scan(*(t[k] for k in NAMES), y_out=torch.empty(1, 12, 16, device="cuda").expand(2, 12, 16))
    states = torch.zeros(3, 16, 4, device="cuda")
    with pytest.raises(dn.DeltaCoreError):
        dn.selective_scan(*(t[k] for k in NAMES[:-1]), states[:2], state_out=states[1:])
