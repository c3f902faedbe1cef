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
