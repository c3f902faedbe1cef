"""The causal depthwise convolution (dc_causal_conv, dc_causal_conv_bwd) on the GPU against the float64 oracle.

Tolerances, per element: pre is `taps` multiply-adds and the bias (at most 9 roundings of 2^-24 of the sum of magnitudes);
SiLU's fast exponential is good to 2 + 1.2 |pre| ulp, its division to 2, and SiLU's slope is under 1.1: together under
2e-6 (1 + |pre|) M, M = 1 + the sum of magnitudes; taken as 4e-6 (1 + |pre|) M.  bfloat16 outputs add half an ulp.
d_x sums `taps` such terms; d_weight, d_bias and d_window sum over tokens, measured against the sum of magnitudes."""
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


def inputs(b, s, c, k, dtype, seed, bias=True, window=True):
    g = gen(seed)
    return (rand(g, b, s, c, dtype=dtype), rand(g, c, k, scale=k ** -0.5), rand(g, c) if bias else None,
            rand(g, b, c, k) if window else None)


def int32(v):
    return None if v is None else torch.tensor(v, device="cuda", dtype=torch.int32)


def magnitude(x, w, bias, win, lens):
    """1 + the sum of magnitudes behind each pre."""
    m, _ = ol.causal_conv(np.abs(f64(x)), np.abs(f64(w)), None if bias is None else np.abs(f64(bias)), None if win is None else np.abs(f64(win)),
                          False, lens)
    return 1 + m


def check_forward(x, w, bias, win, silu=True, lens=None, out_dtype=None):
    y, nxt = dn.causal_conv(x, w, bias, win, silu=silu, lengths=int32(lens), out_dtype=out_dtype)
    clean = x if lens is None else torch.where(torch.arange(x.shape[1], device="cuda")[None, :, None] < int32(lens)[:, None, None], x, 0)
    ry, rn = ol.causal_conv(f64(clean), f64(w), f64(bias), f64(win), silu, lens)
    m = magnitude(clean, w, bias, win, lens)
    err = np.abs(f64(y) - ry)
    off = REL * (1 + m) * m
    bound = off + half_ulp(np.abs(ry) + off, y.dtype)
    assert (err <= bound).all(), float((err / bound).max())
    assert np.array_equal(f64(nxt), rn.astype(np.float32).astype(np.float64))
    return y, nxt


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("s", [0, 1, 2, 3, 7, 64, 130])
@pytest.mark.parametrize("c", [1, 7, 96, 264])
def test_forward(k, s, c):
    x, w, bias, win = inputs(2, s, c, k, BF if c % 2 else F32, seed=s * 8 + k)
    check_forward(x, w, bias, win)
    check_forward(x, w, None, None, silu=False)


@pytest.mark.parametrize("types", [(BF, BF), (BF, F32), (F32, BF), (F32, F32)])
@pytest.mark.parametrize("c", [512, 1000, 77])
def test_types_and_long_sequences(types, c):
    x, w, bias, win = inputs(3, 333, c, 4, types[0], seed=c)
    check_forward(x, w, bias, win, out_dtype=types[1])


@pytest.mark.parametrize("k", [1, 3, 4, 6])
def test_lengths_and_what_is_behind_them(k):
    lens = [0, 1, 2, k, 40, 99, 100, 1000, -3]
    x, w, bias, win = inputs(len(lens), 100, 40, k, F32, seed=k)
    for i, n in enumerate(lens):
        x[i, min(max(n, 0), 100):] = float("nan")
    y, _ = check_forward(x, w, bias, win, lens=np.clip(lens, 0, 100))
    assert torch.isfinite(y).all()


def test_a_prompt_in_pieces_is_the_prompt():
    x, w, bias, win = inputs(2, 90, 24, 4, BF, seed=5)
    y, nxt = dn.causal_conv(x, w, bias, win)
    at, parts, state = 0, [], win
    for n in (1, 1, 2, 3, 50, 33):
        if n == 1:
            p, state = dn.causal_conv_step(x[:, at], w, bias, state)
            p = p[:, None]
        else:
            p, state = dn.causal_conv(x[:, at:at + n], w, bias, state)
        parts.append(p)
        at += n
    assert torch.equal(torch.cat(parts, 1), y) and torch.equal(state, nxt)


@pytest.mark.parametrize("k", [1, 2, 4, 7])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_step_in_place(k, dtype):
    x, w, bias, win = inputs(33, 1, 50, k, dtype, seed=k)
    y, nxt = check_forward(x, w, bias, win)
    y2, n2 = dn.causal_conv_step(x[:, 0], w, bias, win, window_out=win)
    assert n2.data_ptr() == win.data_ptr() and torch.equal(y2, y[:, 0]) and torch.equal(win, nxt)


def test_slices_of_a_projection():
    """x and d_y as column slices (aligned and odd offsets), y into a slice."""
    g = gen(9)
    for c, off in ((64, 16), (64, 3), (31, 1)):
        base = rand(g, 2, 70, 3 * c + 40, dtype=BF)
        x = base[..., off:off + c]
        _, w, bias, win = inputs(2, 1, c, 4, BF, seed=c + off)
        out = torch.zeros(2, 70, 2 * c + 1, device="cuda", dtype=BF)
        y, _ = dn.causal_conv(x, w, bias, win, y_out=out[..., 1:1 + c])
        want, _ = dn.causal_conv(x.contiguous(), w, bias, win)
        assert torch.equal(y, want) and (out[..., 0] == 0).all() and (out[..., 1 + c:] == 0).all()
        gy = rand(g, 2, 70, 2 * c, dtype=BF)[..., :c]
        got = dn.causal_conv_backward(gy, None, x, w, bias, win)
        ref = dn.causal_conv_backward(gy.contiguous(), None, x.contiguous(), w, bias, win)
        for a, b in zip(got, ref):
            assert np.allclose(f64(a), f64(b), rtol=2.0 ** -7, atol=1e-4)


def test_tokens_far_apart():
    """Offsets past 32 bits: 2300 tokens 2^20 elements apart."""
    base = torch.empty(1, 2300, 1 << 20, device="cuda", dtype=BF)
    x = base[..., :40]
    _, w, bias, win = inputs(1, 1, 40, 4, BF, seed=1)
    x.copy_(rand(gen(2), 1, 2300, 40))
    y, _ = dn.causal_conv(x, w, bias, win)
    want, _ = dn.causal_conv(x.contiguous(), w, bias, win)
    assert torch.equal(y, want)


def check_backward(b, s, c, k, dtype, lens=None, silu=True, bias=True, window=True, seed=0):
    x, w, bi, win = inputs(b, s, c, k, dtype, seed, bias, window)
    g = gen(seed + 1)
    gy, gn = rand(g, b, s, c, dtype=dtype), rand(g, b, c, k)
    if lens is not None:
        for i, n in enumerate(lens):
            x[i, n:], gy[i, n:] = float("nan"), float("nan")
    zero = lambda t: t if lens is None else torch.nan_to_num(t)
    got = dn.causal_conv_backward(gy, gn, x, w, bi, win, silu=silu, lengths=int32(lens))
    args = (f64(zero(gy)), f64(gn), f64(zero(x)), f64(w), f64(bi), f64(win))
    ref = ol.causal_conv_backward(*args, silu=silu, lengths=lens)
    mag = magnitude(zero(x), w, bi, win, lens)
    # the gradient of pre: |d_y| times a slope under 1.1, good to REL (1 + |pre|) M
    ge = 1.1 * np.abs(args[0]) * REL * (1 + mag) * mag
    size = ol.causal_conv_backward(1.1 * np.abs(args[0]) + 0 * mag, np.abs(args[1]), np.abs(args[2]), np.abs(args[3]), None,
                                   None if win is None else np.abs(args[5]), False, lens)
    err = ol.causal_conv_backward(ge, None, np.abs(args[2]), np.abs(args[3]), None, None if win is None else np.abs(args[5]), False, lens)
    adds = (s * b / 16 + 80) * 2.0 ** -24  # roundings of the longest chain of additions of the token sums
    for name, t, r, m, e in zip(("d_x", "d_weight", "d_bias", "d_window"), got, ref, size, err):
        if t is None:
            continue
        bound = e + (adds + REL) * m
        bound = bound + half_ulp(np.abs(r) + bound, t.dtype) + 1e-30
        off = np.abs(f64(t) - r)
        assert (off <= bound).all(), (name, float((off / bound).max()))
    again = dn.causal_conv_backward(gy, gn, x, w, bi, win, silu=silu, lengths=int32(lens))
    assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("s", [0, 1, 2, 5, 64, 67])
@pytest.mark.parametrize("c", [1, 40, 135])
def test_backward(k, s, c):
    check_backward(2, s, c, k, F32, seed=k * 100 + s)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("silu", [True, False])
def test_backward_long(dtype, silu):
    check_backward(3, 300, 264, 4, dtype, silu=silu, seed=3)
    check_backward(2, 150, 99, 4, dtype, silu=silu, bias=False, window=False, seed=4)


@pytest.mark.parametrize("k", [1, 2, 4, 8])
def test_backward_with_lengths(k):
    check_backward(7, 100, 48, k, F32, lens=[0, 1, 3, k, 63, 64, 100], seed=k)


def test_autograd_against_differences():
    g = gen(21)
    x, w, bias, win = inputs(2, 9, 6, 4, F32, seed=22)
    gy, gn = rand(g, 2, 9, 6).double(), rand(g, 2, 6, 4).double()
    args = [t.clone().requires_grad_() for t in (x, w, bias, win)]
    y, nxt = dn.CausalConvFunction.apply(*args)
    ((y.double() * gy).sum() + (nxt.double() * gn).sum()).backward()

    def f(*a):
        y, nxt = dn.causal_conv(*a)
        return float((y.double() * gy).sum() + (nxt.double() * gn).sum())

    eps = 2.0 ** -7
    for i in range(4):
        v = rand(g, *args[i].shape)
        plus, minus = ([t + s * eps * v if j == i else t for j, t in enumerate((x, w, bias, win))] for s in (1, -1))
        terms = args[i].grad.double() * v.double()
        assert abs((f(*plus) - f(*minus)) / (2 * eps) - float(terms.sum())) < 2e-3 * float(terms.abs().sum())


def test_refusals():
    x, w, bias, win = inputs(2, 5, 8, 4, F32, seed=0)
    for bad in (dict(weight=w[:7]), dict(bias=bias[:7]), dict(window=win[:, :, :3]), dict(x_bsc=x[0])):
        with pytest.raises((dn.DeltaShapeError, dn.DeltaCoreError)):
            dn.causal_conv(**{**dict(x_bsc=x, weight=w, bias=bias, window=win), **bad})
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv(x, torch.ones(8, 9, device="cuda"))
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv(x, w.bfloat16())
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv(x, w, lengths=torch.tensor([1, 2], device="cuda"))  # int64
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv(x, w, bias, win, window_out=win)  # in place over more than one token
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv(x, w, y_out=x)
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv(x.transpose(1, 2), torch.ones(5, 4, device="cuda"))
    with pytest.raises(dn.DeltaCoreError):
        dn.causal_conv(x.cpu(), w)
    with pytest.raises(dn.DeltaShapeError):
        dn.causal_conv_step(x, w)
    with pytest.raises(dn.DeltaShapeError):
        dn.causal_conv_backward(x[:, :4], None, x, w)
