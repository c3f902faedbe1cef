"""The float64 oracle of the operators around the token mixers against independent evaluations: torch autograd of the
formulas written with torch operations, central differences, and torch's own e4m3 rounding."""
import numpy as np
import pytest
import torch

from oracle import layers as ol

rng = np.random.default_rng(7)


def scan_inputs(b=2, s=6, c=4, n=3, groups=2, seed=0):
    r = np.random.default_rng(seed)
    nrm = r.standard_normal
    return dict(u=nrm((b, s, c)), dt=nrm((b, s, c)), a=-r.uniform(0.3, 3, (c, n)), b=nrm((b, s, groups, n)), c=nrm((b, s, groups, n)),
                d=nrm(c), z=nrm((b, s, c)), dt_bias=nrm(c) - 1, state=nrm((b, c, n)))


def directional(f, args, grads, names, eps=1e-5):
    """Central differences of the scalar f along random directions against <grad, direction>; float64: 1e-8 of the terms' size."""
    for name in names:
        v = np.random.default_rng(len(name)).standard_normal(args[name].shape)
        hi, lo = (f(**{**args, name: args[name] + s * eps * v}) for s in (1, -1))
        want, size = (grads[name] * v).sum(), np.abs(grads[name] * v).sum() + 1e-3
        assert abs((hi - lo) / (2 * eps) - want) < 1e-7 * size + 1e-9, name


def test_rms_norm_gradient():
    x, w = rng.standard_normal((3, 5)), rng.standard_normal(5)
    gy, gr = rng.standard_normal((3, 5)), rng.standard_normal((3, 5))
    d, dw = ol.rms_norm_backward(gy, gr, x, w, 1e-3)

    def f(x, w):
        y, r = ol.rms_norm(x, None, w, 1e-3)
        return (y * gy).sum() + (r * gr).sum()

    directional(f, dict(x=x, w=w), dict(x=d, w=dw), ("x", "w"))


@pytest.mark.parametrize("taps", [1, 2, 4, 6])
@pytest.mark.parametrize("silu", [True, False])
def test_conv_gradient(taps, silu):
    b, s, c = 3, 5, 2
    args = dict(x=rng.standard_normal((b, s, c)), weight=rng.standard_normal((c, taps)), bias=rng.standard_normal(c),
                window=rng.standard_normal((b, c, taps)))
    lens = [5, 0, 2]
    gy, gn = rng.standard_normal((b, s, c)), rng.standard_normal((b, c, taps))
    grads = dict(zip(("x", "weight", "bias", "window"), ol.causal_conv_backward(gy, gn, **args, silu=silu, lengths=lens)))

    def f(**kw):
        y, nxt = ol.causal_conv(**kw, silu=silu, lengths=lens)
        return (y * gy).sum() + (nxt * gn).sum()

    directional(f, args, grads, args)


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("lens", [None, [6, 0], [1, 4]])
def test_scan_gradient(softplus, lens):
    args = scan_inputs()
    if not softplus:
        args["dt"], args["dt_bias"] = np.abs(args["dt"]), np.abs(args["dt_bias"])
    gy, gs = rng.standard_normal(args["u"].shape), rng.standard_normal(args["state"].shape)
    grads = ol.selective_scan_backward(gy, gs, **args, softplus=softplus, lengths=lens)

    def f(**kw):
        y, h = ol.selective_scan(**kw, softplus=softplus, lengths=lens)
        return (y * gy).sum() + (h * gs).sum()

    directional(f, args, grads, args)


def test_scan_without_its_options():
    args = scan_inputs(seed=3)
    for k in ("d", "z", "dt_bias", "state"):
        del args[k]
    gy = rng.standard_normal(args["u"].shape)
    grads = ol.selective_scan_backward(gy, None, **args)
    directional(lambda **kw: (ol.selective_scan(**kw)[0] * gy).sum(), args, grads, args)


def test_scan_against_torch():
    """The whole scan as one torch expression per token, in float64."""
    args = scan_inputs(b=1, s=9, c=3, n=5, groups=1, seed=5)
    t = {k: torch.from_numpy(v) for k, v in args.items()}
    h, ys = t["state"], []
    for i in range(9):
        step = torch.nn.functional.softplus(t["dt"][:, i] + t["dt_bias"])
        h = torch.exp(step[..., None] * t["a"]) * h + (step * t["u"][:, i])[..., None] * t["b"][:, i]
        ys.append(((h * t["c"][:, i]).sum(-1) + t["d"] * t["u"][:, i]) * torch.nn.functional.silu(t["z"][:, i]))
    y, state = ol.selective_scan(**args)
    assert np.abs(y - torch.stack(ys, 1).numpy()).max() < 1e-13
    assert np.abs(state - h.numpy()).max() < 1e-13


def test_conv_against_torch():
    x, w, bias = rng.standard_normal((2, 11, 3)), rng.standard_normal((3, 4)), rng.standard_normal(3)
    y, _ = ol.causal_conv(x, w, bias)
    ref = torch.nn.functional.conv1d(torch.from_numpy(x).transpose(1, 2), torch.from_numpy(w)[:, None], torch.from_numpy(bias), padding=3, groups=3)
    ref = torch.nn.functional.silu(ref[..., :11]).transpose(1, 2).numpy()
    assert np.abs(y - ref).max() < 1e-13


def test_e4m3_rounding_is_torchs():
    v = np.concatenate([rng.standard_normal(4000) * 10.0 ** rng.uniform(-4, 2.3, 4000), ol.E4M3, -ol.E4M3, (ol.E4M3[1:] + ol.E4M3[:-1]) / 2])
    v = v[np.abs(v) <= 448].astype(np.float32)
    ref = torch.from_numpy(v).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(np.abs(ol.to_e4m3(v.astype(np.float64))), np.abs(ref).astype(np.float64))
