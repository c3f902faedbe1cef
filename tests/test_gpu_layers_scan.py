"""The selective scan (dc_selective_scan, its step and its backward) on the GPU against the float64 oracle, token by token.

Tolerances.  A token's decay is off by the exponential's 2^-22.5 and the rounding of its argument step * a (whose own effect
over many tokens is x e^-x of 6e-7, x the sum of the arguments: below 3e-7), and each token's state by two more roundings:
under 3e-7 of the state per token that it survives.  So the state and the read-out are within (3e-7 T + 4e-6) of the same scan
over magnitudes, 4e-6 covering softplus, the gate and the read-out's sum; bfloat16 outputs add half an ulp.  The
gradients pass through two such walks and one sum over tokens or channels: (9e-7 T + 2e-5) of their terms' magnitudes."""
import importlib

import numpy as np
import pytest
import torch

from oracle import layers as ol

pytestmark = pytest.mark.gpu
dn = importlib.import_module("burn-deltanet_b200")
BF, F32 = torch.bfloat16, torch.float32
NAMES = ("u", "dt", "a", "b", "c", "d", "z", "dt_bias", "state")


def half_ulp(ref, dtype):
    """Half the distance between the bfloat16 values around ref (float32's is in the other terms)."""
    return np.exp2(np.floor(np.log2(np.maximum(np.abs(ref), 1e-38))) - 8) if dtype == BF else 0.0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def f64(t):
    return None if t is None else t.double().cpu().numpy()


def int32(v):
    return None if v is None else torch.tensor(v, device="cuda", dtype=torch.int32)


def inputs(b, s, c, n, groups=1, dtype=F32, seed=0, without=()):
    g = gen(seed)
    t = dict(u=rand(g, b, s, c, dtype=dtype), dt=rand(g, b, s, c, dtype=dtype), a=-torch.rand(c, n, device="cuda", generator=g) * 4 - 0.02,
             b=rand(g, b, s, groups, n, dtype=dtype), c=rand(g, b, s, groups, n, dtype=dtype), d=rand(g, c), z=rand(g, b, s, c, dtype=dtype),
             dt_bias=rand(g, c) - 2, state=rand(g, b, c, n))
    return {k: None if k in without else v for k, v in t.items()}


def clean(t, lens):
    """The inputs with their padding zeroed, float64."""
    out = {}
    for k, v in t.items():
        v = f64(v)
        if lens is not None and k in ("u", "dt", "b", "c", "z", "d_y") and v is not None:
            live = np.arange(v.shape[1])[None, :] < np.asarray(lens)[:, None]
            v = np.where(live.reshape(live.shape + (1,) * (v.ndim - 2)), v, 0)
        out[k] = v
    return out


def magnitudes(t64):
    return {k: v if v is None or k in ("a", "dt", "dt_bias") else np.abs(v) for k, v in t64.items()}


def close(name, got, ref, size, rel):
    err = np.abs(f64(got) - ref)
    bound = rel * size + half_ulp(np.abs(ref) + rel * size, got.dtype) + 1e-30
    assert (err <= bound).all(), (name, float((err / bound).max()))


def check(t, lens=None, softplus=True, out_dtype=None, **kw):
    y, h = dn.selective_scan(*(t[k] for k in NAMES), lengths=int32(lens), softplus=softplus, out_dtype=out_dtype, **kw)
    x = clean(t, lens)
    ry, rh = ol.selective_scan(**x, softplus=softplus, lengths=lens)
    sy, sh = ol.selective_scan(**magnitudes(x), softplus=softplus, lengths=lens)
    rel = 3e-7 * t["u"].shape[1] + 4e-6
    close("y", y, ry, np.abs(sy), rel)
    close("state", h, rh, np.abs(sh), rel)
    return y, h


@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 12, 16, 17, 24, 32, 33, 64])
@pytest.mark.parametrize("s", [1, 2, 9, 33, 130])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_forward(n, s, dtype):
    check(inputs(2, s, 40, n, dtype=dtype, seed=n + s))


@pytest.mark.parametrize("c,groups", [(1, 1), (5, 1), (16, 1), (17, 1), (30, 3), (96, 2), (100, 4), (160, 1)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_channels_and_groups(c, groups, dtype):
    check(inputs(3, 45, c, 16, groups, dtype, seed=c))
    check(inputs(1, 20, c, 6, groups, dtype, seed=c))


@pytest.mark.parametrize("without", [("d",), ("z",), ("dt_bias",), ("state",), ("d", "z", "dt_bias", "state")])
@pytest.mark.parametrize("softplus", [True, False])
def test_options(without, softplus):
    t = inputs(2, 37, 24, 16, seed=3, without=without)
    if not softplus:
        t["dt"] = t["dt"].abs() * 0.1
        t["dt_bias"] = None if t["dt_bias"] is None else t["dt_bias"].abs() * 0.1
    check(t, softplus=softplus)


@pytest.mark.parametrize("types", [(BF, F32), (F32, BF)])
def test_output_types(types):
    check(inputs(2, 50, 32, 16, dtype=types[0], seed=4), out_dtype=types[1])


@pytest.mark.parametrize("n", [4, 8, 16, 30, 64])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_lengths_and_what_is_behind_them(n, dtype):
    lens = [0, 1, 2, 31, 32, 33, 64, 99, 100]
    t = inputs(len(lens), 100, 20, n, dtype=dtype, seed=n)
    for i, m in enumerate(lens):
        for k in ("u", "dt", "b", "c", "z"):
            t[k][i, m:] = float("nan")
    y, h = check(t, lens)
    assert torch.isfinite(y).all() and torch.equal(h[0], t["state"][0])
    wide = [-5, 1, 2, 31, 32, 33, 64, 99, 4000]  # clamped
    y2, h2 = dn.selective_scan(*(t[k] for k in NAMES), lengths=int32(wide))
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("n", [4, 8, 16, 24, 64])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_sequences_of_few_channels(n, dtype):
    """Sequences long enough for the time axis to be cut into pieces, whole and with lengths that end inside each of them, the
    state in place; in one piece where there is no workspace."""
    check(inputs(1, 1000, 24, n, dtype=dtype, seed=n))
    t = inputs(5, 700, 20, n, dtype=dtype, seed=n + 1)
    lens = [0, 1, 130, 699, 700]
    want = check(t, lens)
    args = [t[k].clone() if k == "state" else t[k] for k in NAMES]
    y, h = dn.selective_scan(*args, lengths=int32(lens), state_out=args[-1])
    assert torch.equal(y, want[0]) and torch.equal(h, want[1]) and h.data_ptr() == args[-1].data_ptr()


def test_without_a_workspace():
    """The C entry point with workspace NULL walks the sequence in one piece."""
    abi = importlib.import_module("burn-deltanet_b200._abi")
    layers = importlib.import_module("burn-deltanet_b200.layers")
    t = inputs(1, 600, 24, 16, seed=7)
    want = dn.selective_scan(*(t[k] for k in NAMES))
    g = layers._scan_dims(*(t[k] for k in NAMES), True, None)
    assert abi.lib().dc_selective_scan_workspace_size(g) > 0
    layers._scan_inputs(g, *(t[k] for k in NAMES), None)
    y, h = torch.empty_like(t["u"]), torch.empty_like(t["state"])
    g.y, g.state_out, g.y_batch_stride, g.y_token_stride = y.data_ptr(), h.data_ptr(), 600 * 24, 24
    assert abi.lib().dc_selective_scan(g, torch.cuda.current_stream().cuda_stream) == 0
    sy, sh = ol.selective_scan(**magnitudes(clean(t, None)))
    close("y", y, f64(want[0]), np.abs(sy), 2 * (3e-7 * 600 + 4e-6))
    close("state", h, f64(want[1]), np.abs(sh), 2 * (3e-7 * 600 + 4e-6))
    workspace = torch.empty(64, dtype=torch.uint8, device="cuda")
    g.workspace, g.workspace_bytes = workspace.data_ptr(), 64
    assert abi.lib().dc_selective_scan(g, torch.cuda.current_stream().cuda_stream) == abi.DC_EWORKSPACE


def test_no_tokens_and_no_sequences():
    t = inputs(2, 0, 8, 16, seed=1)
    y, h = dn.selective_scan(*(t[k] for k in NAMES))
    assert y.shape == (2, 0, 8) and torch.equal(h, t["state"])
    t = inputs(0, 5, 8, 16, seed=1)
    assert dn.selective_scan(*(t[k] for k in NAMES))[1].shape == (0, 8, 16)


@pytest.mark.parametrize("n", [5, 8, 16, 40])
def test_a_prompt_in_pieces_is_the_prompt(n):
    """Prompts and single tokens in turn, the state in place."""
    t = inputs(2, 70, 24, n, seed=n)
    y, h = check(t)
    state, parts, at = t["state"].clone(), [], 0
    for m in (1, 32, 1, 1, 7, 28):
        cut = {k: t[k][:, at:at + m] for k in ("u", "dt", "b", "c", "z")}
        if m == 1:
            one = {k: v[:, 0] for k, v in cut.items()}
            p, state = dn.selective_scan_step(one["u"], one["dt"], t["a"], one["b"], one["c"], t["d"], one["z"], t["dt_bias"], state, state_out=state)
            p = p[:, None]
        else:
            p, state = dn.selective_scan(cut["u"], cut["dt"], t["a"], cut["b"], cut["c"], t["d"], cut["z"], t["dt_bias"], state, state_out=state)
        parts.append(p)
        at += m
    x = magnitudes(clean(t, None))
    sy, sh = ol.selective_scan(**x)
    close("y", torch.cat(parts, 1), f64(y), np.abs(sy), 2 * (3e-7 * 70 + 4e-6))
    close("state", state, f64(h), np.abs(sh), 2 * (3e-7 * 70 + 4e-6))


@pytest.mark.parametrize("n", [1, 4, 6, 16, 24, 64])
@pytest.mark.parametrize("c,groups", [(3, 1), (48, 2), (200, 1)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_step(n, c, groups, dtype):
    for without in ((), ("d", "z", "dt_bias", "state")):
        t = inputs(5, 1, c, n, groups, dtype, seed=n + c, without=without)
        one = {k: v[:, 0] if v is not None and k in ("u", "dt", "b", "c", "z") else v for k, v in t.items()}
        y, h = dn.selective_scan_step(*(one[k] for k in NAMES))
        x = clean(t, None)
        ry, rh = ol.selective_scan(**x)
        sy, sh = ol.selective_scan(**magnitudes(x))
        close("y", y, ry[:, 0], np.abs(sy[:, 0]), 5e-6)
        close("state", h, rh, np.abs(sh), 5e-6)


def test_slices_of_projections():
    """u, dt, z, b and c as column slices, aligned and at odd offsets, y into a slice."""
    for c, n, off in ((32, 16, 8), (32, 16, 3), (21, 5, 1)):
        g = gen(off)
        t = inputs(2, 50, c, n, dtype=BF, seed=off)
        wide = {k: rand(g, 2, 50, 3 * c + 2 * n + 24, dtype=BF) for k in ("u", "dt", "z", "b", "c")}
        cut = dict(t)
        for k, w in wide.items():
            m = n if k in "bc" else c
            w[..., off:off + m] = t[k].reshape(2, 50, m)
            cut[k] = w[..., off:off + m]
        out = torch.zeros(2, 50, 2 * c + 1, device="cuda", dtype=BF)
        y, h = dn.selective_scan(*(cut[k] for k in NAMES), y_out=out[..., 1:1 + c])
        want = dn.selective_scan(*(t[k] for k in NAMES))
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])
        assert (out[..., 0] == 0).all() and (out[..., 1 + c:] == 0).all()
        gy = rand(g, 2, 50, 2 * c + 3, dtype=BF)[..., 3:3 + c]
        got = dn.selective_scan_backward(gy, None, *(cut[k] for k in NAMES))
        ref = dn.selective_scan_backward(gy.contiguous(), None, *(t[k] for k in NAMES))
        assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, ref))


def test_tokens_far_apart():
    """Offsets past 32 bits: 2300 tokens 2^20 elements apart."""
    t = inputs(1, 2300, 16, 16, dtype=BF, seed=1)
    base = torch.empty(1, 2300, 1 << 20, device="cuda", dtype=BF)
    cut, off = dict(t), 0
    for k in ("u", "dt", "z", "b", "c"):
        base[..., off:off + 16] = t[k].reshape(1, 2300, 16)
        cut[k] = base[..., off:off + 16]
        off += 16
    got, want = (dn.selective_scan(*(v[k] for k in NAMES)) for v in (cut, t))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_large_and_vanishing_steps():
    """Steps so large that the state is forgotten (decay 0), and so small that 1 + e^x rounds e^x away."""
    t = inputs(1, 40, 16, 16, seed=2)
    t["dt"][:, ::3] = 80.0
    t["dt"][:, 1::3] = -25.0
    t["dt_bias"].zero_()
    check(t)


def test_a_nan_stays_in_its_channel():
    t = inputs(2, 40, 32, 16, seed=6)
    want = dn.selective_scan(*(t[k] for k in NAMES))
    t["u"][0, 7, 5] = float("nan")
    y, h = dn.selective_scan(*(t[k] for k in NAMES))
    assert torch.isnan(y[0, 7:, 5]).all() and torch.isnan(h[0, 5]).all()
    y[0, :, 5], h[0, 5] = want[0][0, :, 5], want[1][0, 5]
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])


def check_backward(t, lens=None, softplus=True, out_dtype=None, with_state=True, seed=100):
    g = gen(seed)
    b, s, c = t["u"].shape
    n, dtype = t["a"].shape[1], t["u"].dtype
    gy = rand(g, b, s, c, dtype=out_dtype or dtype)
    gs = rand(g, b, c, n) if with_state else None
    if lens is not None:
        for i, m in enumerate(lens):
            gy[i, m:] = float("nan")
    args = [t[k] for k in NAMES]
    kw = dict(softplus=softplus, lengths=int32(lens))
    got = dn.selective_scan_backward(gy, gs, *args, **kw)
    saved = dn.selective_scan(*args, checkpoints=True, **kw)[2]
    again = dn.selective_scan_backward(gy, gs, *args, checkpoints=saved, **kw)
    assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))
    x = clean(dict(t, d_y=gy), lens)
    x["d_state"] = f64(gs)
    ref = ol.selective_scan_backward(**x, softplus=softplus, lengths=lens)
    size = ol.selective_scan_backward(**magnitudes(x), softplus=softplus, lengths=lens, sizes=True)
    for name, v in zip(NAMES, got):
        if t[name] is None:
            assert v is None
            continue
        assert v.dtype == t[name].dtype and v.shape == t[name].shape
        close("d_" + name, v, ref[name], np.abs(size[name]), 9e-7 * s + 2e-5)


@pytest.mark.parametrize("n", [1, 4, 7, 8, 16, 24, 33, 64])
@pytest.mark.parametrize("s", [1, 2, 9, 33, 100])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_backward(n, s, dtype):
    check_backward(inputs(2, s, 40, n, dtype=dtype, seed=n + s))


@pytest.mark.parametrize("c,groups", [(1, 1), (5, 1), (17, 1), (30, 3), (96, 2), (72, 1), (160, 1)])
def test_backward_channels_and_groups(c, groups):
    check_backward(inputs(3, 45, c, 16, groups, seed=c))
    check_backward(inputs(1, 20, c, 6, groups, seed=c), with_state=False)


def test_backward_of_many_channels():
    """Enough channels that a CTA takes several blocks of 16 one after the other, the last one short."""
    check_backward(inputs(8, 40, 1220, 16, seed=8))
    check_backward(inputs(9, 21, 2440, 8, 2, seed=9), lens=[0, 1, 3, 20, 21, 5, 6, 7, 8])


@pytest.mark.parametrize("without", [("d",), ("z",), ("dt_bias",), ("state",), ("d", "z", "dt_bias", "state")])
@pytest.mark.parametrize("softplus", [True, False])
def test_backward_options(without, softplus):
    t = inputs(2, 37, 24, 16, seed=3, without=without)
    if not softplus:
        t["dt"] = t["dt"].abs() * 0.1
        t["dt_bias"] = None if t["dt_bias"] is None else t["dt_bias"].abs() * 0.1
    check_backward(t, softplus=softplus)


@pytest.mark.parametrize("types", [(BF, F32), (F32, BF)])
def test_backward_types(types):
    check_backward(inputs(2, 50, 32, 16, dtype=types[0], seed=4), out_dtype=types[1])


@pytest.mark.parametrize("n", [4, 8, 16, 30, 64])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_backward_with_lengths(n, dtype):
    lens = [0, 1, 2, 31, 32, 33, 64, 99, 100]
    t = inputs(len(lens), 100, 20, n, dtype=dtype, seed=n)
    for i, m in enumerate(lens):
        for k in ("u", "dt", "b", "c", "z"):
            t[k][i, m:] = float("nan")
    check_backward(t, lens)


@pytest.mark.parametrize("n", [4, 8, 16, 24, 64])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_backward_of_long_sequences_of_few_channels(n, dtype):
    """The time axis in pieces, lengths that end inside each of them."""
    check_backward(inputs(1, 900, 24, n, dtype=dtype, seed=n))
    check_backward(inputs(5, 600, 20, n, 2, dtype, seed=n + 1), lens=[0, 1, 130, 599, 600])


def test_backward_of_no_tokens():
    t = inputs(2, 0, 8, 16, seed=1)
    gs = rand(gen(1), 2, 8, 16)
    got = dict(zip(NAMES, dn.selective_scan_backward(t["u"], gs, *(t[k] for k in NAMES))))
    assert torch.equal(got["state"], gs) and (got["a"] == 0).all() and (got["d"] == 0).all()
    t = inputs(0, 4, 8, 16, seed=1)
    got = dict(zip(NAMES, dn.selective_scan_backward(t["u"], None, *(t[k] for k in NAMES))))
    assert (got["a"] == 0).all() and (got["dt_bias"] == 0).all()


def test_autograd_against_differences():
    g = gen(31)
    t = inputs(2, 11, 6, 4, groups=2, seed=32)
    gy, gs = rand(g, 2, 11, 6).double(), rand(g, 2, 6, 4).double()
    args = [t[k].clone().requires_grad_() for k in NAMES]
    y, h = dn.SelectiveScanFunction.apply(*args)
    ((y.double() * gy).sum() + (h.double() * gs).sum()).backward()

    def f(*a):
        y, h = dn.selective_scan(*a)
        return float((y.double() * gy).sum() + (h.double() * gs).sum())

    eps = 2.0 ** -7
    for i, name in enumerate(NAMES):
        v = rand(g, *args[i].shape)
        plus, minus = ([t[k] + s * eps * v if k == name else t[k] for k in NAMES] for s in (1, -1))
        terms = args[i].grad.double() * v.double()
        assert abs((f(*plus) - f(*minus)) / (2 * eps) - float(terms.sum())) < 2e-3 * float(terms.abs().sum()), name


def test_on_a_side_stream():
    t = inputs(4, 300, 256, 16, dtype=BF, seed=12)
    want = dn.selective_scan(*(t[k] for k in NAMES))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = dict(t, u=t["u"] * 1)
        got = dn.selective_scan(*(late[k] for k in NAMES))
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    t = inputs(2, 5, 8, 4, seed=0)
    call = lambda **bad: dn.selective_scan(*({**t, **bad}[k] for k in NAMES))
    for bad in (dict(dt=t["dt"][:, :4]), dict(a=t["a"][:, :3]), dict(b=t["b"][..., :3]), dict(d=t["d"][:7]), dict(z=t["z"][:1]),
                dict(state=t["state"][:1]), dict(u=t["u"][0])):
        with pytest.raises(dn.DeltaShapeError):
            call(**bad)
    for bad in (dict(dt=t["dt"].bfloat16()), dict(a=t["a"].bfloat16()), dict(u=t["u"].half()), dict(z=t["z"].cpu()),
                dict(u=t["u"].transpose(1, 2).contiguous().transpose(1, 2)), dict(state=t["state"].transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(dn.DeltaCoreError):
            call(**bad)
    with pytest.raises(dn.DeltaShapeError):  # three groups do not divide eight channels
        call(b=rand(gen(0), 2, 5, 3, 4), c=rand(gen(0), 2, 5, 3, 4))
    with pytest.raises(dn.DeltaCoreError):  # more states than the kernels hold
        u = inputs(1, 3, 8, 65, seed=0)
        dn.selective_scan(*(u[k] for k in NAMES))
    with pytest.raises(dn.DeltaCoreError):
        dn.selective_scan(*(t[k] for k in NAMES), y_out=t["u"])
    with pytest.raises(dn.DeltaShapeError):
        dn.selective_scan(*(t[k] for k in NAMES), state_out=torch.empty(2, 8, 5, device="cuda"))
    with pytest.raises(dn.DeltaShapeError):
        dn.selective_scan_step(*(t[k] for k in NAMES))
    with pytest.raises(dn.DeltaShapeError):
        dn.selective_scan_backward(t["u"], None, *(t[k] for k in NAMES), checkpoints=torch.empty(3, device="cuda"))
    with pytest.raises(dn.DeltaCoreError):
        dn.selective_scan_backward(t["u"], None, *(t[k] for k in NAMES), workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("batch,seq,channels,state", [(1, 256, 64, 16), (8, 256, 2048, 16), (2, 256, 96, 24)])
def test_a_remembered_state_does_not_drift(batch, seq, channels, state):
    """With nothing added, the state is the product of its decays: its mean relative error stays under an eighth of the
    float32 spacing below 1 (2^-24) per token, so that the exponential is low or high on no account."""
    g = torch.Generator(device="cuda").manual_seed(5)
    uniform = lambda lo, hi, *shape: torch.rand(*shape, device="cuda", generator=g) * (hi - lo) + lo
    dt, a = uniform(0.02, 0.1, batch, seq, channels), -uniform(0.3, 1.4, channels, state)
    u, bc = torch.zeros_like(dt), torch.ones(batch, seq, 1, state, device="cuda")
    _, h = dn.selective_scan(u, dt, a, bc, bc, state=torch.ones(batch, channels, state, device="cuda"), softplus=False)
    ref = torch.exp(dt.double().sum(1)[..., None] * a.double())
    assert abs(float((h.double() / ref - 1).mean())) < seq * 2.0 ** -27
