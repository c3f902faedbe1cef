"""The block-level operators around the delta-rule core, as timed workloads.

Three operators, each in the directions that a program calls:

* ``norm``: a residual stream's addition and the root-mean-square norm of the sum, as float32 / bfloat16
  or as float8 (e4m3) values with scales; ``train`` adds its backward pass;
* ``conv``: the short causal depthwise convolution in front of a selective scan, over a prompt (``prompt``),
  one token with a rolling window (``step``), and with its backward pass (``train``);
* ``scan``: the selective state space scan, in the same three directions.

``own`` selects the implementation: elementary torch operations in float32, or the framework's kernels.
"""
import importlib

import torch

own = False

EPS = 1e-5
F8_MAX = 448.0  # the largest e4m3 value
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decode tick of eight sequences at the width of 16 heads x 128: the smallest call
        dict(name="norm-tick", op="norm", mode="apply", rows=8, width=2048, dtype="bf16", residual="bf16", out="bf16"),
        # a prompt batch, 8 x 4096 tokens at the same width
        dict(name="norm-prompt", op="norm", mode="apply", rows=32768, width=2048, dtype="bf16", residual="bf16", out="bf16"),
        # the same stream into an 8-bit input projection, one scale per 128 columns, the residual kept in float32
        dict(name="norm-f8", op="norm", mode="apply", rows=16384, width=4096, dtype="bf16", residual="f32", out="f8", group=128),
        # a training step of an odd number of tokens at a width that is no power of two
        dict(name="norm-train", op="norm", mode="train", rows=16381, width=1560, dtype="bf16", residual="f32", out="bf16"),
        # the convolution over a prompt batch
        dict(name="conv-prompt", op="conv", mode="prompt", batch=8, seq=4096, channels=2048, taps=4, dtype="bf16", ragged=False),
        # one decode tick of 256 sequences, the windows rolled in place
        dict(name="conv-tick", op="conv", mode="step", batch=256, seq=1, channels=2048, taps=4, dtype="bf16", ragged=False),
        # a training step over padded sequences of unequal lengths
        dict(name="conv-train", op="conv", mode="train", batch=6, seq=2049, channels=1536, taps=4, dtype="bf16", ragged=True),
        # one decode tick of 256 sequences, the states updated in place
        dict(name="scan-tick", op="scan", mode="step", batch=256, seq=1, channels=2048, state=16, groups=1, dtype="bf16", ragged=False),
        # one long prompt at a small width: few rows, a long time axis
        dict(name="scan-long", op="scan", mode="prompt", batch=1, seq=16384, channels=1024, state=16, groups=1, dtype="bf16", ragged=False),
        # a prompt batch: the largest case
        dict(name="scan-prompt", op="scan", mode="prompt", batch=8, seq=4096, channels=2048, state=16, groups=1, dtype="bf16", ragged=False),
        # padded float32 sequences of unequal lengths, odd sizes, two groups of b and c
        dict(name="scan-ragged", op="scan", mode="prompt", batch=5, seq=777, channels=1000, state=24, groups=2, dtype="f32", ragged=True),
        # a training step
        dict(name="scan-train", op="scan", mode="train", batch=4, seq=2048, channels=2048, state=16, groups=1, dtype="bf16", ragged=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["norm", "norm", "conv", "scan", "scan"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "norm":
        width = rng.choice([_spread(rng, 64, 8192), 8 * _spread(rng, 16, 1024)])
        out = rng.choice([dtype, dtype, "f8"])
        mode = "train" if out != "f8" and rng.random() < 0.4 else "apply"
        case = dict(op=op, mode=mode, rows=_spread(rng, 1, max(1, (1 << 26) // width)), width=width, dtype=dtype,
                    residual=rng.choice(["bf16", "f32"]), out=out)
        if out == "f8":
            case["width"] = width = -(-width // 128) * 128
            case["group"] = rng.choice([0, 32, 64, 128])  # 0: one scale per row
            case["rows"] = min(case["rows"], max(1, (1 << 26) // width))
        return case
    mode = rng.choice(["prompt", "prompt", "step", "train"])
    channels = _spread(rng, 96, 4096)
    if mode == "step":
        batch, seq = _spread(rng, 1, 512), 1
    else:
        seq = _spread(rng, 1, 16384)
        most = (1 << 26) // 4 if mode == "train" else (1 << 26)
        if op == "scan":
            most //= 2
        batch = _spread(rng, 1, max(1, min(16, most // (seq * channels))))
    case = dict(op=op, mode=mode, batch=batch, seq=seq, channels=channels, dtype=dtype,
                ragged=mode != "step" and rng.random() < 0.4)
    if op == "conv":
        case["taps"] = rng.choice([2, 3, 4, 4])
    else:
        case["groups"] = rng.choice([1, 1, 2])
        case["channels"] = channels - channels % case["groups"]
        case["state"] = rng.choice([16, 16, 8, 24])
    return case


def _lengths(case):
    """The sequences' lengths in a padded batch: from a third of the longest up to it."""
    b, s = case["batch"], case["seq"]
    return [s if b == 1 else max(1, s // 3 + (s - s // 3) * i // (b - 1)) for i in range(b)]


def _tokens(case):
    return sum(_lengths(case)) if case["ragged"] else case["batch"] * case["seq"]


def work(case):
    size = {"bf16": 2, "f32": 4, "f8": 1}
    e = size[case["dtype"]]
    if case["op"] == "norm":
        n, r, o = case["rows"] * case["width"], size[case["residual"]], size[case["out"]]
        nbytes, flops = n * (e + 2 * r + o) + 4 * case["width"], 6 * n
        if case["out"] == "f8":
            nbytes += 4 * n // (case["group"] or case["width"])
            flops += 3 * n
        if case["mode"] == "train":  # d_y, d_r and r in, d_x and d_residual out
            nbytes, flops = nbytes + n * (o + 2 * r + r + e) + 8 * case["width"], flops + 12 * n
        return {"bytes": nbytes, "flops": flops}
    m = _tokens(case)  # sequence positions that are computed
    pad = case["batch"] * case["seq"] - m  # written as zeros
    c = case["channels"]
    if case["op"] == "conv":
        k = case["taps"]
        window = 8 * case["batch"] * c * k
        nbytes, flops = (2 * m + pad) * c * e + window + 4 * c * (k + 1), m * c * (2 * k + 5)
        if case["mode"] == "train":
            nbytes, flops = nbytes + (3 * m + pad) * c * e + 8 * c * (k + 1), flops + m * c * (6 * k + 10)
        return {"bytes": nbytes, "flops": flops}
    n = case["state"]
    bc = 2 * m * case["groups"] * n * e
    states = 8 * case["batch"] * c * n
    nbytes, flops = (4 * m + pad) * c * e + bc + states + 4 * c * (n + 2), m * c * (7 * n + 16)
    if case["mode"] == "train":
        nbytes += (7 * m + 3 * pad) * c * e + 2 * bc + states + 8 * c * (n + 2)
        flops += m * c * (15 * n + 30)
    return {"bytes": nbytes, "flops": flops}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    f32 = torch.float32

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, device="cuda", generator=g) * (hi - lo) + lo

    s = dict(case=case)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        rd = DTYPES[case["residual"]]
        s.update(x=normal(rows, width), residual=normal(rows, width, scale=3.0, dtype=rd), weight=uniform(width, lo=0.5, hi=1.5))
        if case["mode"] == "train":
            s.update(d_y=normal(rows, width, dtype=DTYPES[case["out"]]), d_r=normal(rows, width, dtype=rd))
        return s
    b, t, c = case["batch"], case["seq"], case["channels"]
    step = case["mode"] == "step"
    lead = (b,) if step else (b, t)
    s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None
    if case["op"] == "conv":
        k = case["taps"]
        s.update(x=normal(*lead, c), weight=normal(c, k, scale=k ** -0.5, dtype=f32), bias=normal(c, scale=0.2, dtype=f32),
                 window=normal(b, c, k, dtype=f32))
        if case["mode"] == "train":
            s.update(d_y=normal(*lead, c))
        return s
    n, gr = case["state"], case["groups"]
    # the step sizes softplus(dt + dt_bias) spread over [0.001, 0.1] as at a model's initialisation; a of real parts -1 .. -state
    step0 = torch.exp(uniform(c, lo=-6.9, hi=-2.3))
    a = -torch.arange(1, n + 1, device="cuda", dtype=f32) * uniform(c, n, lo=0.8, hi=1.25)
    # z is the second half of the input projection, b and c slices of the projection that makes them: views with longer rows
    zz, bcs = normal(*lead, 2 * c), normal(*lead, 8 + 2 * gr * n)
    s.update(u=normal(*lead, c), dt=normal(*lead, c, scale=0.5), a=a, b=bcs[..., 8:8 + gr * n].unflatten(-1, (gr, n)),
             c=bcs[..., 8 + gr * n:].unflatten(-1, (gr, n)), d=uniform(c, lo=0.5, hi=1.5), z=zz[..., c:],
             dt_bias=step0 + torch.log(-torch.expm1(-step0)), state=normal(b, c, n, scale=0.3, dtype=f32))
    if case["mode"] == "train":
        s.update(d_y=normal(*lead, c), d_state=normal(b, c, n, scale=0.3, dtype=f32))
    return s


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    dn = importlib.import_module("burn-deltanet_b200")
    case = s["case"]
    mode = case["mode"]
    if case["op"] == "norm":
        if case["out"] == "f8":
            q, scale, r = dn.add_rms_norm_f8(s["x"], s["weight"], s["residual"], EPS, group=case["group"])
            return dict(q=q, scale=scale, r=r)
        y, r = dn.add_rms_norm(s["x"], s["weight"], s["residual"], EPS, out_dtype=DTYPES[case["out"]])
        if mode == "apply":
            return dict(y=y, r=r)
        d_x, d_residual, d_weight = dn.add_rms_norm_backward(s["d_y"], s["d_r"], r, s["weight"], EPS, x_dtype=s["x"].dtype)
        return dict(y=y, r=r, d_x=d_x, d_residual=d_residual, d_weight=d_weight)
    if case["op"] == "conv":
        if mode == "step":
            y, window = dn.causal_conv_step(s["x"], s["weight"], s["bias"], s["window"], window_out=s["window"])
            return dict(y=y, window=window)
        y, window = dn.causal_conv(s["x"], s["weight"], s["bias"], s["window"], lengths=s["lengths"])
        if mode == "prompt":
            return dict(y=y, window=window)
        d_x, d_weight, d_bias, d_window = dn.causal_conv_backward(s["d_y"], None, s["x"], s["weight"], s["bias"], s["window"],
                                                                  lengths=s["lengths"])
        return dict(y=y, window=window, d_x=d_x, d_weight=d_weight, d_bias=d_bias, d_window=d_window)
    args = [s[k] for k in ("u", "dt", "a", "b", "c", "d", "z", "dt_bias", "state")]
    if mode == "step":
        y, h = dn.selective_scan_step(*args, state_out=s["state"])
        return dict(y=y, state=h)
    if mode == "prompt":
        y, h = dn.selective_scan(*args, lengths=s["lengths"])
        return dict(y=y, state=h)
    y, h, saved = dn.selective_scan(*args, lengths=s["lengths"], checkpoints=True)
    grads = dn.selective_scan_backward(s["d_y"], s["d_state"], *args, lengths=s["lengths"], checkpoints=saved)
    names = ("d_u", "d_dt", "d_a", "d_b", "d_c", "d_d", "d_z", "d_dt_bias", "d_state")
    return dict(zip(names, grads), y=y, state=h)


# ------------------------------------------------------------------------------------ the plain forms
def _plain_norm(s):
    case = s["case"]
    total = s["x"].float() + s["residual"].float()
    r = total.to(s["residual"].dtype)
    inv = torch.rsqrt(total.square().mean(-1, keepdim=True) + EPS)
    y = total * inv * s["weight"]
    if case["out"] == "f8":
        rows, width = y.shape
        parts = y.view(rows, -1, case["group"] or width)
        amax = parts.abs().amax(-1, keepdim=True)
        scale = torch.where(amax > 0, amax / F8_MAX, torch.ones_like(amax))
        return dict(q=(parts / scale).view(rows, width).to(torch.float8_e4m3fn), scale=scale.squeeze(-1), r=r)
    out = dict(y=y.to(DTYPES[case["out"]]), r=r)
    if case["mode"] == "train":  # through the sum as it was stored
        v = r.float()
        inv = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
        d_y = s["d_y"].float()
        wd = d_y * s["weight"]
        d = inv * wd - v * inv ** 3 * (wd * v).mean(-1, keepdim=True) + s["d_r"].float()
        out.update(d_x=d.to(s["x"].dtype), d_residual=d.to(r.dtype), d_weight=(d_y * v * inv).sum(0))
    return out


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _valid(s, t):
    """[batch, t, 1]: whether a position is inside its sequence."""
    return (torch.arange(t, device="cuda") < s["lengths"][:, None])[..., None]


def _plain_conv(s):
    case, w, k = s["case"], s["weight"], s["case"]["taps"]
    x = s["x"].float()
    if case["mode"] == "step":
        window = torch.cat([s["window"][:, :, 1:], x[:, :, None]], -1)
        pre = (window * w).sum(-1) + s["bias"]
        s["window"].copy_(window)
        return dict(y=(pre * _sigmoid(pre)).to(s["x"].dtype), window=s["window"])
    t = x.shape[1]
    if case["ragged"]:
        valid = _valid(s, t)
        x = torch.where(valid, x, 0.0)
    padded = torch.cat([s["window"].transpose(1, 2), x], 1)  # row i: token i - k
    pre = s["bias"] + sum(w[:, j] * padded[:, j + 1:j + 1 + t] for j in range(k))
    sig = _sigmoid(pre)
    y = pre * sig
    last = s["lengths"].long() if case["ragged"] else torch.full((case["batch"],), t, device="cuda")
    at = last[:, None] + torch.arange(k, device="cuda")
    window = torch.gather(padded, 1, at[..., None].expand(-1, -1, x.shape[2])).transpose(1, 2).contiguous()
    if case["ragged"]:
        y = torch.where(valid, y, 0.0)
    out = dict(y=y.to(s["x"].dtype), window=window)
    if case["mode"] == "train":
        d_pre = s["d_y"].float() * sig * (1.0 + pre * (1.0 - sig))
        if case["ragged"]:
            d_pre = torch.where(valid, d_pre, 0.0)
        d_padded = torch.zeros_like(padded)
        d_w = []
        for j in range(k):
            d_padded[:, j + 1:j + 1 + t] += w[:, j] * d_pre
            d_w.append((d_pre * padded[:, j + 1:j + 1 + t]).sum((0, 1)))
        out.update(d_x=d_padded[:, k:].to(s["x"].dtype), d_weight=torch.stack(d_w, -1), d_bias=d_pre.sum((0, 1)),
                   d_window=d_padded[:, :k].transpose(1, 2).contiguous())
    return out


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-torch.abs(x)))


def _doubling(decay, add, h):
    """h_t = decay_t h_{t-1} + add_t over axis 1, from h: the segments' maps joined pair by pair. Overwrites its arguments."""
    add[:, 0] += decay[:, 0] * h
    step, t = 1, add.shape[1]
    while step < t:
        add[:, step:] += decay[:, step:] * add[:, :-step]
        decay[:, step:] *= decay[:, :-step].clone()
        step *= 2
    return add


def _plain_scan(s):
    case, a = s["case"], s["a"]
    u, b, c, z = (s[k].float() for k in ("u", "b", "c", "z"))
    raw = s["dt"].float() + s["dt_bias"]
    dt = _softplus(raw)
    per = case["channels"] // case["groups"]
    b, c = (v.repeat_interleave(per, dim=-2) for v in (b, c))  # [.., channels, state]
    sig = _sigmoid(z)
    gate = z * sig
    if case["mode"] == "step":
        h = torch.exp(dt[..., None] * a) * s["state"] + (dt * u)[..., None] * b
        y = ((h * c).sum(-1) + s["d"] * u) * gate
        s["state"].copy_(h)
        return dict(y=y.to(s["u"].dtype), state=s["state"])
    t = u.shape[1]
    if case["ragged"]:
        valid = _valid(s, t)
        dt, u = torch.where(valid, dt, 0.0), torch.where(valid, u, 0.0)
    decay = torch.exp(dt[..., None] * a)
    h = _doubling(decay.clone(), (dt * u)[..., None] * b, s["state"])
    read = (h * c).sum(-1) + s["d"] * u
    y = read * gate
    if case["ragged"]:
        y = torch.where(valid, y, 0.0)
    out = dict(y=y.to(s["u"].dtype), state=h[:, -1].clone())
    if case["mode"] == "prompt":
        return out
    d_y = s["d_y"].float()
    if case["ragged"]:
        d_y = torch.where(valid, d_y, 0.0)
    d_z = d_y * read * sig * (1.0 + z * (1.0 - sig))
    d_read = d_y * gate
    # g_t = d_read_t c_t + decay_{t+1} g_{t+1}, from the last token back
    d_h = d_read[..., None] * c
    back = torch.cat([torch.ones_like(decay[:, :1]), decay.flip(1)[:, :-1]], 1)
    g = _doubling(back, d_h.flip(1), s["d_state"]).flip(1)
    before = torch.cat([s["state"][:, None], h[:, :-1]], 1)  # h_{t-1}
    gb = (g * b).sum(-1)
    w = g * decay * before
    d_dt = gb * u + (w * a).sum(-1)
    d_raw = d_dt * _sigmoid(raw)
    if case["ragged"]:
        d_raw = torch.where(valid, d_raw, 0.0)
    lead = u.shape[:2]
    d_b = (g * (dt * u)[..., None]).view(*lead, case["groups"], per, -1).sum(3)
    d_c = (h * d_read[..., None]).view(*lead, case["groups"], per, -1).sum(3)
    kind = s["u"].dtype
    out.update(d_u=(gb * dt + d_read * s["d"]).to(kind), d_dt=d_raw.to(kind), d_a=(w * dt[..., None]).sum((0, 1)), d_b=d_b.to(kind),
               d_c=d_c.to(kind), d_d=(d_read * u).sum((0, 1)), d_z=d_z.to(kind), d_dt_bias=d_raw.sum((0, 1)),
               d_state=(g[:, 0] * decay[:, 0]))
    return out


# ------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](case, s)


def _exact_norm(case, s):
    r = s["x"] + s["residual"]
    rms = torch.sqrt((r * r).mean(1) + EPS)
    y = r / rms[:, None] * s["weight"]
    if case["out"] == "f8":
        groups = y.unflatten(1, (-1, case["group"] or case["width"]))
        scale = groups.abs().amax(2) / F8_MAX
        scale[scale == 0] = 1.0
        return dict(q=(groups / scale[..., None]).flatten(1), scale=scale, r=r)
    if case["mode"] == "apply":
        return dict(y=y, r=r)
    v = r.to(DTYPES[case["residual"]]).double().requires_grad_()  # the sum as it is stored
    weight = s["weight"].requires_grad_()
    out = v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS) * weight
    d_v, d_weight = torch.autograd.grad([out, v], [v, weight], [s["d_y"], s["d_r"]])
    return dict(y=y, r=r, d_x=d_v, d_residual=d_v, d_weight=d_weight)


def _exact_conv(case, s):
    b, t, k, c = case["batch"], case["seq"], case["taps"], case["channels"]
    train = case["mode"] == "train"
    x = s["x"].view(b, t, c)
    leaves = [v.requires_grad_(train) for v in (x, s["weight"], s["bias"], s["window"])]
    lengths = _lengths(case) if case["ragged"] else [t] * b
    ys, windows = [], []
    for i, n in enumerate(lengths):
        line = torch.cat([s["window"][i].T, x[i, :n]])  # [k + n, c]
        pre = (line[1:].unfold(0, k, 1) * s["weight"]).sum(-1) + s["bias"]
        ys.append(torch.cat([pre * torch.sigmoid(pre), torch.zeros(t - n, c, device="cuda", dtype=torch.float64)]))
        windows.append(line[n:].T)
    y, window = torch.stack(ys), torch.stack(windows)
    if not train:
        return dict(y=y.view(s["x"].shape), window=window)
    grads = torch.autograd.grad(y, leaves, s["d_y"])
    return dict(zip(("d_x", "d_weight", "d_bias", "d_window"), grads), y=y.detach(), window=window.detach())


def _exact_scan(case, s):
    b, t, c, n = case["batch"], case["seq"], case["channels"], case["state"]
    if b * t * c * n > 1 << 30 or (case["mode"] == "train" and b * t * c * n > 1 << 29):
        return None  # the states of every token would not fit, or take too long
    u, z, raw = s["u"].view(b, t, c), s["z"].reshape(b, t, c), (s["dt"] + s["dt_bias"]).view(b, t, c)
    per = c // case["groups"]
    bb, cc = s["b"].reshape(b, t, -1, n), s["c"].reshape(b, t, -1, n)
    lengths = torch.tensor(_lengths(case) if case["ragged"] else [t] * b, device="cuda")
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    train = case["mode"] == "train"
    h, y, states = s["state"].clone(), torch.zeros_like(u), []
    for i in range(t):
        live = (i < lengths).double()[:, None]
        step = dt[:, i] * live
        states.append(h if train else None)
        h = h * torch.exp(step[..., None] * s["a"]) + (step * u[:, i])[..., None] * bb[:, i].repeat_interleave(per, 1)
        y[:, i] = ((h * cc[:, i].repeat_interleave(per, 1)).sum(-1) + s["d"] * u[:, i]) * live
    out = dict(y=(y * z * torch.sigmoid(z)).view(s["u"].shape), state=h)
    if not train:
        return out
    grads = {k: torch.zeros_like(v) for k, v in dict(d_u=u, d_dt=u, d_a=s["a"], d_b=bb, d_c=cc, d_d=s["d"], d_z=u, d_dt_bias=s["d"]).items()}
    g = s["d_state"].clone()
    after = h
    for i in reversed(range(t)):
        live = (i < lengths).double()[:, None]
        step, before = dt[:, i] * live, states.pop()
        sig = torch.sigmoid(z[:, i])
        d_out = s["d_y"][:, i] * live
        grads["d_z"][:, i] = d_out * y[:, i] * (sig + z[:, i] * sig * (1 - sig))
        d_read = d_out * z[:, i] * sig
        g = g + d_read[..., None] * cc[:, i].repeat_interleave(per, 1)
        grads["d_c"][:, i] = (after * d_read[..., None]).view(b, -1, per, n).sum(2)
        grads["d_b"][:, i] = (g * (step * u[:, i])[..., None]).view(b, -1, per, n).sum(2)
        through = (g * bb[:, i].repeat_interleave(per, 1)).sum(-1)
        decay = torch.exp(step[..., None] * s["a"])
        moved = g * decay * before
        d_step = (through * u[:, i] + (moved * s["a"]).sum(-1)) * live * torch.sigmoid(raw[:, i])
        grads["d_dt"][:, i] = d_step
        grads["d_dt_bias"] += d_step.sum(0)
        grads["d_u"][:, i] = through * step + d_read * s["d"]
        grads["d_d"] += (d_read * u[:, i]).sum(0)
        grads["d_a"] += (moved * step[..., None]).sum(0)
        g, after = g * decay, before
    return dict(grads, **out, d_state=g)
