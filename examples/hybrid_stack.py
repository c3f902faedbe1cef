"""A small hybrid stack: gated delta-rule mixers and selective-scan mixers in turn, on one residual stream.

    python examples/hybrid_stack.py

Each layer is add_rms_norm -> input projection -> mixer -> output projection, whose result the next layer's norm adds to the
stream.  Serving runs the norm into 8 bits with one scale per row and the input projection as an 8-bit matrix product; a prompt
goes through the chunked prefill, the convolution and the scan, single tokens through their steps on the states that the prompt
left.  Training runs the scan mixer through the autograd nodes.  The script checks that a prompt followed by single tokens
gives what the whole sequence gives, and trains a one-layer model for a few steps.
"""
import importlib
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
dn = importlib.import_module("burn-deltanet_b200")

EPS = 1e-5
TAPS = 4


def randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


class Linear8:
    """y = x W^T with x in e4m3 and one scale per row, W in e4m3 and one scale per output."""

    def __init__(self, weight):
        w = weight.float()
        self.scale = (w.abs().amax(1, keepdim=True) / 448.0).clamp_min(1e-12)
        self.w = (w / self.scale).to(torch.float8_e4m3fn)

    def __call__(self, q, scale):
        lead = q.shape[:-1]
        q, scale = q.flatten(0, -2), scale.flatten(0, -2)
        y = torch._scaled_mm(q, self.w.t(), scale_a=scale, scale_b=self.scale.t().contiguous(), out_dtype=torch.bfloat16)
        return y.unflatten(0, lead)


class DeltaMixer:
    """A gated delta rule of `heads` heads of 64: convolution and norms, gates, the prefill or the tick, the output norm."""

    def __init__(self, g, width, heads=4):
        self.h, self.dk = heads, 64
        c = 3 * heads * self.dk
        self.c = c
        self.in_proj = randn(g, c + 2 * heads, width, scale=width ** -0.5)
        self.conv = randn(g, c, TAPS, scale=0.5, dtype=torch.float32)
        self.dt_bias, self.a_log = randn(g, heads, dtype=torch.float32), randn(g, heads, scale=0.3, dtype=torch.float32)
        self.norm = torch.ones(self.dk, device="cuda")
        self.out_proj = randn(g, width, heads * self.dk, scale=(heads * self.dk) ** -0.5)

    def cache(self, batch):
        return dict(window=torch.zeros(batch, self.c, TAPS, device="cuda"), state=torch.zeros(batch, self.h, self.dk, self.dk, device="cuda"))

    def __call__(self, xz, cache):
        q, k, v, cache["window"] = dn.qkv_prologue(xz, self.h, self.dk, self.dk, self.conv, None, cache["window"])
        beta = dn.write_gate(xz[..., self.c:self.c + self.h]).unsqueeze(-1)
        decay = dn.head_log_decay(xz[..., self.c + self.h:self.c + 2 * self.h], self.dt_bias, self.a_log).unsqueeze(-1)
        scale = self.dk ** -0.5
        if xz.shape[1] > 1:
            y, cache["state"] = dn.delta_chunk_recalculated(q, k, v, beta, beta, decay, cache["state"], True, 64, scale)
        else:
            one = lambda t: t[:, 0]
            y, _ = dn.delta_step(one(q), one(k), one(v), one(beta), one(beta), one(decay), cache["state"], scale, state_out=cache["state"])
            y = y.unsqueeze(1)
        return dn.out_norm(y, None, self.norm).flatten(2) @ self.out_proj.t()


class ScanMixer:
    """A selective state space scan over `channels` channels: convolution, the projections that make the steps, b and c, the
    scan or its step, gated by the input projection's second half."""

    def __init__(self, g, width, channels=256, state=16, rank=16):
        self.channels, self.n, self.rank = channels, state, rank
        self.in_proj = randn(g, 2 * channels, width, scale=width ** -0.5)
        self.conv, self.conv_bias = randn(g, channels, TAPS, scale=0.5, dtype=torch.float32), randn(g, channels, scale=0.1, dtype=torch.float32)
        self.x_proj = randn(g, rank + 2 * state, channels, scale=channels ** -0.5)
        self.dt_proj = randn(g, channels, rank, scale=rank ** -0.5)
        step = torch.exp(torch.rand(channels, device="cuda", generator=g) * 4.6 - 6.9)
        self.dt_bias = step + torch.log(-torch.expm1(-step))  # softplus gives the step back
        self.a_log = torch.log(torch.arange(1, state + 1, device="cuda", dtype=torch.float32)).repeat(channels, 1)
        self.d = torch.ones(channels, device="cuda")
        self.out_proj = randn(g, width, channels, scale=channels ** -0.5)

    def cache(self, batch):
        return dict(window=torch.zeros(batch, self.channels, TAPS, device="cuda"), state=torch.zeros(batch, self.channels, self.n, device="cuda"))

    def __call__(self, xz, cache):
        x, z = xz[..., :self.channels], xz[..., self.channels:]
        a = -torch.exp(self.a_log)
        if xz.shape[1] > 1:
            u, cache["window"] = dn.causal_conv(x, self.conv, self.conv_bias, cache["window"])
            dbc = u @ self.x_proj.t()
            dt = dbc[..., :self.rank] @ self.dt_proj.t()
            b, c = dbc[..., self.rank:self.rank + self.n], dbc[..., self.rank + self.n:]
            y, cache["state"] = dn.selective_scan(u, dt, a, b, c, self.d, z, self.dt_bias, cache["state"])
        else:
            u, _ = dn.causal_conv_step(x[:, 0], self.conv, self.conv_bias, cache["window"], window_out=cache["window"])
            dbc = u @ self.x_proj.t()
            dt = dbc[..., :self.rank] @ self.dt_proj.t()
            b, c = dbc[..., self.rank:self.rank + self.n], dbc[..., self.rank + self.n:]
            y, _ = dn.selective_scan_step(u, dt, a, b, c, self.d, z[:, 0], self.dt_bias, cache["state"], state_out=cache["state"])
            y = y.unsqueeze(1)
        return y @ self.out_proj.t()

    def train(self, xz, a_log):
        """The same over whole sequences from zero, through the autograd nodes."""
        x, z = xz[..., :self.channels], xz[..., self.channels:]
        u, _ = dn.CausalConvFunction.apply(x, self.conv, self.conv_bias)
        dbc = u @ self.x_proj.t()
        dt = dbc[..., :self.rank] @ self.dt_proj.t()
        b, c = dbc[..., self.rank:self.rank + self.n], dbc[..., self.rank + self.n:]
        y, _ = dn.SelectiveScanFunction.apply(u, dt, -torch.exp(a_log), b, c, self.d, z, self.dt_bias)
        return y @ self.out_proj.t()


class HybridStack:
    """Layers in turn, for serving: 8-bit input projections, the residual stream in float32."""

    def __init__(self, width=256, layers=4, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.mixers = [DeltaMixer(g, width) if i % 2 == 0 else ScanMixer(g, width) for i in range(layers)]
        # the 8-bit product wants its sizes in multiples of 16
        pad = lambda w: torch.nn.functional.pad(w, (0, 0, 0, -w.shape[0] % 16))
        self.in_projs = [Linear8(pad(m.in_proj)) for m in self.mixers]
        self.norms = [torch.ones(width, device="cuda") for _ in range(layers + 1)]

    def caches(self, batch):
        return [m.cache(batch) for m in self.mixers]

    def __call__(self, x, caches):
        """x [batch, tokens, width] (one token or a prompt) to the normalised stream; the caches move on."""
        stream = None
        for mixer, proj, norm, cache in zip(self.mixers, self.in_projs, self.norms, caches):
            q, scale, stream = dn.add_rms_norm_f8(x, norm, stream, EPS, residual_dtype=torch.float32)
            x = mixer(proj(q, scale), cache)
        return dn.add_rms_norm(x, self.norms[-1], stream, EPS)[0]


def serve(batch=16, prompt=96, tokens=8, width=256):
    """The largest difference, over the typical size, between a prompt followed by single tokens and the whole sequence."""
    stack = HybridStack(width)
    x = randn(torch.Generator(device="cuda").manual_seed(1), batch, prompt + tokens, width)
    whole = stack(x, stack.caches(batch))
    caches = stack.caches(batch)
    parts = [stack(x[:, :prompt].contiguous(), caches)]
    for t in range(prompt, prompt + tokens):
        parts.append(stack(x[:, t:t + 1].contiguous(), caches))
    got = torch.cat(parts, 1)
    return float((got.float() - whole.float()).abs().max() / whole.float().square().mean().sqrt())


def train(steps=12, batch=4, tokens=64, width=128):
    """The losses of a norm and a scan mixer that learn to give each token's predecessor."""
    g = torch.Generator(device="cuda").manual_seed(2)
    mixer = ScanMixer(g, width, channels=256)
    norm, a_log = torch.ones(width, device="cuda"), mixer.a_log.clone()
    params = [norm, a_log, mixer.in_proj, mixer.conv, mixer.conv_bias, mixer.x_proj, mixer.dt_proj, mixer.dt_bias, mixer.d, mixer.out_proj]
    params = [p.requires_grad_() for p in params]
    opt = torch.optim.Adam(params, lr=1e-2)
    x = randn(g, batch, tokens, width)
    target = torch.cat([torch.zeros_like(x[:, :1]), x[:, :-1]], 1).float()
    losses = []
    for _ in range(steps):
        h = dn.AddRmsNormFunction.apply(x, norm, None, EPS)
        loss = (mixer.train(h @ mixer.in_proj.t(), a_log).float() - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert all(math.isfinite(v) for v in losses)
    return losses


if __name__ == "__main__":
    print(f"prompt + single tokens against the whole sequence: {serve():.4f} of the typical size")
    losses = train()
    print("training loss: " + " ".join(f"{v:.3f}" for v in losses))
