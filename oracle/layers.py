"""float64 restatements of the operators around the token mixers (include/deltacore_layers.h), token by token.

rms_norm / rms_norm_backward, causal_conv / causal_conv_backward, selective_scan / selective_scan_backward, and the nearest
e4m3 value.  numpy arrays in and out; the shapes are the C ABI's.
"""
from __future__ import annotations

import numpy as np


def rms_norm(x, residual, weight, eps):
    """(y, r): s = x + residual (None: 0), y = s / sqrt(mean(s^2) + eps) * weight."""
    r = x if residual is None else x + residual
    return r / np.sqrt((r * r).mean(-1, keepdims=True) + eps) * weight, r


def rms_norm_backward(d_y, d_r, r, weight, eps):
    """(d_r_in, d_weight) through y = r / sqrt(mean(r^2) + eps) * weight and r itself."""
    inv = 1 / np.sqrt((r * r).mean(-1, keepdims=True) + eps)
    g = d_y * weight
    d = inv * g - r * inv ** 3 * (g * r).mean(-1, keepdims=True)
    axes = tuple(range(r.ndim - 1))
    return d + (0 if d_r is None else d_r), (d_y * r * inv).sum(axes)


E4M3 = np.array([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)])[:-1]


def to_e4m3(v):
    """The nearest e4m3 value (ties to the even mantissa), saturating at 448."""
    a = np.minimum(np.abs(v), E4M3[-1])
    hi = np.clip(np.searchsorted(E4M3, a), 1, len(E4M3) - 1)
    lo = hi - 1
    up = (E4M3[hi] - a < a - E4M3[lo]) | ((E4M3[hi] - a == a - E4M3[lo]) & (hi % 2 == 0))
    return np.sign(v) * np.where(up, E4M3[hi], E4M3[lo])


def _sigmoid(x):
    return 0.5 * (1 + np.tanh(0.5 * x))


def _lengths(lengths, b, s):
    return np.full(b, s) if lengths is None else np.clip(np.asarray(lengths), 0, s)


def causal_conv(x, weight, bias=None, window=None, silu=True, lengths=None):
    """(y, next window) of x [B, S, C]."""
    b, s, c = x.shape
    k = weight.shape[1]
    y, nxt = np.zeros((b, s, c)), np.zeros((b, c, k))
    for i, n in enumerate(_lengths(lengths, b, s)):
        line = np.concatenate([np.zeros((k, c)) if window is None else window[i].T, x[i, :n]])
        for t in range(n):
            pre = (line[t + 1:t + 1 + k] * weight.T).sum(0) + (0 if bias is None else bias)
            y[i, t] = pre * _sigmoid(pre) if silu else pre
        nxt[i] = line[n:].T
    return y, nxt


def causal_conv_backward(d_y, d_next, x, weight, bias=None, window=None, silu=True, lengths=None):
    """(d_x, d_weight, d_bias, d_window)."""
    b, s, c = x.shape
    k = weight.shape[1]
    d_x, d_w, d_b, d_win = np.zeros((b, s, c)), np.zeros((c, k)), np.zeros(c), np.zeros((b, c, k))
    for i, n in enumerate(_lengths(lengths, b, s)):
        line = np.concatenate([np.zeros((k, c)) if window is None else window[i].T, x[i, :n]])
        d_line = np.zeros_like(line)
        for t in range(n):
            g = d_y[i, t]
            if silu:
                pre = (line[t + 1:t + 1 + k] * weight.T).sum(0) + (0 if bias is None else bias)
                sig = _sigmoid(pre)
                g = g * sig * (1 + pre * (1 - sig))
            d_line[t + 1:t + 1 + k] += g * weight.T
            d_w += (g * line[t + 1:t + 1 + k]).T
            d_b += g
        if d_next is not None:
            d_line[n:] += d_next[i].T
        d_x[i, :n], d_win[i] = d_line[k:], d_line[:k].T
    return d_x, d_w, d_b, d_win


def _spread(v, channels):
    """b or c of one token [B, G, N] to its channels [B, C, N]."""
    return np.repeat(v, channels // v.shape[1], axis=1)


def selective_scan(u, dt, a, b, c, d=None, z=None, dt_bias=None, state=None, softplus=True, lengths=None, keep=False):
    """(y, final state) of u [B, S, C], b and c [B, S, G, N]; with keep also every token's incoming state and step."""
    bs, s, ch = u.shape
    n = _lengths(lengths, bs, s)
    h = np.zeros((bs, ch, a.shape[1])) if state is None else state.copy()
    y, steps, before = np.zeros(u.shape), np.zeros(u.shape), []
    for t in range(s):
        live = (t < n)[:, None]
        raw = np.where(live, dt[:, t], 0) + (0 if dt_bias is None else dt_bias)
        step = np.where(live, np.logaddexp(0, raw) if softplus else raw, 0)
        ut, bt, ct = (np.where(live if v.ndim == 2 else live[..., None], v, 0) for v in (u[:, t], b[:, t], c[:, t]))
        if keep:
            before.append(h)
        steps[:, t] = step
        h = np.exp(step[..., None] * a) * h + (step * ut)[..., None] * _spread(bt, ch)
        read = (h * _spread(ct, ch)).sum(-1) + (0 if d is None else d * ut)
        if z is not None:
            zt = np.where(live, z[:, t], 0)
            read = read * zt * _sigmoid(zt)
        y[:, t] = np.where(live, read, 0)
    return (y, h, before, steps) if keep else (y, h)


def selective_scan_backward(d_y, d_state, u, dt, a, b, c, d=None, z=None, dt_bias=None, state=None, softplus=True, lengths=None,
                            sizes=False):
    """The gradients of <y, d_y> + <final state, d_state> as a dict by the input's name.  With `sizes`, on inputs without
    signs (all but a and dt), the sums of the magnitudes of each gradient's terms."""
    bs, s, ch = u.shape
    lens = _lengths(lengths, bs, s)
    _, h, before, steps = selective_scan(u, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, keep=True)
    groups, n = b.shape[2:]
    out = dict(u=np.zeros(u.shape), dt=np.zeros(u.shape), a=np.zeros(a.shape), b=np.zeros(b.shape), c=np.zeros(c.shape), d=np.zeros(ch),
               z=np.zeros(u.shape), dt_bias=np.zeros(ch))
    g = np.zeros((bs, ch, n)) if d_state is None else d_state.copy()
    for t in reversed(range(s)):
        live = (t < lens)[:, None]
        clean = lambda v: np.where(live if v.ndim == 2 else live[..., None], v, 0)
        step, ut, bt, ct, gy = steps[:, t], clean(u[:, t]), clean(b[:, t]), clean(c[:, t]), clean(d_y[:, t])
        skip = 0 if d is None else d * ut
        r = gy
        if z is not None:
            zt = clean(z[:, t])
            sig = _sigmoid(zt)
            out["z"][:, t] = gy * ((h * _spread(ct, ch)).sum(-1) + skip) * sig * (1 + zt * (1 - sig))
            r = gy * zt * sig
        g = g + r[..., None] * _spread(ct, ch)
        fold = lambda v: v.reshape(bs, groups, ch // groups, n).sum(2)
        out["c"][:, t] = fold(r[..., None] * h)
        out["b"][:, t] = fold((step * ut)[..., None] * g)
        through = (g * _spread(bt, ch)).sum(-1)
        decay = np.exp(step[..., None] * a)
        w = g * decay * before[t]
        d_step = through * ut + (w * (np.abs(a) if sizes else a)).sum(-1)
        raw = clean(dt[:, t]) + (0 if dt_bias is None else dt_bias)
        d_raw = np.where(live, d_step * (_sigmoid(raw) if softplus else 1), 0)
        out["u"][:, t] = through * step + r * (0 if d is None else d)
        out["dt"][:, t] = d_raw
        out["a"] += (w * step[..., None]).sum(0)
        out["d"] += (r * ut).sum(0)
        out["dt_bias"] += d_raw.sum(0)
        g, h = g * decay, before[t]
    out["state"] = g
    return out
