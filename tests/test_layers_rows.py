"""The overlap checks of the block-level operators without a GPU: csrc/rows.hpp against a byte-by-byte evaluation, and the
refusals through the C entry points, which come before anything touches a device."""
import ctypes
import importlib
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
abi = importlib.import_module("burn-deltanet_b200._abi")

SOURCE = r"""
#include "rows.hpp"
using dc::host::Rows;
extern "C" int meet(const int64_t *x, const int64_t *y) {
    return dc::host::rows_meet(Rows{(void *)x[0], x[1], x[2], x[3], x[4], x[5]}, Rows{(void *)y[0], y[1], y[2], y[3], y[4], y[5]});
}
extern "C" int fold(const int64_t *x) { return dc::host::rows_fold(Rows{(void *)x[0], x[1], x[2], x[3], x[4], x[5]}); }
"""


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    at = tmp_path_factory.mktemp("rows")
    (at / "rows.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O2", "-shared", "-fPIC", "-std=c++17", "-I", os.path.join(ROOT, "burn-deltanet_b200", "csrc"),
                    str(at / "rows.cpp"), "-o", str(at / "rows.so")], check=True)
    lib = ctypes.CDLL(str(at / "rows.so"))
    six = ctypes.c_int64 * 6
    return (lambda x, y: bool(lib.meet(six(*x), six(*y)))), (lambda x: bool(lib.fold(six(*x))))


def bytes_of(r):
    """Every row's bytes, by row."""
    p, batch, seq, bs, ts, width = r
    return [range(p + b * bs + t * ts, p + b * bs + t * ts + width) for b in range(batch) for t in range(seq)]


def some_rows(rng, like=None):
    width = rng.randint(1, 5)
    if like is not None and rng.random() < 0.6:  # the same strides, another place: slices of one buffer
        return (like[0] + rng.randint(-12, 12), like[1], like[2], like[3], like[4], width)
    return (1000 + rng.randint(-40, 40), rng.randint(1, 4), rng.randint(1, 4), rng.randint(0, 24), width + rng.randint(0, 12), width)


def test_against_every_byte(rows):
    meet, fold = rows
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(20000):
        x = some_rows(rng)
        y = some_rows(rng, x)
        bx, by = (set().union(*bytes_of(r)) for r in (x, y))
        assert meet(x, y) == meet(y, x) == bool(bx & by), (x, y)
        assert fold(x) == (sum(map(len, bytes_of(x))) != len(bx)), x
        seen[bool(bx & by)] += 1
    assert min(seen.values()) > 2000


def test_large_layouts(rows):
    """Slices of a projection, transposed layouts, token slices, and strides whose products pass 64 bits."""
    meet, fold = rows
    p, b, t, c = 1 << 40, 8, 4096, 4096
    whole = lambda at, width: (p + at, b, t, t * c, c, width)
    assert not meet(whole(0, 2048), whole(2048, 2048)) and meet(whole(0, 2048), whole(2047, 2048)) and meet(whole(0, 2049), whole(2048, 2048))
    assert not meet(whole(2048, 2048), whole(0, 2048)) and not fold(whole(0, c)) and fold(whole(0, c + 1))
    turned = lambda at, width: (p + at, b, t, c, b * c, width)
    assert not fold(turned(0, c)) and not meet(turned(0, 100), turned(100, 100)) and meet(turned(0, 100), turned(99, 100))
    assert not meet(whole(0, 2048), turned(2048, 2048)) and meet(whole(0, 2048), turned(2047, 2048)) and meet(whole(0, 1), turned(c * b, 1))
    halves = lambda at: (p + at, b, t // 2, t * c, c, c)  # the first or the second half of the tokens
    assert not meet(halves(0), halves(t // 2 * c)) and meet(halves(0), halves((t // 2 - 1) * c))
    one = lambda at: (p + at, 256, 1, 2 * c, 0, c)
    assert not meet(one(0), one(c)) and meet(one(0), one(c - 1)) and not fold(one(0))
    assert not meet((p, 2, 2, 1 << 62, 1 << 61, 8), (p + 8, 2, 2, 1 << 62, 1 << 61, 8)) and not fold((p, 1 << 31, 1 << 31, 1 << 62, 64, 64))
    assert not meet((0, 2, 2, 8, 8, 8), (p, 2, 2, 8, 8, 8)) and not fold((p, 0, 2, 0, 0, 8)) and fold((p, 2, 1, 0, 8, 8))


P = 0x10000000  # addresses that are never read: every call below is refused


def conv(bwd=False, **over):
    a = abi.CausalConvBwdArgs() if bwd else abi.CausalConvArgs()
    a.batch, a.seq, a.channels, a.taps = 2, 6, 32, 4
    for f, _ in a._fields_:
        if f.endswith("_batch_stride"):
            setattr(a, f, 192)
        elif f.endswith("_token_stride"):
            setattr(a, f, 32)
    for i, f in enumerate(f for f, t in a._fields_ if t is ctypes.c_void_p and f != "lengths"):
        setattr(a, f, P + i * 0x100000)
    if bwd:
        a.workspace_bytes = 1 << 20
    for k, v in over.items():
        setattr(a, k, v)
    return a


# sequences on top of each other: all of them, by a token, by a channel
@pytest.mark.parametrize("stride", [0, 32, 160, 31, 191])
def test_conv_refuses_outputs_that_fold(stride):
    assert abi.lib().dc_causal_conv(conv(y_batch_stride=stride), None) == abi.DC_EINVAL_SHAPE
    assert abi.lib().dc_causal_conv_bwd(conv(True, d_x_batch_stride=stride), None) == abi.DC_EINVAL_SHAPE


def test_conv_step_refuses_outputs_that_fold():
    for stride in (0, 31):
        assert abi.lib().dc_causal_conv(conv(seq=1, y_batch_stride=stride), None) == abi.DC_EINVAL_SHAPE


def test_conv_refuses_outputs_over_inputs():
    x = conv().x
    for at in (4, 124, 192 * 4, (192 + 5 * 32) * 4, -4, -124):
        assert abi.lib().dc_causal_conv(conv(y=x + at), None) == abi.DC_EINVAL_ARG
    a = conv(True)
    for buffer in (a.x, a.d_y):
        for at in (0, 4, 124, -124, (192 + 5 * 32) * 4 + 4):
            assert abi.lib().dc_causal_conv_bwd(conv(True, d_x=buffer + at), None) == abi.DC_EINVAL_ARG


def test_conv_bwd_refuses_windows_over_windows():
    a = conv(True)
    for buffer in (a.d_window_out, a.window_in):
        for at in (0, 16, -16, 2 * 32 * 4 * 4 - 4):
            assert abi.lib().dc_causal_conv_bwd(conv(True, d_window_in=buffer + at), None) == abi.DC_EINVAL_ARG


def scan(**over):
    """Inputs 1 MB apart; y, state_out and checkpoints behind them."""
    a = abi.SelectiveScanArgs()
    a.batch, a.seq, a.channels, a.state, a.groups = 2, 6, 32, 16, 2
    for f, _ in a._fields_:
        if f.endswith("_batch_stride"):
            setattr(a, f, 192)
        elif f.endswith("_token_stride"):
            setattr(a, f, 32)
    for i, f in enumerate(f for f, t in a._fields_ if t is ctypes.c_void_p and f not in ("lengths", "workspace")):
        setattr(a, f, P + i * 0x100000)
    for k, v in over.items():
        setattr(a, k, v)
    return a


LAST = (192 + 5 * 32) * 4  # of a tensor's rows


@pytest.mark.parametrize("name", ["u", "dt", "z", "b", "c"])
def test_scan_refuses_outputs_over_inputs(name):
    at = getattr(scan(), name)
    for off in (0, 4, 124, -4, -124, LAST, LAST + 124):
        assert abi.lib().dc_selective_scan(scan(y=at + off), None) == abi.DC_EINVAL_ARG
    for off in (0, 4, 124, -124, 192 * 4 + 4):
        assert abi.lib().dc_selective_scan_step(scan(seq=1, y=at + off), None) == abi.DC_EINVAL_ARG


@pytest.mark.parametrize("name,size", [("a", 32 * 16 * 4), ("d", 128), ("dt_bias", 128), ("state_in", 2 * 32 * 16 * 4)])
def test_scan_refuses_outputs_over_parameters_and_state(name, size):
    at = getattr(scan(), name)
    for off in (0, size - 4, -LAST - 124):
        assert abi.lib().dc_selective_scan(scan(y=at + off), None) == abi.DC_EINVAL_ARG


def test_scan_refuses_outputs_that_fold():
    for over in (dict(y_batch_stride=160), dict(y_batch_stride=32), dict(y_batch_stride=191)):
        assert abi.lib().dc_selective_scan(scan(**over), None) == abi.DC_EINVAL_SHAPE


def test_scan_refuses_states_that_meet():
    size = 2 * 32 * 16 * 4
    for off in (4, -4, size - 4, 4 - size):  # (the very same buffer is in place)
        for call, seq in ((abi.lib().dc_selective_scan, 6), (abi.lib().dc_selective_scan_step, 1)):
            assert call(scan(seq=seq, state_out=scan().state_in + off), None) == abi.DC_EINVAL_ARG
    assert abi.lib().dc_selective_scan(scan(state_out=scan().y + 64), None) == abi.DC_EINVAL_ARG


def test_scan_bwd_refuses_outputs_over_inputs():
    def call(**over):
        w = abi.SelectiveScanBwdArgs()
        w.fwd = scan()
        w.d_y_batch_stride, w.d_y_token_stride = 192, 32
        for i, f in enumerate(f for f, t in w._fields_ if t is ctypes.c_void_p):
            setattr(w, f, P + 0x2000000 + i * 0x100000)
        w.workspace_bytes = 1 << 24
        d_y, d_state = w.d_y, w.d_state_out
        for k, v in over.items():
            setattr(w, k, v(w))
        return abi.lib().dc_selective_scan_bwd(w, None)

    for out in ("d_u", "d_dt", "d_z"):
        for name in ("u", "dt", "z", "b", "c"):
            for off in (0, 4, -4, LAST + 124):
                assert call(**{out: lambda w: getattr(w.fwd, name) + off}) == abi.DC_EINVAL_ARG
        assert call(**{out: lambda w: w.d_y + 64}) == abi.DC_EINVAL_ARG
    for off in (0, 4, -4):
        assert call(d_state_in=lambda w: w.d_state_out + off) == abi.DC_EINVAL_ARG


def norm(bwd=False, **over):
    a = abi.RmsNormBwdArgs() if bwd else abi.RmsNormArgs()
    a.rows, a.width, a.eps = 4, 128, 1e-5
    for f, _ in a._fields_:
        if f.endswith("_stride"):
            setattr(a, f, 200)
    for i, f in enumerate(f for f, t in a._fields_ if t is ctypes.c_void_p):
        setattr(a, f, P + i * 0x100000)
    if bwd:
        a.workspace_bytes = 1 << 24
    for k, v in over.items():
        setattr(a, k, v)
    return a


END = (3 * 200 + 127) * 4  # a row buffer's last element


@pytest.mark.parametrize("out", ["y", "residual_out"])
def test_norm_refuses_outputs_that_meet_others(out):
    others = ["x", "residual_in", "y" if out == "residual_out" else "residual_out"]
    for other in others:
        at = getattr(norm(), other)
        for off in (4, -4, 127 * 4, -127 * 4, END, 200 * 4 + 4):
            assert abi.lib().dc_rms_norm(norm(**{out: at + off}), None) == abi.DC_EINVAL_ARG
        # a whole row further is no in-place call either
        assert abi.lib().dc_rms_norm(norm(**{out: at + 800}), None) == abi.DC_EINVAL_ARG
    at = norm().weight
    for off in (0, 127 * 4, -END):
        assert abi.lib().dc_rms_norm(norm(**{out: at + off}), None) == abi.DC_EINVAL_ARG


def test_norm_refuses_scales_that_meet_others():
    for other in ("x", "residual_in", "residual_out", "y"):
        for off in (0, 4, 127 * 4 if other != "y" else 124):
            a = norm(out_dtype=abi.DC_E4M3, group=32, scale=getattr(norm(), other) + off)
            assert abi.lib().dc_rms_norm(a, None) == abi.DC_EINVAL_ARG


@pytest.mark.parametrize("out", ["d_x", "d_residual"])
def test_norm_bwd_refuses_outputs_that_meet_others(out):
    for other in ("d_y", "d_r", "r", "d_residual" if out == "d_x" else "d_x"):
        at = getattr(norm(True), other)
        for off in (4, -4, 127 * 4, END, 800):
            assert abi.lib().dc_rms_norm_bwd(norm(True, **{out: at + off}), None) == abi.DC_EINVAL_ARG
    at = norm(True).weight
    assert abi.lib().dc_rms_norm_bwd(norm(True, **{out: at + 4}), None) == abi.DC_EINVAL_ARG
