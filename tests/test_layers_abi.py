"""The C ABI of the operators around the token mixers (include/deltacore_layers.h) without a GPU: exported symbols, struct
layouts, the Rust mirror, and the refusals, which come before anything touches a device."""
import ctypes
import importlib
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "deltacore_layers.h")).read()
RUST = open(os.path.join(ROOT, "burn-deltanet_b200", "rust", "deltacore-sys", "src", "layers.rs")).read()
abi = importlib.import_module("burn-deltanet_b200._abi")
STRUCTS = {"dc_rms_norm_args": abi.RmsNormArgs, "dc_rms_norm_bwd_args": abi.RmsNormBwdArgs, "dc_causal_conv_args": abi.CausalConvArgs,
           "dc_causal_conv_bwd_args": abi.CausalConvBwdArgs, "dc_selective_scan_args": abi.SelectiveScanArgs,
           "dc_selective_scan_bwd_args": abi.SelectiveScanBwdArgs}


def functions():
    return re.findall(r"DC_API \w+ (dc_\w+)\(", HEADER)


def fields():
    """{struct: [(field, C type)]} of the header."""
    out = {}
    for body, name in re.findall(r"typedef struct \w+ \{(.*?)\} (\w+);", HEADER, re.S):
        out[name] = []
        for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
            m = re.match(r"((?:const )?\w+)\s*(.*)", decl.strip(), re.S)
            for n in m.group(2).split(",") if m else ():
                n, ty = n.strip(), m.group(1)
                while n.startswith("*"):
                    n, ty = n[1:].strip(), ty + " *"
                out[name].append((n, ty))
    return out


def test_symbols():
    lib = abi.lib()
    assert len(functions()) == 12 and set(functions()) <= set(abi.EXPORTS)
    for name in functions():
        assert hasattr(lib, name)


def test_struct_layouts(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    assert set(fields()) == set(STRUCTS)
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "deltacore_layers.h"', "int main(void) {"]
    for st, names in fields().items():
        lines.append(f'printf("{st} sizeof %zu\\n", sizeof({st}));')
        lines += [f'printf("{st} {n} %zu\\n", offsetof({st}, {n}));' for n, _ in names]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    want = {tuple(l.split()[:2]): int(l.split()[2]) for l in out if l}
    for st, cls in STRUCTS.items():
        assert [n for n, _ in cls._fields_] == [n for n, _ in fields()[st]]
        assert want[(st, "sizeof")] == ctypes.sizeof(cls)
        for n, _ in cls._fields_:
            assert want[(st, n)] == getattr(cls, n).offset, (st, n)


def test_the_rust_mirror():
    rust = {"int64_t": "i64", "int32_t": "i32", "uint32_t": "u32", "uint64_t": "u64", "float": "f32", "const void *": "*const c_void",
            "void *": "*mut c_void", "const float *": "*const f32", "float *": "*mut f32", "const int32_t *": "*const i32",
            "dc_selective_scan_args": "dc_selective_scan_args"}
    got = {name: [(n, t) for n, t in re.findall(r"pub (\w+): ([^,]+),", body)]
           for name, body in re.findall(r"pub struct (\w+) \{(.*?)\n\}", RUST, re.S)}
    assert got == {name: [(n, rust[t]) for n, t in fs] for name, fs in fields().items()}
    consts = dict(re.findall(r"pub const (\w+): \w+ = ([^;]+);", RUST))
    for name, val in re.findall(r"#define (DC_\w+) (0x[0-9a-f]+|\d+)u?", HEADER):
        assert int(consts[name], 0) == int(val, 0) == getattr(abi, name), name
    assert set(re.findall(r"pub fn (dc_\w+)\(", RUST)) == set(functions())
    lib = os.path.join(ROOT, "burn-deltanet_b200", "rust", "deltacore-sys", "src", "lib.rs")
    assert "pub mod layers;" in open(lib).read()


P = 0x10000  # addresses that are never read: every call below is refused


def norm(**over):
    a = abi.RmsNormArgs()
    a.rows, a.width = 4, 128
    a.x_stride = a.residual_in_stride = a.residual_out_stride = a.y_stride = 128
    a.eps = 1e-5
    a.x, a.residual_in, a.weight, a.residual_out, a.y, a.scale = P, P + 0x10000, P + 0x20000, P + 0x30000, P + 0x40000, P + 0x50000
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(rows=-1), abi.DC_EINVAL_SHAPE), (dict(width=0), abi.DC_EINVAL_SHAPE), (dict(width=16385), abi.DC_EUNSUPPORTED),
    (dict(x_dtype=2), abi.DC_EUNSUPPORTED_DTYPE), (dict(out_dtype=3), abi.DC_EUNSUPPORTED_DTYPE), (dict(residual_dtype=2), abi.DC_EUNSUPPORTED_DTYPE),
    (dict(eps=-1.0), abi.DC_EINVAL_ARG), (dict(eps=float("nan")), abi.DC_EINVAL_ARG), (dict(group=128), abi.DC_EINVAL_ARG),
    (dict(out_dtype=abi.DC_E4M3, group=48), abi.DC_EINVAL_WIDTH), (dict(out_dtype=abi.DC_E4M3, group=256), abi.DC_EINVAL_SHAPE),
    (dict(out_dtype=abi.DC_E4M3, scale=None), abi.DC_EINVAL_ARG), (dict(x=None), abi.DC_EINVAL_ARG), (dict(weight=None), abi.DC_EINVAL_ARG),
    (dict(y=None), abi.DC_EINVAL_ARG), (dict(x=P + 2), abi.DC_EINVAL_ARG), (dict(x_stride=127), abi.DC_EINVAL_SHAPE),
    (dict(residual_out_stride=100), abi.DC_EINVAL_SHAPE), (dict(y=P, out_dtype=abi.DC_BF16), abi.DC_EINVAL_ARG),
    (dict(y=P + 0x30000), abi.DC_EINVAL_ARG), (dict(residual_out=P, residual_out_stride=256), abi.DC_EINVAL_ARG),
    (dict(residual_out=P + 0x10000, residual_out_stride=256), abi.DC_EINVAL_ARG), (dict(y=P + 0x10000, y_stride=256), abi.DC_EINVAL_ARG),
])
def test_norm_refusals(over, status):
    assert abi.lib().dc_rms_norm(norm(**over), None) == status


def test_norm_without_rows_is_done():
    assert abi.lib().dc_rms_norm(norm(rows=0), None) == abi.DC_OK
    assert abi.lib().dc_rms_norm(None, None) == abi.DC_EINVAL_ARG


def norm_bwd(**over):
    a = abi.RmsNormBwdArgs()
    a.rows, a.width, a.eps = 4, 128, 1e-5
    a.d_y_stride = a.d_r_stride = a.r_stride = a.d_x_stride = a.d_residual_stride = 128
    a.d_y, a.d_r, a.r, a.weight, a.d_x, a.d_residual, a.d_weight = (P + i * 0x10000 for i in range(7))
    a.workspace, a.workspace_bytes = P + 0x80000, 1 << 20
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(width=0), abi.DC_EINVAL_SHAPE), (dict(width=20000), abi.DC_EUNSUPPORTED), (dict(y_dtype=2), abi.DC_EUNSUPPORTED_DTYPE),
    (dict(x_dtype=2), abi.DC_EUNSUPPORTED_DTYPE), (dict(d_y=None), abi.DC_EINVAL_ARG), (dict(r=None), abi.DC_EINVAL_ARG),
    (dict(d_r_stride=1), abi.DC_EINVAL_SHAPE), (dict(d_x=P + 0x50000), abi.DC_EINVAL_ARG), (dict(d_residual=P + 0x20000), abi.DC_EINVAL_ARG),
    (dict(workspace_bytes=16), abi.DC_EWORKSPACE), (dict(workspace=None), abi.DC_EINVAL_ARG), (dict(workspace=P + 8), abi.DC_EINVAL_ARG),
])
def test_norm_bwd_refusals(over, status):
    assert abi.lib().dc_rms_norm_bwd(norm_bwd(**over), None) == status


def conv(cls=abi.CausalConvArgs, **over):
    a = cls()
    a.batch, a.seq, a.channels, a.taps = 2, 6, 32, 4
    for f, _ in cls._fields_:
        if f.endswith("_batch_stride"):
            setattr(a, f, 192)
        elif f.endswith("_token_stride"):
            setattr(a, f, 32)
    names = [f for f, t in cls._fields_ if t is ctypes.c_void_p and f != "lengths"]
    for i, f in enumerate(names):
        setattr(a, f, P + i * 0x10000)
    if cls is abi.CausalConvBwdArgs:
        a.workspace_bytes = 1 << 20
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(batch=-1), abi.DC_EINVAL_SHAPE), (dict(taps=0), abi.DC_EINVAL_ARG), (dict(taps=9), abi.DC_EUNSUPPORTED),
    (dict(in_dtype=2), abi.DC_EUNSUPPORTED_DTYPE), (dict(flags=2), abi.DC_EINVAL_ARG), (dict(x=None), abi.DC_EINVAL_ARG),
    (dict(weight=None), abi.DC_EINVAL_ARG), (dict(x=P + 1), abi.DC_EINVAL_ARG), (dict(x_token_stride=31), abi.DC_EINVAL_SHAPE),
    (dict(y=P), abi.DC_EINVAL_ARG), (dict(y=P + 128), abi.DC_EINVAL_ARG),
    (dict(window_in=P + 0x60000, window_out=P + 0x60000), abi.DC_EINVAL_ARG), (dict(window_in=P + 0x60000, window_out=P + 0x60010), abi.DC_EINVAL_ARG),
    (dict(seq=1, window_in=P + 0x60000, window_out=P + 0x60010), abi.DC_EINVAL_ARG),
])
def test_conv_refusals(over, status):
    assert abi.lib().dc_causal_conv(conv(**over), None) == status


@pytest.mark.parametrize("over,status", [
    (dict(seq=-1), abi.DC_EINVAL_SHAPE), (dict(taps=9), abi.DC_EUNSUPPORTED), (dict(d_weight=None), abi.DC_EINVAL_ARG),
    (dict(d_x=None), abi.DC_EINVAL_ARG), (dict(d_y_token_stride=3), abi.DC_EINVAL_SHAPE), (dict(workspace_bytes=8), abi.DC_EWORKSPACE),
    (dict(workspace=None), abi.DC_EINVAL_ARG),
])
def test_conv_bwd_refusals(over, status):
    assert abi.lib().dc_causal_conv_bwd(conv(abi.CausalConvBwdArgs, **over), None) == status


def scan(**over):
    a = abi.SelectiveScanArgs()
    a.batch, a.seq, a.channels, a.state, a.groups = 2, 6, 32, 16, 2
    for f, _ in a._fields_:
        if f.endswith("_batch_stride"):
            setattr(a, f, 192)
        elif f.endswith("_token_stride"):
            setattr(a, f, 32)
    for i, f in enumerate(f for f, t in a._fields_ if t is ctypes.c_void_p and f not in ("lengths", "workspace")):
        setattr(a, f, P + i * 0x10000)
    for k, v in over.items():
        setattr(a, k, v)
    return a


SCAN_REFUSALS = [
    (dict(batch=-1), abi.DC_EINVAL_SHAPE), (dict(state=0), abi.DC_EINVAL_SHAPE), (dict(state=65), abi.DC_EUNSUPPORTED),
    (dict(groups=3), abi.DC_EINVAL_SHAPE), (dict(groups=0), abi.DC_EINVAL_SHAPE), (dict(in_dtype=2), abi.DC_EUNSUPPORTED_DTYPE),
    (dict(out_dtype=-1), abi.DC_EUNSUPPORTED_DTYPE), (dict(flags=4), abi.DC_EINVAL_ARG), (dict(u=None), abi.DC_EINVAL_ARG),
    (dict(a=None), abi.DC_EINVAL_ARG), (dict(b=P + 2), abi.DC_EINVAL_ARG), (dict(state_in=P + 2), abi.DC_EINVAL_ARG),
]


@pytest.mark.parametrize("over,status", SCAN_REFUSALS + [
    (dict(y=None), abi.DC_EINVAL_ARG), (dict(y=P), abi.DC_EINVAL_ARG), (dict(b_token_stride=31), abi.DC_EINVAL_SHAPE),
    (dict(z_batch_stride=5), abi.DC_EINVAL_SHAPE), (dict(y_token_stride=5), abi.DC_EINVAL_SHAPE),
])
def test_scan_refusals(over, status):
    assert abi.lib().dc_selective_scan(scan(**over), None) == status


@pytest.mark.parametrize("over,status", [({**dict(seq=1), **o}, s) for o, s in SCAN_REFUSALS] + [(dict(seq=2), abi.DC_EINVAL_SHAPE), (dict(seq=1, y=None), abi.DC_EINVAL_ARG)])
def test_scan_step_refusals(over, status):
    assert abi.lib().dc_selective_scan_step(scan(**over), None) == status


@pytest.mark.parametrize("over,bwd,status", [(o, {}, s) for o, s in SCAN_REFUSALS] + [
    (dict(checkpoints=None), {}, abi.DC_EINVAL_ARG), ({}, dict(d_u=None), abi.DC_EINVAL_ARG), ({}, dict(d_z=None), abi.DC_EINVAL_ARG),
    ({}, dict(d_a=None), abi.DC_EINVAL_ARG), ({}, dict(d_u=P), abi.DC_EINVAL_ARG), ({}, dict(d_y_token_stride=3), abi.DC_EINVAL_SHAPE),
    ({}, dict(workspace_bytes=64), abi.DC_EWORKSPACE), ({}, dict(workspace=None), abi.DC_EINVAL_ARG),
])
def test_scan_bwd_refusals(over, bwd, status):
    w = abi.SelectiveScanBwdArgs()
    w.fwd = scan(**over)
    w.d_y_batch_stride, w.d_y_token_stride = 192, 32
    for i, f in enumerate(f for f, t in w._fields_ if t is ctypes.c_void_p):
        setattr(w, f, P + 0x200000 + i * 0x10000)
    w.workspace_bytes = 1 << 24
    for k, v in bwd.items():
        setattr(w, k, v)
    assert abi.lib().dc_selective_scan_bwd(w, None) == status


def test_sizes():
    L = abi.lib()
    tile = {4: 16, 8: 16, 16: 16, 32: 16, 64: 16}  # tokens between checkpoints by state
    for n, t in tile.items():
        for seq in (0, 1, t, t + 1, 1000):
            assert L.dc_selective_scan_checkpoint_size(scan(state=n, seq=seq)) == 2 * -(-seq // t) * 32 * n * 4
    assert L.dc_selective_scan_checkpoint_size(scan(state=65)) == 0
    assert L.dc_rms_norm_bwd_workspace_size(norm_bwd(d_weight=None)) == 0
    assert L.dc_rms_norm_bwd_workspace_size(norm_bwd()) >= 128 * 4


def test_python_layer_refuses_before_the_library():
    """Placement and shapes are checked on the host: CPU tensors are an error, not another path."""
    import torch

    dn = importlib.import_module("burn-deltanet_b200")
    x = torch.zeros(2, 3, 8)
    for call in (lambda: dn.add_rms_norm(x, torch.ones(8)), lambda: dn.add_rms_norm_f8(x, torch.ones(8)),
                 lambda: dn.add_rms_norm_backward(x, None, x, torch.ones(8)), lambda: dn.causal_conv(x, torch.ones(8, 4)),
                 lambda: dn.causal_conv_backward(x, None, x, torch.ones(8, 4)), lambda: dn.selective_scan(x, x, x, x, x),
                 lambda: dn.selective_scan_step(x[0], x[0], x, x, x), lambda: dn.selective_scan_backward(x, None, x, x, x, x, x)):
        with pytest.raises(dn.DeltaCoreError):
            call()
