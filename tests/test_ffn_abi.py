"""The third header of the C ABI (feed-forward layer): symbols, struct layouts, and the refusals that come before any launch, at the C
boundary and in the Python entry points.  No GPU is touched."""

import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cppmega_mlx_amd import _lib
from cppmega_mlx_amd.nn import gated_ffn as gf, w4_gemm as w4

HEADER = Path(__file__).resolve().parents[1] / "include" / "cppmega_mi355_ffn.h"
STRUCTS = {
    "cppmega_mi355_gated_gemm_args_t": _lib.GatedGemmArgs,
    "cppmega_mi355_gated_gemm_bwd_args_t": _lib.GatedGemmBwdArgs,
    "cppmega_mi355_w4_gemm_args_t": _lib.W4GemmArgs,
}
FAKE = 0x1000     # never dereferenced: validation fails first


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = set(re.findall(r"\b(cppmega_mi355_[a-z0-9_]+)\s*\(", text))
    assert declared == set(_lib.FFN_SYMBOLS)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name), name
    assert f"GATED_MAX_OUTPUTS {_lib.GATED_MAX_OUTPUTS}" in text and f"W4_MAX_CHANNELS {_lib.W4_MAX_CHANNELS}" in text
    assert f"GATE_NONE = {_lib.GATE_NONE}" in text and f"GATE_SILU = {_lib.GATE_SILU}" in text and f"GATE_GELU_TANH = {_lib.GATE_GELU_TANH}" in text


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for ctype, struct in STRUCTS.items():
        lines.append(f'printf("{ctype} size %zu\\n", sizeof({ctype}));')
        lines += [f'printf("{ctype} {n} %zu\\n", offsetof({ctype}, {n}));' for n, _ in struct._fields_]
    lines.append("return 0;}")
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n")
    seen = 0
    for line in filter(None, out):
        ctype, name, value = line.split()
        struct = STRUCTS[ctype]
        assert (C.sizeof(struct) if name == "size" else getattr(struct, name).offset) == int(value), line
        seen += 1
    assert seen == sum(len(s._fields_) + 1 for s in STRUCTS.values())


def _call(a, fn, over):
    a.struct_size = C.sizeof(a)
    for k, v in over.items():
        setattr(a, k, v)
    return getattr(_lib.load(), fn)(C.byref(a), C.sizeof(a), None)


@pytest.mark.parametrize("over, code", [
    (dict(activation=2), _lib.ERR_SHAPE), (dict(activation=-1), _lib.ERR_SHAPE), (dict(n=0), _lib.ERR_SHAPE), (dict(n=_lib.GATED_MAX_OUTPUTS + 1), _lib.ERR_SHAPE),
    (dict(n=(1 << 31) - 1), _lib.ERR_SHAPE), (dict(k=0), _lib.ERR_SHAPE), (dict(k=_lib.GROUPED_MAX_SIZE + 1), _lib.ERR_SHAPE), (dict(rows=-1), _lib.ERR_SHAPE), (dict(rows=1 << 29), _lib.ERR_SHAPE),
    (dict(experts=0), _lib.ERR_SHAPE), (dict(experts=513), _lib.ERR_UNSUPPORTED), (dict(x_dtype=_lib.F32), _lib.ERR_DTYPE), (dict(y_dtype=_lib.F16), _lib.ERR_DTYPE),
    (dict(pre=FAKE, pre_dtype=_lib.F16), _lib.ERR_DTYPE), (dict(offsets_dtype=_lib.F32), _lib.ERR_DTYPE), (dict(offsets=None), _lib.ERR_NULL), (dict(x=None), _lib.ERR_NULL), (dict(y=None), _lib.ERR_NULL),
    (dict(w=None), _lib.ERR_NULL), (dict(x_dtype=_lib.E4M3), _lib.ERR_NULL), (dict(x_dtype=_lib.E4M3, pre=FAKE), _lib.ERR_DTYPE), (dict(x_dtype=_lib.E4M3, x_scale_block=64), _lib.ERR_SHAPE),
    (dict(struct_size=16), _lib.ERR_STRUCT_SIZE), (dict(rows=0), _lib.OK), (dict(rows=0, experts=1, offsets=None), _lib.OK)])
def test_gated_refusals(over, code):
    a = _lib.GatedGemmArgs()
    a.x = a.w = a.y = a.offsets = FAKE
    a.x_dtype = a.y_dtype = a.pre_dtype = _lib.BF16
    a.offsets_dtype = _lib.I32
    a.rows, a.experts, a.n, a.k, a.x_pitch, a.y_pitch, a.pre_pitch = 4, 2, 64, 64, 64, 64, 128
    assert _call(a, "cppmega_mi355_gated_gemm", over) == code


@pytest.mark.parametrize("over, code", [
    (dict(activation=2), _lib.ERR_SHAPE), (dict(n=0), _lib.ERR_SHAPE), (dict(n=_lib.GATED_MAX_OUTPUTS + 1), _lib.ERR_SHAPE), (dict(k=0), _lib.ERR_SHAPE), (dict(rows=-1), _lib.ERR_SHAPE),
    (dict(dtype=_lib.F32), _lib.ERR_DTYPE), (dict(pre_dtype=_lib.F16), _lib.ERR_DTYPE), (dict(dx_dtype=_lib.F16), _lib.ERR_DTYPE), (dict(dw_dtype=_lib.F16), _lib.ERR_DTYPE),
    (dict(offsets_dtype=_lib.F32), _lib.ERR_DTYPE), (dict(dy=None), _lib.ERR_NULL), (dict(pre=None), _lib.ERR_NULL), (dict(x=None), _lib.ERR_NULL), (dict(w=None), _lib.ERR_NULL),
    (dict(offsets=None), _lib.ERR_NULL), (dict(workspace=None), _lib.ERR_WORKSPACE), (dict(workspace_bytes=16), _lib.ERR_WORKSPACE), (dict(workspace=FAKE + 2), _lib.ERR_ALIGNMENT),
    (dict(experts=513), _lib.ERR_UNSUPPORTED), (dict(dx=None, dw=None), _lib.OK), (dict(rows=0, dw=None), _lib.OK)])
def test_gated_gradient_refusals(over, code):
    a = _lib.GatedGemmBwdArgs()
    a.dy = a.pre = a.x = a.w = a.dx = a.dw = a.offsets = a.workspace = FAKE
    a.dtype = a.pre_dtype = a.dx_dtype = a.dw_dtype = _lib.BF16
    a.offsets_dtype = _lib.I32
    a.rows, a.experts, a.n, a.k, a.dy_pitch, a.pre_pitch, a.x_pitch, a.dx_pitch, a.workspace_bytes = 4, 2, 63, 64, 63, 126, 64, 64, 1 << 20
    a.struct_size = C.sizeof(a)
    need = C.c_size_t(0)
    lib = _lib.load()
    assert lib.cppmega_mi355_gated_gemm_bwd_workspace_bytes(C.byref(a), C.sizeof(a), C.byref(need)) == _lib.OK and need.value == 4 * 128 * 2
    assert lib.cppmega_mi355_gated_gemm_bwd_workspace_bytes(C.byref(a), C.sizeof(a), None) == _lib.ERR_NULL
    assert _call(a, "cppmega_mi355_gated_gemm_bwd", over) == code


@pytest.mark.parametrize("over, code", [
    (dict(activation=2), _lib.ERR_SHAPE), (dict(activation=-2), _lib.ERR_SHAPE), (dict(n=0), _lib.ERR_SHAPE), (dict(n=_lib.GROUPED_MAX_SIZE + 1), _lib.ERR_SHAPE), (dict(activation=0, n=_lib.GATED_MAX_OUTPUTS + 1), _lib.ERR_SHAPE),
    (dict(k=0), _lib.ERR_SHAPE), (dict(k=96), _lib.ERR_SHAPE), (dict(k=_lib.W4_MAX_CHANNELS + 64), _lib.ERR_SHAPE), (dict(x_pitch=_lib.W4_MAX_CHANNELS + 1), _lib.ERR_SHAPE), (dict(x_pitch=-128), _lib.ERR_SHAPE), (dict(rows=-1), _lib.ERR_SHAPE), (dict(rows=1 << 29), _lib.ERR_SHAPE), (dict(group=16), _lib.ERR_SHAPE),
    (dict(group=256), _lib.ERR_SHAPE), (dict(experts=0), _lib.ERR_SHAPE), (dict(experts=513), _lib.ERR_UNSUPPORTED), (dict(x_dtype=_lib.F32), _lib.ERR_DTYPE), (dict(y_dtype=_lib.F16), _lib.ERR_DTYPE),
    (dict(scale_dtype=_lib.F16), _lib.ERR_DTYPE), (dict(offsets_dtype=_lib.F32), _lib.ERR_DTYPE), (dict(x=None), _lib.ERR_NULL), (dict(w=None), _lib.ERR_NULL), (dict(scale=None), _lib.ERR_NULL),
    (dict(y=None), _lib.ERR_NULL), (dict(offsets=None), _lib.ERR_NULL), (dict(struct_size=16), _lib.ERR_STRUCT_SIZE), (dict(rows=0), _lib.OK)])
def test_w4_refusals(over, code):
    a = _lib.W4GemmArgs()
    a.x = a.w = a.scale = a.y = a.offsets = FAKE
    a.x_dtype = a.y_dtype = a.scale_dtype = _lib.BF16
    a.activation, a.offsets_dtype = _lib.GATE_NONE, _lib.I32
    a.rows, a.experts, a.n, a.k, a.group, a.x_pitch, a.y_pitch = 4, 2, 64, 128, 64, 128, 64
    assert _call(a, "cppmega_mi355_w4_gemm", over) == code


@pytest.mark.parametrize("over", [
    dict(k=1 << 18, n=1 << 20), dict(k=1 << 18, n=1 << 20, dx=None), dict(k=(1 << 18) + 1, n=1 << 20), dict(k=1 << 20, n=33, rows=(1 << 29) - 1), dict(k=1 << 20, n=33, rows=(1 << 29) - 1, dw=None)],
    ids=lambda o: " ".join(f"{k}={v}" for k, v in o.items()))
def test_gradients_of_more_tiles_than_a_launch_has_are_refused_before_the_first_launch(over):
    """(Where no GPU is there, a launch that were tried would give the code of a failed one.)"""
    a = _lib.GatedGemmBwdArgs()
    a.dy = a.pre = a.x = a.w = a.dx = a.dw = a.workspace = FAKE
    a.dtype = a.pre_dtype = a.dx_dtype = a.dw_dtype = _lib.BF16
    a.offsets_dtype = _lib.I32
    a.rows, a.experts = 4, 1
    for k, v in over.items():
        setattr(a, k, v)
    a.dy_pitch, a.pre_pitch, a.x_pitch, a.dx_pitch, a.workspace_bytes = a.n, 2 * a.n, a.k, a.k, 1 << 62
    assert _call(a, "cppmega_mi355_gated_gemm_bwd", {}) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("n, k", [(1 << 21, 1 << 18), (1 << 21, (1 << 18) + 1), ((1 << 21) + 1, 1 << 18)])
def test_grouped_gradients_of_more_tiles_than_a_launch_has_are_refused_before_the_first_launch(n, k):
    rows, weights = _lib.GroupedGemmArgs(), _lib.GroupedGemmArgs()
    for a, op in ((rows, _lib.GROUPED_ROWS_GRAD), (weights, _lib.GROUPED_WEIGHTS_GRAD)):
        a.struct_size, a.op = C.sizeof(a), op
        a.x = a.w = a.y = a.offsets = FAKE
        a.x_dtype = a.y_dtype = _lib.BF16
        a.offsets_dtype = _lib.I32
        a.rows, a.experts, a.n, a.k = 4, 1, n, k
    rows.x_pitch, rows.y_pitch, weights.x_pitch, weights.w_pitch = n, k, n, k
    assert _lib.load().cppmega_mi355_grouped_gemm_bwd(C.byref(rows), C.byref(weights), C.sizeof(rows), None) == _lib.ERR_UNSUPPORTED


def _refused_by(fn, *args):
    assert getattr(_lib.load(), fn)(*args) not in (_lib.OK, _lib.ERR_LAUNCH)
    return _lib.load().cppmega_mi355_last_error().decode()


def test_a_refusal_names_the_call():
    """The gated block and the 4-bit products share checks with the grouped products: sizes, experts, tiles of a launch."""
    g = _lib.GatedGemmArgs()
    g.x = g.w = g.y = FAKE
    g.x_dtype = g.y_dtype = _lib.BF16
    g.offsets_dtype = _lib.I32
    for over in (dict(rows=-1), dict(experts=513, offsets=FAKE), dict(k=0), dict(x_dtype=_lib.F32), dict(y_dtype=_lib.F16), dict(x=None), dict(rows=(1 << 29) - 1, n=1 << 22)):
        a = _lib.GatedGemmArgs.from_buffer_copy(g)
        a.rows, a.experts, a.n, a.k, a.x_pitch, a.y_pitch, a.struct_size = 4, 1, 64, 64, 64, 64, C.sizeof(a)
        for k, v in over.items():
            setattr(a, k, v)
        assert _refused_by("cppmega_mi355_gated_gemm", C.byref(a), C.sizeof(a), None).startswith("gated_gemm: "), over
    b = _lib.GatedGemmBwdArgs()
    b.dy = b.pre = b.x = b.w = b.dx = b.dw = b.workspace = FAKE
    b.dtype = b.pre_dtype = b.dx_dtype = b.dw_dtype = _lib.BF16
    b.offsets_dtype = _lib.I32
    for over in (dict(rows=-1), dict(experts=513, offsets=FAKE), dict(k=0), dict(dx_dtype=_lib.F16), dict(w=None), dict(n=1 << 20, k=1 << 18), dict(rows=(1 << 29) - 1, n=1 << 20)):
        a = _lib.GatedGemmBwdArgs.from_buffer_copy(b)
        a.rows, a.experts, a.n, a.k, a.struct_size, a.workspace_bytes = 4, 1, 64, 64, C.sizeof(a), 1 << 62
        for k, v in over.items():
            setattr(a, k, v)
        a.dy_pitch, a.pre_pitch, a.x_pitch, a.dx_pitch = a.n, 2 * a.n, a.k, a.k
        assert _refused_by("cppmega_mi355_gated_gemm_bwd", C.byref(a), C.sizeof(a), None).startswith("gated_gemm_bwd: "), over
    w = _lib.W4GemmArgs()
    w.x = w.w = w.scale = w.y = FAKE
    w.x_dtype = w.y_dtype = w.scale_dtype = _lib.BF16
    w.activation, w.offsets_dtype = _lib.GATE_NONE, _lib.I32
    for n, k in ((1 << 30, 32), (1 << 30, 1024)):
        w.rows, w.experts, w.n, w.k, w.group, w.x_pitch, w.y_pitch, w.struct_size = 64, 1, n, k, 32, k, n, C.sizeof(w)
        assert _refused_by("cppmega_mi355_w4_gemm", C.byref(w), C.sizeof(w), None).startswith("w4_gemm: "), n
    r = _lib.GroupedGemmArgs()
    r.op, r.rows, r.struct_size = _lib.GROUPED_ROWS, -1, C.sizeof(r)
    assert _refused_by("cppmega_mi355_grouped_gemm", C.byref(r), C.sizeof(r), None).startswith("grouped_gemm: ")


@pytest.mark.parametrize("rows, n, gated", [(1, 1 << 29, False), (4, 1 << 28, True), (5, 1 << 30, False), (16, 1 << 29, True)])
def test_w4_outputs_that_one_launch_has_no_threads_for_are_refused(rows, n, gated):
    a = _lib.W4GemmArgs()
    a.x = a.w = a.scale = a.y = FAKE
    a.x_dtype = a.y_dtype = a.scale_dtype = _lib.BF16
    a.activation, a.offsets_dtype = _lib.GATE_SILU if gated else _lib.GATE_NONE, _lib.I32
    a.rows, a.experts, a.n, a.k, a.group, a.x_pitch, a.y_pitch = rows, 1, n, 32, 32, 32, n
    assert _call(a, "cppmega_mi355_w4_gemm", {}) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("rows", [1, 16])
def test_gated_outputs_that_one_launch_has_no_threads_for_are_refused(rows):
    a = _lib.GatedGemmArgs()
    a.x = a.w = a.y = FAKE
    a.x_dtype = a.y_dtype = _lib.BF16
    a.offsets_dtype = _lib.I32
    a.rows, a.experts, a.n, a.k, a.x_pitch, a.y_pitch = rows, 1, 1 << 29, 8, 8, 1 << 29
    assert _call(a, "cppmega_mi355_gated_gemm", {}) == _lib.ERR_UNSUPPORTED


def test_python_entry_points_refuse_host_tensors_and_bad_arguments():
    x, w, off = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    pre, dy, codes, scale = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, 4, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1, dtype=torch.bfloat16)
    for call in (lambda: gf.gated_gemm(x, w), lambda: gf.gated_gemm(x, w[None], off), lambda: gf.gated_gemm_bwd(dy, pre, x, w), lambda: gf.gated_gemm_apply(x, w),
                 lambda: gf.fp8_gated_gemm(x.to(torch.uint8), torch.ones(4), w.to(torch.uint8), torch.ones(2, 1, 1)), lambda: w4.w4_gemm(x, codes, scale),
                 lambda: w4.w4_gated_gemm(x, codes, scale), lambda: w4.w4_gemm(x, codes[None], scale[None], None, off)):
        with pytest.raises(_lib.NativeCallError, match="no CPU path"):
            call()
    for call in (lambda: gf.gated_gemm(x, w, activation="relu"), lambda: gf.gated_gemm_bwd(dy, pre, x, w, activation="relu"), lambda: w4.w4_gated_gemm(x, codes, scale, activation="relu")):
        with pytest.raises(ValueError, match="activation must be one of"):
            call()
    with pytest.raises(ValueError, match=r"w must be \[E, 2 F, K\]"):
        gf.gated_gemm(x, w, off)
    with pytest.raises(ValueError, match="w must be"):
        gf.gated_gemm(x, w[:7])
    with pytest.raises(ValueError, match="w must be"):
        w4.w4_gemm(x, codes, scale, None, off)
