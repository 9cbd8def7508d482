"""The second header of the C ABI (norm and grouped products): symbols, struct layouts, and the refusals that come before any
launch, at the C boundary and in the Python entry points.  No GPU is touched."""

import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cppmega_mlx_amd import _lib
from cppmega_mlx_amd.nn import grouped_gemm as gg, rms_norm as rn

HEADER = Path(__file__).resolve().parents[1] / "include" / "cppmega_mi355_layer.h"
STRUCTS = {
    "cppmega_mi355_rms_norm_args_t": _lib.RmsNormArgs,
    "cppmega_mi355_rms_norm_bwd_args_t": _lib.RmsNormBwdArgs,
    "cppmega_mi355_grouped_gemm_args_t": _lib.GroupedGemmArgs,
}
FAKE = 0x1000     # never dereferenced: validation fails first


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = set(re.findall(r"\b(cppmega_mi355_[a-z0-9_]+)\s*\(", text))
    assert declared == set(_lib.LAYER_SYMBOLS)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name), name
    assert f"NORM_MAX_WIDTH {_lib.NORM_MAX_WIDTH}" in text and f"GROUPED_MAX_EXPERTS {_lib.GROUPED_MAX_EXPERTS}" in text


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


def _norm(**over):
    a = _lib.RmsNormArgs()
    a.struct_size = C.sizeof(a)
    a.x = a.weight = a.out = a.scale = FAKE
    a.x_dtype = a.weight_dtype = a.out_dtype = _lib.BF16
    a.rows, a.width, a.eps = 4, 64, 1e-6
    for k, v in over.items():
        setattr(a, k, v)
    return _lib.load().cppmega_mi355_rms_norm(C.byref(a), C.sizeof(a), None)


@pytest.mark.parametrize("over, code", [
    (dict(width=0), _lib.ERR_SHAPE), (dict(width=_lib.NORM_MAX_WIDTH + 1), _lib.ERR_SHAPE), (dict(rows=-1), _lib.ERR_SHAPE),
    (dict(rows=1 << 31), _lib.ERR_SHAPE), (dict(x_dtype=_lib.E4M3), _lib.ERR_DTYPE), (dict(weight_dtype=_lib.F16), _lib.ERR_DTYPE),
    (dict(out_dtype=_lib.F32), _lib.ERR_DTYPE), (dict(out_dtype=_lib.E4M3, scale_block=64), _lib.ERR_SHAPE), (dict(eps=-1.0), _lib.ERR_SHAPE),
    (dict(eps=float("nan")), _lib.ERR_SHAPE), (dict(eps=float("inf")), _lib.ERR_SHAPE), (dict(x=None), _lib.ERR_NULL),
    (dict(out_dtype=_lib.E4M3, scale=None), _lib.ERR_NULL), (dict(residual_out=FAKE), _lib.ERR_NULL), (dict(struct_size=8), _lib.ERR_STRUCT_SIZE),
    (dict(rows=0), _lib.OK)])
def test_norm_refusals(over, code):
    assert _norm(**over) == code


@pytest.mark.parametrize("over, code", [
    (dict(width=0), _lib.ERR_SHAPE), (dict(rows=-1), _lib.ERR_SHAPE), (dict(dtype=_lib.I32), _lib.ERR_DTYPE),
    (dict(weight_dtype=_lib.F16), _lib.ERR_DTYPE), (dict(eps=-1.0), _lib.ERR_SHAPE), (dict(dweight=None), _lib.ERR_NULL), (dict(dy=None), _lib.ERR_NULL),
    (dict(workspace=None), _lib.ERR_WORKSPACE), (dict(workspace_bytes=16), _lib.ERR_WORKSPACE)])
def test_norm_gradient_refusals(over, code):
    a = _lib.RmsNormBwdArgs()
    a.struct_size = C.sizeof(a)
    a.dy = a.h = a.weight = a.dx = a.dweight = a.workspace = FAKE
    a.dtype = a.weight_dtype = _lib.BF16
    a.rows, a.width, a.eps, a.workspace_bytes = 4, 64, 1e-6, 1 << 20
    need = C.c_size_t(0)
    lib = _lib.load()
    assert lib.cppmega_mi355_rms_norm_bwd_workspace_bytes(C.byref(a), C.sizeof(a), C.byref(need)) == _lib.OK and need.value == 4 * 64 * 4
    assert lib.cppmega_mi355_rms_norm_bwd_workspace_bytes(C.byref(a), C.sizeof(a), None) == _lib.ERR_NULL
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.cppmega_mi355_rms_norm_bwd(C.byref(a), C.sizeof(a), None) == code


@pytest.mark.parametrize("over, code", [
    (dict(op=3), _lib.ERR_SHAPE), (dict(experts=0), _lib.ERR_SHAPE), (dict(experts=_lib.GROUPED_MAX_EXPERTS + 1), _lib.ERR_UNSUPPORTED), (dict(n=0), _lib.ERR_SHAPE),
    (dict(k=0), _lib.ERR_SHAPE), (dict(rows=-1), _lib.ERR_SHAPE), (dict(rows=1 << 29), _lib.ERR_SHAPE), (dict(x_dtype=_lib.F32), _lib.ERR_DTYPE), (dict(y_dtype=_lib.F16), _lib.ERR_DTYPE),
    (dict(offsets_dtype=_lib.F32), _lib.ERR_DTYPE), (dict(x_dtype=_lib.E4M3, op=1), _lib.ERR_DTYPE), (dict(x_dtype=_lib.E4M3, x_scale_block=64), _lib.ERR_SHAPE),
    (dict(x_dtype=_lib.E4M3), _lib.ERR_NULL), (dict(offsets=None), _lib.ERR_NULL), (dict(y=None), _lib.ERR_NULL), (dict(w=None), _lib.ERR_NULL),
    (dict(rows=0), _lib.OK), (dict(op=2, rows=0, y=None), _lib.ERR_NULL)])
def test_grouped_refusals(over, code):
    a = _lib.GroupedGemmArgs()
    a.struct_size = C.sizeof(a)
    a.x = a.w = a.y = a.offsets = FAKE
    a.x_dtype = a.y_dtype = _lib.BF16
    a.offsets_dtype = _lib.I32
    a.rows, a.experts, a.n, a.k, a.x_pitch, a.y_pitch = 4, 2, 64, 64, 64, 64
    for k, v in over.items():
        setattr(a, k, v)
    assert _lib.load().cppmega_mi355_grouped_gemm(C.byref(a), C.sizeof(a), None) == code


@pytest.mark.parametrize("rows, weights, code", [
    (dict(op=2), dict(), _lib.ERR_SHAPE), (dict(), dict(op=1), _lib.ERR_SHAPE), (dict(op=0), dict(), _lib.ERR_SHAPE), (dict(n=0), dict(), _lib.ERR_SHAPE),
    (dict(), dict(k=0), _lib.ERR_SHAPE), (dict(y=None), dict(), _lib.ERR_NULL), (dict(), dict(y=None), _lib.ERR_NULL), (dict(), dict(x_dtype=_lib.E4M3), _lib.ERR_DTYPE),
    (dict(struct_size=8), dict(), _lib.ERR_STRUCT_SIZE), (dict(), dict(struct_size=8), _lib.ERR_STRUCT_SIZE), (dict(rows=0), dict(rows=0, offsets=None), _lib.ERR_NULL)])
def test_both_gradients_refusals(rows, weights, code):
    """Both blocks are checked before either is launched."""
    blocks = []
    for op, over in ((1, rows), (2, weights)):
        a = _lib.GroupedGemmArgs()
        a.struct_size, a.op = C.sizeof(a), op
        a.x = a.w = a.y = a.offsets = FAKE
        a.x_dtype = a.y_dtype = _lib.BF16
        a.offsets_dtype = _lib.I32
        a.rows, a.experts, a.n, a.k, a.x_pitch, a.y_pitch, a.w_pitch = 4, 2, 64, 64, 64, 64, 64
        for k, v in over.items():
            setattr(a, k, v)
        blocks.append(a)
    assert _lib.load().cppmega_mi355_grouped_gemm_bwd(C.byref(blocks[0]), C.byref(blocks[1]), C.sizeof(blocks[0]), None) == code


def test_python_entry_points_refuse_host_tensors_and_bad_arguments():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    off = torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: rn.rms_norm(x, w), lambda: rn.rms_norm_fp8(x, w), lambda: rn.rms_norm_bwd(x, x, w), lambda: rn.rms_norm_apply(x, w),
                 lambda: gg.grouped_gemm(x, x.view(1, 4, 64), off), lambda: gg.grouped_gemm_bwd(torch.zeros(4, 4, dtype=torch.bfloat16), x, x.view(1, 4, 64), off),
                 lambda: gg.grouped_fp8_gemm(x.to(torch.uint8), torch.ones(4), x.to(torch.uint8).view(1, 4, 64), torch.ones(1, 1, 1), off)):
        with pytest.raises(_lib.NativeCallError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match=r"w must be \[E, N, K\]"):
        gg.grouped_gemm(x, x, off)
    with pytest.raises(ValueError, match="shape mismatch"):
        gg.grouped_gemm_bwd(x, x, x.view(1, 4, 64), off)
    with pytest.raises(TypeError, match="one type"):
        gg.grouped_gemm_bwd(torch.zeros(4, 4), x, x.view(1, 4, 64), off)
    with pytest.raises(TypeError, match="codes must be uint8"):
        rn.rms_norm_fp8(x, w, codes=x)


@pytest.mark.parametrize("make, want", [
    (lambda t: t, (24, 8)), (lambda t: t[:, 1:2], (4, 48)), (lambda t: t[0, 0], (1, 8)), (lambda t: t[:, :, :3], (24, 8)), (lambda t: t[0, ::2], (3, 16)),
    (lambda t: t[:1].expand(5, 6, 8)[:, :1], (5, 0)), (lambda t: t[:0], (0, 8))])
def test_row_pitch_of_views(make, want):
    assert _lib.row_pitch(make(torch.zeros(4, 6, 8)), "t") == want


@pytest.mark.parametrize("make, what", [
    (lambda t: t.transpose(1, 2), "last axis"), (lambda t: t[:, :3], "evenly spaced"), (lambda t: t[..., ::2], "last axis"), (lambda t: t.sum(), "at least one axis")])
def test_row_pitch_refuses_what_would_need_a_copy(make, what):
    with pytest.raises(ValueError, match=what):
        _lib.row_pitch(make(torch.zeros(4, 6, 8)), "t")


@pytest.mark.parametrize("op", [0, 1, 2])
@pytest.mark.parametrize("name", ["n", "k"])
def test_grouped_sizes_that_the_kernels_cannot_count_are_refused(op, name):
    """Column and contraction counters are 32 bits wide and run a tile past the end."""
    for size in ((1 << 31) - 1, (1 << 31) - 64, _lib.GROUPED_MAX_SIZE + 1):
        a = _lib.GroupedGemmArgs()
        a.struct_size, a.op = C.sizeof(a), op
        a.x = a.w = a.y = a.offsets = FAKE
        a.x_dtype = a.y_dtype = _lib.BF16
        a.offsets_dtype = _lib.I32
        a.rows, a.experts, a.n, a.k, a.x_pitch, a.y_pitch, a.w_pitch = 1, 1, 1, 1, 1, 1, 1
        setattr(a, name, size)
        assert _lib.load().cppmega_mi355_grouped_gemm(C.byref(a), C.sizeof(a), None) == _lib.ERR_SHAPE
