"""The C entries of the grouped products without offsets: one expert has all rows, as with offsets 0, T."""

import ctypes as C

import pytest
import torch

from cppmega_mlx_amd import _lib
from cppmega_mlx_amd.nn.grouped_gemm import grouped_fp8_gemm, grouped_gemm, grouped_gemm_bwd
from tests.test_gpu_gated_ffn import BF16, F16, F32, _normal, _offsets

pytestmark = pytest.mark.gpu


def _args(op, x, w, y, n, k, **over):
    a = _lib.GroupedGemmArgs()
    a.struct_size, a.op = C.sizeof(a), op
    a.x, a.w, a.y, a.offsets = x.data_ptr(), w.data_ptr(), y.data_ptr(), None
    a.x_dtype, a.y_dtype, a.offsets_dtype = _lib.dtype_code(x), _lib.dtype_code(y), _lib.I32
    a.rows, a.experts, a.n, a.k, a.zero_tail = x.shape[0], 1, n, k, 1
    a.x_pitch, a.y_pitch, a.w_pitch = x.shape[1], y.shape[1], w.shape[-1]
    for name, value in over.items():
        setattr(a, name, value)
    return a


def _run(a, x, other=None):
    stream = _lib.current_stream(x.device)
    if other is None:
        rc = _lib.load().cppmega_mi355_grouped_gemm(C.byref(a), C.sizeof(a), stream)
    else:
        rc = _lib.load().cppmega_mi355_grouped_gemm_bwd(C.byref(a), C.byref(other), C.sizeof(a), stream)
    _lib.check(rc, "grouped_gemm")


# one row, few rows (weights streamed), small and large tiles, rows that do not begin on 16 bytes, a contraction without rows
@pytest.mark.parametrize("rows, n, k", [(1, 64, 128), (13, 100, 72), (200, 130, 264), (2100, 1300, 1024), (150, 33, 65)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_expert_without_offsets(device, rows, n, k, dtype):
    x, w, dy = _normal(device, rows, k, dtype=dtype, seed=1), _normal(device, 1, n, k, dtype=dtype, seed=2), _normal(device, rows, n, dtype=dtype, seed=3)
    off = _offsets([rows], device)
    y, dx, dw = torch.full((rows, n), 7.0, dtype=dtype, device=device), torch.full((rows, k), 7.0, dtype=dtype, device=device), torch.full((n, k), 7.0, device=device)
    _run(_args(_lib.GROUPED_ROWS, x, w, y, n, k), x)
    assert torch.equal(y, grouped_gemm(x, w, off))
    wide = torch.empty(1, n, k, device=device)
    want = grouped_gemm_bwd(dy, x, w, off, dw=wide)
    ops = _args(_lib.GROUPED_ROWS_GRAD, dy, w, dx, n, k), _args(_lib.GROUPED_WEIGHTS_GRAD, dy, x, dw, n, k)
    _run(*ops[:1], x, ops[1])
    assert torch.equal(dx, want[0]) and torch.equal(dw, wide[0])
    for a, t, of in ((ops[0], dx, lambda: grouped_gemm_bwd(dy, x, w, off, need_dw=False)[0]),
                     (ops[1], dw, lambda: grouped_gemm_bwd(dy, x, w, off, dw=wide, need_dx=False)[1][0])):
        t.fill_(7.0)
        _run(a, x)
        assert torch.equal(t, of())


@pytest.mark.parametrize("rows, n, k", [(3, 100, 384), (300, 256, 272), (70, 33, 129)])
def test_one_expert_without_offsets_in_e4m3(device, rows, n, k):
    x, w = (_normal(device, *s, seed=i).to(torch.float8_e4m3fn).view(torch.uint8) for i, s in enumerate(((rows, k), (1, n, k))))
    xs, ws = torch.exp(_normal(device, rows, seed=3)), torch.exp(_normal(device, 1, (n + 127) // 128, (k + 127) // 128, seed=4))
    for dtype in (BF16, F32):
        y = torch.full((rows, n), 7.0, dtype=dtype, device=device)
        _run(_args(_lib.GROUPED_ROWS, x, w, y, n, k, x_scale=xs.data_ptr(), w_scale=ws.data_ptr()), x)
        want = grouped_fp8_gemm(x, xs, w, ws, _offsets([rows], device), out=torch.empty_like(y))
        assert torch.equal(y, want)
