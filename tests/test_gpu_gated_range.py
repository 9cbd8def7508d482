"""The range of dg and du between the two launches of the gated block's gradients: what float16 does not hold there."""

import pytest
import torch

from cppmega_mlx_amd.nn.gated_ffn import gated_gemm_bwd
from tests.test_gpu_gated_ffn import BF16, F16, F32, _assert_within, _grads, _normal, _rounded

pytestmark = pytest.mark.gpu


# the kernel of any alignment, tiles
@pytest.mark.parametrize("rows, n, k", [(9, 5, 7), (700, 64, 128)])
def test_far_gradients(device, rows, n, k):
    """dg beyond 65504 in one row: infinities or NaN in that row of dx and those rows of dw in float16, the values in bfloat16."""
    for dtype in (BF16, F16):
        pre = torch.cat([_normal(device, rows, n, seed=1), _normal(device, rows, n, seed=2)], 1)
        dy, x, w = _normal(device, rows, n, dtype=dtype, seed=3), _normal(device, rows, k, dtype=dtype, seed=4), (_normal(device, 2 * n, k, seed=5) * 2.0 ** -10).to(dtype)
        at = rows - 2
        pre[at, 1], pre[at, n + 1], dy[at, 1] = 20.0, 200.0, 600.0  # (dg 120000, du 12000)
        dx, dw = gated_gemm_bwd(dy, pre, x, w)
        wx, ex, ww, ew = _grads(dy, pre, x, w, None, "silu")
        assert wx.abs().max() < 65504
        whole = torch.ones(rows, dtype=torch.bool, device=device)
        held = torch.ones(2 * n, dtype=torch.bool, device=device)
        if dtype == F16:
            whole[at], held[1] = False, False
            assert not torch.isfinite(dx[at]).any() and not torch.isfinite(dw[1]).any()
        _assert_within(dx[whole], wx[whole], _rounded(wx, ex, dtype)[whole])
        _assert_within(dw[held], ww[held], _rounded(ww, ew, dtype)[held])


@pytest.mark.parametrize("rows, n, k", [(9, 5, 7), (700, 64, 128)])
@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** -18, 2.0 ** -24])
def test_near_gradients(device, rows, n, k, size):
    """dg and du below float16's least normal number: each is off by 2^-25 at most, and nothing else is (float32 results show it)."""
    pre, x = _normal(device, rows, 2 * n, seed=1), _normal(device, rows, k, dtype=F16, seed=4)
    dy, w = (_normal(device, rows, n, seed=3) * size).to(F16), _normal(device, 2 * n, k, dtype=F16, seed=5)
    dx, dw = gated_gemm_bwd(dy, pre, x, w, dx=torch.empty(rows, k, device=device), dw=torch.empty(2 * n, k, device=device))
    wx, ex, ww, ew = _grads(dy, pre, x, w, None, "silu")
    _assert_within(dx, wx, _rounded(wx, ex, F32))
    _assert_within(dw, ww, _rounded(ww, ew, F32))
