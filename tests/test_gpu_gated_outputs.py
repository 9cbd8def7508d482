"""Two outputs of the gated block in one place."""

import pytest
import torch

from cppmega_mlx_amd.nn.gated_ffn import gated_gemm, gated_gemm_bwd
from tests.test_gpu_gated_ffn import BF16, F32, _normal

pytestmark = pytest.mark.gpu


def test_one_place_for_two_results_is_refused(device):
    rows, n, k = 32, 16, 24
    x, w, dy = _normal(device, rows, k, dtype=BF16, seed=1), _normal(device, 2 * n, k, dtype=BF16, seed=2), _normal(device, rows, n, dtype=BF16, seed=3)
    pre = torch.zeros(rows, 2 * n, dtype=BF16, device=device)
    for out, kept in ((pre[:, :n], pre), (torch.zeros(rows, 4 * n, dtype=BF16, device=device)[:, :n], None)):
        kept = out._base.view(F32) if kept is None else kept       # (the same bytes as float32)
        with pytest.raises(ValueError, match="one place"):
            gated_gemm(x, w, out=out, pre=kept)
        assert (out._base == 0).all()
    grad = torch.zeros(2 * n, k, dtype=BF16, device=device)
    with pytest.raises(ValueError, match="one place"):
        gated_gemm_bwd(dy, pre, x, w, dx=grad, dw=grad)
    assert (grad == 0).all()
    # beside each other in one buffer they are two places; empty ones are none
    both = torch.zeros(rows, 3 * n, dtype=BF16, device=device)
    gated_gemm(x, w, out=both[:, 2 * n:], pre=both[:, :2 * n])
    assert torch.equal(both[:, 2 * n:], gated_gemm(x, w, pre=pre)) and torch.equal(both[:, :2 * n], pre)
    gated_gemm(x[:0], w, out=dy[:0], pre=pre[:0])
    assert (gated_gemm_bwd(dy[:0], pre[:0], x[:0], w, dx=x[:0], dw=torch.empty_like(w))[1] == 0).all()
