"""Calls of the gated block and of the 4-bit products that their documentation allows: one row under many names, a captured training step,
several threads at once."""

import threading

import pytest
import torch

from cppmega_mlx_amd.nn.gated_ffn import fp8_gated_gemm, gated_gemm, gated_gemm_apply, gated_gemm_bwd
from cppmega_mlx_amd.nn.w4_gemm import w4_gated_gemm, w4_gemm
from tests.test_gpu_gated_ffn import BF16, F32, _normal, _offsets
from tests.test_gpu_w4_gemm import _weights

pytestmark = pytest.mark.gpu


# weights streamed, tiles, the kernel of any alignment; 4-bit: 16 and 64 rows at a time
@pytest.mark.parametrize("rows, n, k", [(5, 64, 128), (700, 400, 512), (300, 70, 65)])
def test_a_row_that_stands_for_all(device, rows, n, k):
    """Rows of a pitch of 0."""
    off = _offsets([rows // 2, 0, rows - rows // 2], device)
    w = (_normal(device, 3, 2 * n, k, seed=2) * 0.1).to(BF16)
    x, dy, pre = (_normal(device, 1, c, dtype=BF16, seed=s).expand(rows, c) for c, s in ((k, 1), (n, 3), (2 * n, 4)))
    assert torch.equal(gated_gemm(x, w, off), gated_gemm(x.contiguous(), w, off))
    got, want = gated_gemm_bwd(dy, pre, x, w, off), gated_gemm_bwd(dy.contiguous(), pre.contiguous(), x.contiguous(), w, off)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x8, w8 = (t.float().to(torch.float8_e4m3fn).view(torch.uint8) for t in (x[:1], w))
    xs, ws = torch.ones(rows, device=device), torch.ones(3, 2, (n + 127) // 128, (k + 127) // 128, device=device)
    assert torch.equal(fp8_gated_gemm(x8.expand(rows, k), xs, w8, ws, off), fp8_gated_gemm(x8.expand(rows, k).contiguous(), xs, w8, ws, off))


@pytest.mark.parametrize("rows, n, k", [(40, 100, 320), (300, 2200, 1056)])
def test_a_row_that_stands_for_all_over_4_bits(device, rows, n, k):
    off = _offsets([rows // 2, 0, rows - rows // 2], device)
    w, scale, bias = _weights(device, (3,), 2 * n, k, 32, True, BF16, seed=1)
    x = _normal(device, 1, k, dtype=BF16, seed=1).expand(rows, k)
    for call in (w4_gemm, w4_gated_gemm):
        assert torch.equal(call(x, w, scale, bias, off), call(x.contiguous(), w, scale, bias, off))


@pytest.mark.parametrize("rows, n, k", [(96, 64, 128), (700, 400, 512)])
@pytest.mark.parametrize("kept", [F32, BF16])
def test_a_captured_training_step(device, rows, n, k, kept):
    """Forward and backward pass of the autograd form in one graph, whose leaves no eager graph has."""
    x, w, dy = _normal(device, rows, k, dtype=BF16, seed=1), (_normal(device, 3, 2 * n, k, seed=2) * 0.1).to(BF16), _normal(device, rows, n, dtype=BF16, seed=3)
    off = _offsets([rows // 3, 0, rows // 2], device)

    def eager():
        pre = torch.empty(rows, 2 * n, dtype=kept, device=device)
        return (gated_gemm(x, w, off, pre=pre), *gated_gemm_bwd(dy, pre, x, w, off))

    eager()
    leaves = x.requires_grad_(), w.requires_grad_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gated_gemm_apply(x, w, off, pre_dtype=kept)
        got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    del y
    x, w = x.detach(), w.detach()
    for i, counts in enumerate([[rows // 3, 0, rows // 2], [0, rows, 0], [1, 2, 3], [0, 0, 0]]):
        off.copy_(_offsets(counts, device))
        x.copy_(_normal(device, rows, k, dtype=BF16, seed=20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager())), i


def test_threads(device):
    """Calls of several threads, each on a stream of its own."""
    sets = []
    for i in range(4):
        w4, scale, bias = _weights(device, (2,), 200, 256, 64, True, BF16, seed=i)
        sets.append((_normal(device, 90, 256, dtype=BF16, seed=i), (_normal(device, 2, 200, 256, seed=9 + i) * 0.1).to(BF16), _normal(device, 90, 100, dtype=BF16, seed=30 + i),
                     w4, scale, bias, _offsets([50, 40], device), torch.cuda.Stream(device)))

    def step(x, w, dy, w4, scale, bias, off, stream):
        with torch.cuda.stream(stream):
            pre = torch.empty(90, 200, device=device)
            out = [gated_gemm(x, w, off, pre=pre), *gated_gemm_bwd(dy, pre, x, w, off), w4_gated_gemm(x, w4, scale, bias, off)]
            stream.synchronize()
            return out

    torch.cuda.synchronize()
    want = [step(*s) for s in sets]
    got = [[] for _ in sets]

    def work(i):
        for _ in range(20):
            got[i].append(step(*sets[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, expected in zip(got, want):
        assert len(outs) == 20 and all(torch.equal(a, b) for out in outs for a, b in zip(out, expected))
