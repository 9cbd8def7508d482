"""The gated block where many rows take its tiles: tails, pitches, NaN around the operands, broken offsets, graphs and streams, in 16 bits with the
gradients and in e4m3.  Tolerances as in test_gpu_gated_ffn.py.

The sizes are such that each kernel is met: rings of four stages (few tiles, 768 bytes of contraction or more), rings of two (fewer bytes), tiles of
256 rows (rounds of tiles over the CUs), the streaming kernel (few outputs), and, with rows that do not begin on 16 bytes or an odd
contraction, the kernel of any alignment."""

import pytest
import torch

from cppmega_mlx_amd.nn.gated_ffn import fp8_gated_gemm, gated_gemm, gated_gemm_bwd
from tests.test_gpu_gated_ffn import ACTIVATIONS, BF16, DROPPED, F16, F32, U, _assert_within, _gated, _grads, _normal, _offsets, _products, _rounded

pytestmark = pytest.mark.gpu

# rows of three experts (none of the second), outputs, channels
SHAPES = {"deep": (700, 400, 512), "low": (700, 400, 192), "high": (3500, 1300, 144)}
FP8_SHAPES = {"stream": (24, 100, 400), "deep": (700, 400, 1040), "low": (700, 400, 400), "high": (3500, 1300, 272)}
TAIL = 300                                                         # rows behind the last expert: more than a tile


def _held(t, rows, pitch, shift, value):
    """t in a larger tensor: rows of `pitch` elements more, from `shift` elements on, `value` everywhere else."""
    big = torch.full((rows, t.shape[1] + pitch), value, dtype=t.dtype, device=t.device)
    view = big[:, shift:shift + t.shape[1]]
    view[:t.shape[0]] = t
    return big, view


def _counts(rows):
    return [rows // 2 - 3, 0, rows - rows // 2 + 3]


# rows of x that begin on 16 bytes (tiles), and others (the kernel of any alignment)
@pytest.mark.parametrize("pitch, shift", [(24, 0), (24, 8), (17, 1)])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype, name", [(BF16, "silu"), (F16, "gelu_tanh")])
def test_tails_and_pitched_rows(device, shape, dtype, name, pitch, shift):
    rows, n, k = SHAPES[shape]
    counts, every = _counts(rows), rows + TAIL
    offsets, nan = _offsets(counts, device), float("nan")
    x, dy = _normal(device, rows, k, dtype=dtype, seed=1), _normal(device, rows, n, dtype=dtype, seed=3)
    w = (_normal(device, 3, 2 * n, k, seed=2) * 2.0 * k ** -0.5).to(dtype)
    p, size = _products(x, w, offsets)
    want, bound = _gated(p, size, k, name)
    w[1] = nan
    _, xv = _held(x, every, pitch, shift, nan)
    _, dv = _held(dy, every, pitch, shift, nan)
    big_y, yv = _held(dy[:0], every, pitch, shift, 7.0)
    for kept in (dtype, F32):
        big_p, pv = _held(torch.empty(0, 2 * n, dtype=kept, device=device), every, pitch, shift, 7.0)
        assert gated_gemm(xv, w, offsets, activation=name, out=yv, pre=pv) is yv
        _assert_within(yv[:rows], want, _rounded(want, bound, dtype))
        _assert_within(pv[:rows], p, _rounded(p, size * (k * U) * 1.01, kept))
        pre = pv[:rows].clone()
        yv[:rows] = 7.0
        pv[:rows] = 7.0
        assert (big_y == 7.0).all() and (big_p == 7.0).all()       # what belongs to no row of an expert is as it was
    fresh = gated_gemm(xv, w, offsets, activation=name)
    _assert_within(fresh[:rows], want, _rounded(want, bound, dtype))
    assert (fresh[rows:] == 0).all()
    # gradients, from float32 products
    _, pv = _held(pre, every, pitch, shift, nan)
    big_x, gv = _held(x[:0], every, pitch, shift, 7.0)
    gw = torch.empty_like(w)
    assert gated_gemm_bwd(dv, pv, xv, w, offsets, activation=name, dx=gv, dw=gw)[0] is gv
    wx, ex, ww, ew = _grads(dy, pre, x, torch.nan_to_num(w), offsets, name)
    _assert_within(gv[:rows], wx, _rounded(wx, ex, dtype), "dx")
    _assert_within(gw, ww, _rounded(ww, ew, dtype), "dw")
    assert (gw[1] == 0).all()
    gv[:rows] = 7.0
    assert (big_x == 7.0).all()
    fx, fw = gated_gemm_bwd(dv, pv, xv, w, offsets, activation=name)
    _assert_within(fx[:rows], wx, _rounded(wx, ex, dtype), "dx")
    assert (fx[rows:] == 0).all() and torch.equal(fw, gw)


def _fp8(device, rows, n, k, experts, block):
    def codes(*shape, seed):
        return (_normal(device, *shape, seed=seed) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)

    bn, bk = (n + 127) // 128, (k + 127) // 128
    x, w = codes(rows, k, seed=1), codes(experts, 2 * n, k, seed=2)
    return x, torch.exp(_normal(device, *((rows, bk) if block else (rows,)), seed=3)), w, torch.exp(_normal(device, experts, 2, bn, bk, seed=4)) * (2.0 / 3600 / k ** 0.5)


@pytest.mark.parametrize("pitch, shift", [(48, 0), (48, 16), (17, 1)])
@pytest.mark.parametrize("shape", FP8_SHAPES)
@pytest.mark.parametrize("block", [0, 128])
def test_fp8_tails_and_pitched_rows(device, shape, block, pitch, shift):
    rows, n, k = FP8_SHAPES[shape]
    counts, every = _counts(rows), rows + TAIL
    offsets = _offsets(counts, device)
    x, xs, w, ws = _fp8(device, rows, n, k, 3, block)
    wide_x = x.view(torch.float8_e4m3fn).double() * (xs.double().repeat_interleave(128, 1)[:, :k] if block else xs.double()[:, None])
    scale = ws.double().repeat_interleave(128, -2)[..., :n, :].flatten(-3, -2).repeat_interleave(128, -1)[..., :k]
    p, size = _products(wide_x, w.view(torch.float8_e4m3fn).double() * scale, offsets)
    w[1], ws[1] = 0x7f, float("nan")                               # (0x7f: NaN in e4m3)
    _, xv = _held(x, every, pitch, shift, 0x7f)
    xs = torch.cat([xs, torch.full((TAIL, *xs.shape[1:]), float("nan"), device=device)])
    for name in ACTIVATIONS:
        for dtype in (BF16, F16, F32):
            want, bound = _gated(p, size, k + 3 + (DROPPED if dtype == BF16 else 0), name)
            big, out = _held(torch.empty(0, n, dtype=dtype, device=device), every, pitch, shift, 7.0)
            assert fp8_gated_gemm(xv, xs, w, ws, offsets, activation=name, out=out) is out
            _assert_within(out[:rows], want, _rounded(want, bound, dtype), (name, dtype))
            out[:rows] = 7.0
            assert (big == 7.0).all()
            if dtype == BF16:
                for of in (xv, xv.contiguous()):                   # (the second by the native path)
                    fresh = fp8_gated_gemm(of, xs, w, ws, offsets, activation=name)
                    _assert_within(fresh[:rows], want, _rounded(want, bound, dtype), name)
                    assert (fresh[rows:] == 0).all()


def _broken(rows):
    return [[0, rows // 5, rows // 9, 3 * rows // 2], [0, 3, 2 ** 30, rows // 8], [rows // 8, -7, rows, rows], [rows] * 4, [0, 0, 0, -1], [0, rows, 0, rows]]


# (an odd contraction: the kernel of any alignment)
@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("rows, n, k", [*SHAPES.values(), (300, 70, 65)])
def test_offsets_that_break_the_rules_stay_inside(device, which, rows, n, k):
    """Unspecified values, no access outside: the places around the outputs keep theirs."""
    off = torch.tensor(_broken(rows)[which], dtype=torch.int64, device=device)
    x, w, dy = _normal(device, rows, k, dtype=BF16, seed=1), _normal(device, 3, 2 * n, k, dtype=BF16, seed=2), _normal(device, rows, n, dtype=BF16, seed=3)
    y, pre = torch.full((rows + 2, n), 7.0, dtype=BF16, device=device), torch.full((rows + 2, 2 * n), 7.0, device=device)
    dx, dw = torch.full((rows + 2, k), 7.0, dtype=BF16, device=device), torch.full((5, 2 * n, k), 7.0, dtype=BF16, device=device)
    gated_gemm(x, w, off, out=y[1:-1], pre=pre[1:-1])
    gated_gemm(x, w, off)                                          # (with zeros behind the last expert)
    gated_gemm_bwd(dy, pre[1:-1], x, w, off, dx=dx[1:-1], dw=dw[1:-1])
    gated_gemm_bwd(dy, pre[1:-1], x, w, off)
    for t in (y, pre, dx, dw):
        assert (t[0] == 7).all() and (t[-1] == 7).all()


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("rows, n, k", [*FP8_SHAPES.values(), (300, 70, 65)])
def test_offsets_that_break_the_rules_stay_inside_in_e4m3(device, which, rows, n, k):
    off = torch.tensor(_broken(rows)[which], dtype=torch.int32, device=device)
    x, xs, w, ws = _fp8(device, rows, n, k, 3, 128)
    for dtype in (BF16, F32):
        y = torch.full((rows + 2, n), 7.0, dtype=dtype, device=device)
        fp8_gated_gemm(x, xs, w, ws, off, out=y[1:-1])
        assert (y[0] == 7).all() and (y[-1] == 7).all()
    fp8_gated_gemm(x, xs, w, ws, off)


def _sets(device, rows, n, k, seed):
    x, w, dy = _normal(device, rows, k, dtype=BF16, seed=seed), (_normal(device, 4, 2 * n, k, seed=seed + 1) * 0.1).to(BF16), _normal(device, rows, n, dtype=BF16, seed=seed + 2)
    return x, w, dy, *_fp8(device, rows, n, k, 4, 128)


def _step(x, w, dy, x8, xs, w8, ws, off):
    pre = torch.empty(x.shape[0], w.shape[1], device=x.device)
    y = gated_gemm(x, w, off, pre=pre)
    return (y, *gated_gemm_bwd(dy, pre, x, w, off), fp8_gated_gemm(x8, xs, w8, ws, off))


# (k as in SHAPES and FP8_SHAPES at once: multiples of 16)
@pytest.mark.parametrize("rows, n, k", [(800, 400, 784), (800, 400, 192), (3700, 1300, 144), (300, 70, 65)])
def test_graphs_replay_with_other_rows(device, rows, n, k):
    sets = _sets(device, rows, n, k, 1)
    off = _offsets([rows // 3, 0, rows // 2, 20], device)
    _step(*sets, off)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(*sets, off)
        graphs.append((g, out))
    for i, counts in enumerate([[rows // 3, 0, rows // 2, 20], [rows, 0, 0, 0], [1, 2, 3, 4], [0, 0, 0, 0], [0, rows // 2, rows // 4, 1]]):
        off.copy_(_offsets(counts, device))
        sets[0].copy_(_normal(device, rows, k, dtype=BF16, seed=20 + i))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = _step(*sets, off)
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("rows, n, k", [(800, 400, 784), (3700, 1300, 144), (300, 70, 65)])
def test_streams(device, rows, n, k):
    """Calls on several streams at once, operands made on another one."""
    off = _offsets([rows // 3, 0, rows // 2, 20], device)
    sets = [(*_sets(device, rows, n, k, 10 * i + 1), off) for i in range(3)]
    want = [_step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in sets]
    for _ in range(3):
        got = []
        for stream, s in zip(streams, sets):
            stream.wait_stream(torch.cuda.current_stream(device))
            with torch.cuda.stream(stream):
                got.append(_step(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
