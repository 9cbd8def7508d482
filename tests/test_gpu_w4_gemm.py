"""GPU parity of the products with 4-bit weights, plain and gated, against the formulas in 64 bits.

Tolerances, U = 2^-24.  x (16 + q) is exact in float32; a group's sums are off by at most G U of their magnitudes, and every group adds four roundings
(b - 16 s, its product, the two additions) to partial sums that stay below m = sum |x| (|s| (16 + q) + |b| + 16 |s|) (without biases 24 |s|); up
to 8 wavefronts' sums are added: (K + 16) U m in all, for G + 4 K / G + 8 <= K + 16 at every K.  The result is rounded once, by
eps(type) / 2 of itself (float16 below 6e-5 by 2^-25).  The gated form as in the block of 16-bit weights: s is off by (6 |z| (1 - s) + 5) U of
itself, two products follow, an error of g reaches act(g) by its slope, at most 1.13."""

import pytest
import torch

from cppmega_mlx_amd import _lib, ops
from cppmega_mlx_amd.nn.rms_norm import rms_norm
from cppmega_mlx_amd.nn.w4_gemm import w4_gated_gemm, w4_gemm
from tests.test_gpu_gated_ffn import BF16, F16, F32, TINY, U, _assert_within, _gated, _half, _normal, _offsets, _rounded

pytestmark = pytest.mark.gpu


def _weights(device, lead, n, k, group, bias, dtype, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    w = torch.randint(0, 256, (*lead, n, k // 2), generator=g, device=device, dtype=torch.uint8)
    scale = (torch.exp(0.5 * torch.randn(*lead, n, k // group, generator=g, device=device)) * (0.3 * k ** -0.5)).to(dtype)
    return w, scale, (scale.float() * (-7.5 + torch.randn(scale.shape, generator=g, device=device))).to(dtype) if bias else None


def _wide(w, scale, bias):
    """(weights, the magnitudes that pass through the sums) in 64 bits."""
    q = torch.stack([w & 15, w >> 4], -1).flatten(-2).double()
    group = q.shape[-1] // scale.shape[-1]
    s = scale.double().repeat_interleave(group, -1)
    b = -8 * s if bias is None else bias.double().repeat_interleave(group, -1)
    return s * q + b, s.abs() * (16 + q) + (24 * s.abs() if bias is None else b.abs() + 16 * s.abs())


def _products(x, w, scale, bias, offsets):
    m, size = _wide(w, scale, bias)
    if offsets is None:
        return x.double() @ m.T, x.double().abs() @ size.T
    p = torch.zeros(x.shape[0], w.shape[-2], dtype=torch.float64, device=x.device)
    z = torch.zeros_like(p)
    b = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(b, b[1:])):
        p[lo:hi], z[lo:hi] = x[lo:hi].double() @ m[e].T, x[lo:hi].double().abs() @ size[e].T
    return p, z


# rows (a list: of every expert), outputs, channels in groups of 32
CASES = [(1, 1, 1), (1, 16, 4), (2, 17, 8), (16, 40, 36), (5, 1001, 33), (17, 100, 12), (33, 64, 20), (64, 130, 68), (100, 48, 8), (3, 2000, 64), (1, 4099, 224), (13, 33, 513),
         ([1, 0, 3, 0, 20], 50, 12), ([0, 0], 16, 4), ([40, 1, 7], 70, 24), ([1] * 70, 24, 8), ([0, 200, 0, 3], 33, 40)]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0] if isinstance(c[0], int) else f'{sum(c[0])}of{len(c[0])}'}x{c[1]}x{c[2] * 32}")
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bias", [True, False])
def test_products(device, case, group, dtype, bias):
    _check_products(device, case, group, dtype, bias)


# many rows: 64 at a time, the contraction in 4 and 2 parts, passes and groups that end inside, experts of fewer rows and of none
MANY = [(64, 10300, 33), (51, 10250, 36), (130, 4600, 35), (300, 2200, 68), (500, 4100, 32), ([200, 0, 33, 300, 1], 1500, 37), ([64, 65, 0, 190], 1901, 100)]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{c[0] if isinstance(c[0], int) else f'{sum(c[0])}of{len(c[0])}'}x{c[1]}x{c[2] * 32}")
@pytest.mark.parametrize("group, dtype, bias", [(32, BF16, True), (64, F16, False), (64, BF16, True), (128, BF16, False), (128, F16, True)])
def test_products_of_many_rows(device, case, group, dtype, bias):
    _check_products(device, case, group, dtype, bias)


def _check_products(device, case, group, dtype, bias):
    rows, n, k = case[0], case[1], case[2] * 32
    k = (k + group - 1) // group * group
    offsets = None if isinstance(rows, int) else _offsets(rows, device)
    lead = () if offsets is None else (len(rows),)
    rows = rows if offsets is None else sum(rows)
    x = _normal(device, rows, k, dtype=dtype, seed=1)
    for scale_type in (dtype, F32):
        w, scale, b = _weights(device, lead, n, k, group, bias, scale_type, seed=2)
        y = w4_gemm(x, w, scale, b, offsets)
        assert y.dtype == dtype and y.shape == (rows, n)
        want, size = _products(x, w, scale, b, offsets)
        bound = size * (k + 16) * U
        _assert_within(y, want, _rounded(want, bound, dtype))
        wide = torch.empty(rows, n, device=device)
        assert w4_gemm(x, w, scale, b, None if offsets is None else offsets.long(), out=wide) is wide and torch.equal(wide.to(dtype), y)
        _assert_within(wide, want, _rounded(want, bound, F32))
        both, scales, b = _weights(device, lead, 2 * n, k, group, bias, scale_type, seed=3)
        p, size = _products(x, both, scales, b, offsets)
        for name in ("silu", "gelu_tanh"):
            want, bound = _gated(p, size, k + 16, name)
            _assert_within(w4_gated_gemm(x, both, scales, b, offsets, activation=name), want, _rounded(want, bound, dtype), name)


def test_every_code_in_every_place(device):
    """One-hot rows read single weights: their values are exact products of scale and code."""
    for group, dtype in ((32, F16), (64, BF16), (128, F16), (128, BF16)):
        k, n = 256, 48
        q = (torch.arange(n * k, device=device).view(n, k) * 7 + torch.arange(n, device=device)[:, None]) % 16
        w = (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8)
        scale = torch.exp2(torch.arange(n * (k // group), device=device).view(n, -1) % 5 - 2.0).to(dtype)
        bias = (scale.float() * -3).to(dtype)
        s, b = scale.double().repeat_interleave(group, 1), bias.double().repeat_interleave(group, 1)
        x = torch.eye(k, dtype=dtype, device=device)
        got = torch.empty(k, n, device=device)
        assert torch.equal(w4_gemm(x, w, scale, bias, out=got).double(), (s * q + b).T)
        assert torch.equal(w4_gemm(x, w, scale, out=got).double(), (s * (q - 8)).T)


@pytest.mark.parametrize("shape", [(7, 40, 320), (37, 33, 96), (380, 1700, 1056)], ids=str)
def test_views_and_tails(device, shape):
    rows, n, k = shape
    tail, counts = 9, [rows // 3, 0, rows - rows // 3]
    offsets = _offsets(counts, device)
    w, scale, bias = _weights(device, (3,), n, k, 32, True, BF16, seed=1)
    x = _normal(device, rows, k, dtype=BF16, seed=2)
    want = w4_gemm(x, w, scale, bias, offsets)
    scale[1] = float("nan")
    bias[1] = float("inf")
    for shift in (0, 1, 8):
        big = torch.full((rows + tail, k + 11), float("nan"), dtype=BF16, device=device)
        xv = big[:, shift:shift + k]
        xv[:rows] = x
        out = torch.full((rows + tail, n + 5), 7.0, dtype=BF16, device=device)
        yv = out[:, shift % 4:shift % 4 + n]
        assert w4_gemm(xv, w, scale, bias, offsets, out=yv) is yv
        assert (yv[:rows].double() - want.double()).abs().max() <= 2 * _half(BF16) * float(want.double().abs().max())
        yv[:rows] = 7.0
        assert (out == 7.0).all()
        fresh = w4_gemm(xv, w, scale, bias, offsets)
        assert (fresh[rows:] == 0).all() and torch.isfinite(fresh).all()
    # weights and scales that begin anywhere
    held = torch.zeros(w.numel() + 3, dtype=torch.uint8, device=device)
    held[3:] = w.view(-1)
    shifted = torch.zeros(scale.numel() + 1, dtype=BF16, device=device)
    shifted[1:] = scale.view(-1)
    assert torch.equal(w4_gemm(x, held[3:].view(w.shape), shifted[1:].view(scale.shape), bias, offsets), want)


@pytest.mark.parametrize("values", [[0, 9, 4, 60], [0, 3, 2 ** 30, 5], [5, -7, 40, 40], [40, 40, 40, 40], [0, 0, 0, -1]], ids=str)
@pytest.mark.parametrize("rows, n, k", [(40, 48, 64), (200, 1500, 1024)])
def test_offsets_that_break_the_rules_stay_inside(device, values, rows, n, k):
    w, scale, bias = _weights(device, (3,), 2 * n, k, 32, True, BF16, seed=1)
    x = _normal(device, rows, k, dtype=BF16, seed=2)
    off = torch.tensor(values, dtype=torch.int64, device=device)
    for width, call in ((2 * n, w4_gemm), (n, w4_gated_gemm)):
        y = torch.full((rows + 2, width), 7.0, dtype=BF16, device=device)
        call(x, w, scale, bias, off, out=y[1:-1])
        assert (y[0] == 7).all() and (y[-1] == 7).all()


def test_large_magnitudes_and_nan(device):
    w, scale, bias = _weights(device, (), 20, 128, 64, True, BF16, seed=1)
    x = _normal(device, 3, 128, dtype=BF16, seed=2) * 1e30
    want, size = _products(x, w, scale, bias, None)
    _assert_within(w4_gemm(x, w, scale, bias), want, _rounded(want, size * (128 + 16) * U, BF16))
    x[1, 5] = float("nan")
    x[2, 9] = float("inf")
    y = w4_gemm(x, w, scale, bias)
    assert torch.isfinite(y[0]).all() and y[1:].isnan().all()


@pytest.mark.parametrize("per, n, k", [(1, 128, 256), (9, 2700, 1088)])
def test_graphs_streams_and_repeats(device, per, n, k):
    w, scale, bias = _weights(device, (4,), n, k, 64, True, BF16, seed=1)
    x, off = _normal(device, 24 * per, k, dtype=BF16, seed=2), _offsets([10 * per, 0, 2 * per, 12 * per], device)

    def call():
        return w4_gemm(x, w, scale, bias, off), w4_gated_gemm(x, w, scale, None, off), w4_gemm(x, w[0], scale[0])

    want = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i, counts in enumerate([[10, 0, 2, 12], [24, 0, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0]]):
        off.copy_(_offsets([c * per for c in counts], device))
        x.copy_(_normal(device, 24 * per, k, dtype=BF16, seed=5 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    off.copy_(_offsets([10 * per, 0, 2 * per, 12 * per], device))
    want = call()
    streams = [torch.cuda.Stream(device) for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_the_native_path_and_the_helpers_agree(device, monkeypatch):
    w, scale, bias = _weights(device, (2,), 96, 128, 32, True, F16, seed=1)
    x, off = _normal(device, 11, 128, dtype=F16, seed=2), _offsets([5, 6], device)

    def call():
        return (w4_gemm(x, w, scale, bias, off), w4_gemm(x, w[1], scale[1], None), w4_gated_gemm(x, w, scale.float(), bias.float(), off.long(), activation="gelu_tanh"))

    native, host = call(), ops.host
    assert host.w4_gemm(x[:, ::2], w, scale, bias, off, -1) is None and host.w4_gemm(x, w, scale.double(), None, off, -1) is None and host.w4_gemm(x, w, scale, bias[:1], off, -1) is None
    assert host.w4_gemm(x, w, scale, bias, None, -1) is None and host.w4_gemm(x, w, scale, bias, off, 9) is None
    monkeypatch.setattr(ops, "host", type("Declines", (), {"__getattr__": lambda self, name: lambda *a: None})())
    for a, b in zip(native, call()):
        assert torch.equal(a, b)


def test_refusals(device):
    w, scale, bias = _weights(device, (2,), 32, 128, 32, True, BF16, seed=1)
    x, off = _normal(device, 8, 128, dtype=BF16, seed=2), _offsets([3, 5], device)
    y = torch.empty(8, 32, dtype=BF16, device=device)
    for error, call in [
        (TypeError, lambda: w4_gemm(x.float(), w, scale, bias, off)), (TypeError, lambda: w4_gemm(x, w.to(torch.int32), scale, bias, off)), (TypeError, lambda: w4_gemm(x, w, scale.half(), None, off)),
        (ValueError, lambda: w4_gemm(x, w, scale, bias.float(), off)), (ValueError, lambda: w4_gemm(x, w, scale, bias[:, :, :2].contiguous(), off)), (ValueError, lambda: w4_gemm(x, w, scale, bias)),
        (ValueError, lambda: w4_gemm(x, w[0], scale[0], None, off)), (ValueError, lambda: w4_gemm(x, w, scale[:, :, :3].contiguous(), None, off)), (ValueError, lambda: w4_gemm(x[:, :96], w, scale, bias, off)),
        (ValueError, lambda: w4_gemm(x, w, torch.ones(2, 32, 8, dtype=BF16, device=device), None, off)), (ValueError, lambda: w4_gemm(x, w, scale[..., 0], None, off)), (ValueError, lambda: w4_gemm(x, w, scale, bias, off[:2])),
        (TypeError, lambda: w4_gemm(x, w, scale, bias, off.float())), (_lib.NativeCallError, lambda: w4_gemm(x, w, scale, bias, off.cpu())), (TypeError, lambda: w4_gemm(x, w, scale, bias, off, out=y.half())),
        (ValueError, lambda: w4_gemm(x, w, scale, bias, off, out=y[:, :16])), (ValueError, lambda: w4_gemm(x, w, scale, bias, off, out=y[:1].expand(8, 32))), (ValueError, lambda: w4_gemm(x, w.transpose(1, 2), scale, bias, off)),
        (ValueError, lambda: w4_gated_gemm(x, w, scale, bias, off, activation="relu")), (ValueError, lambda: w4_gated_gemm(x, w[:, :31].contiguous(), scale[:, :31].contiguous(), None, off)),
        (_lib.NativeCallError, lambda: w4_gemm(x, torch.zeros(513, 2, 64, dtype=torch.uint8, device=device), torch.ones(513, 2, 4, dtype=BF16, device=device), None, torch.zeros(514, dtype=torch.int32, device=device))),
    ]:
        with pytest.raises(error):
            call()
    assert w4_gemm(x[:0], w, scale, bias, off * 0).shape == (0, 32) and w4_gated_gemm(x[:0], w, scale, bias, off * 0).shape == (0, 16)
    out = torch.empty(8, 32, dtype=BF16, device=device)
    before = out._version
    w4_gemm(x, w, scale, bias, off, out=out)
    assert out._version > before


def test_a_decode_step_runs_through(device):
    """Norm, the gated block and the down projection of a few tokens over 4-bit experts."""
    rows, k, f = 6, 128, 96
    off = _offsets([2, 0, 4], device)
    up, us, ub = _weights(device, (3,), 2 * f, k, 64, True, BF16, seed=1)
    down, ds, _ = _weights(device, (3,), k, f, 32, False, BF16, seed=2)
    x = rms_norm(_normal(device, rows, k, dtype=BF16, seed=3), torch.ones(k, dtype=BF16, device=device))
    mid = w4_gated_gemm(x, up, us, ub, off)
    out = w4_gemm(mid, down, ds, None, off)
    p, size = _products(x, up, us, ub, off)
    want, bound = _gated(p, size, k + 16, "silu")
    _assert_within(mid, want, _rounded(want, bound, BF16))
    want, size = _products(mid, down, ds, None, off)
    _assert_within(out, want, _rounded(want, size * (f + 16) * U, BF16))


@pytest.mark.parametrize("rows, n, k", [(65535 * 16 + 40, 17, 32), (65535 * 64 + 70, 33, 1024)])
def test_more_tiles_of_rows_than_a_grid_is_high(device, rows, n, k):
    w, scale, bias = _weights(device, (), n, k, 32, True, BF16, seed=1)
    x = _normal(device, 1024, k, dtype=BF16, seed=2).repeat((rows + 1023) // 1024, 1)[:rows]
    y = w4_gemm(x, w, scale, bias)
    want, size = _products(x[:1024], w, scale, bias, None)
    _assert_within(y[:1024], want, _rounded(want, size * (k + 16) * U, BF16))
    last = (rows - 1024) // 1024 * 1024                            # (rows repeat, and their results with them)
    assert torch.equal(y[:last].view(-1, 1024, n), y[:1024].expand(last // 1024, 1024, n)) and torch.equal(y[last:], y[:1024].repeat(2, 1)[:rows - last])


@pytest.mark.parametrize("n", [64, 10300])
def test_rows_far_apart(device, n):
    rows, k, pitch = 64, 1024, 1 << 24
    w, scale, bias = _weights(device, (), n, k, 64, True, F16, seed=1)
    x = _normal(device, rows, k, dtype=F16, seed=2)
    far = torch.empty(rows, pitch, dtype=F16, device=device)[:, pitch - k:]
    far.copy_(x)
    assert torch.equal(w4_gemm(far, w, scale, bias), w4_gemm(x, w, scale, bias))
