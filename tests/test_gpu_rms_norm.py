"""GPU parity of the RMS norm (rows, 8-bit rows, gradients) against the formulas in 64 bits.

Tolerances.  One rounding to the rows' type: eps(type) / 2 of the value.  Float32 work: the sum of n squares is made of chains of at
most 32 additions, 6 steps over a wavefront and 16 wavefronts, all terms positive: 54 roundings, half of that on its root, then a
division, a square root and two products: 32 * 2^-24 relative in y.  Gradients: the same roundings on sums with signs, so relative to
the sums of magnitudes."""

import pytest
import torch

from cppmega_mlx_amd import _lib, ops
from cppmega_mlx_amd.nn.rms_norm import rms_norm, rms_norm_apply, rms_norm_bwd, rms_norm_fp8

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
TINY = {BF16: 0.0, F16: 2.0 ** -25, F32: 2.0 ** -149}           # half a step of the type's subnormal numbers (bf16: below float32's own)
SHAPES = [(1, 1), (3, 7), (5, 64), (2, 128), (7, 333), (4, 512), (6, 513), (3, 1536), (2, 2048), (3, 2049), (5, 4096), (4, 5003), (2, 7168), (700, 7168),
          (2, 8193), (3, 16384), (2, 20001), (2, 32768)]


def _normal(device, *shape, dtype, seed, size=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=device) * size).to(dtype)


def _inputs(device, rows, n, dtype, wdtype=None, seed=0):
    return (_normal(device, rows, n, dtype=dtype, seed=seed, size=3.0), (1 + 0.3 * _normal(device, n, dtype=F32, seed=seed + 1)).to(wdtype or dtype),
            _normal(device, rows, n, dtype=dtype, seed=seed + 2))


def _plain(h, weight, eps):
    v = h.double()
    s = 1.0 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    return v * s * weight.double()


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _assert_y(y, want, dtype):
    bound = want.abs() * (_half(dtype) + 34 * U) + TINY[dtype]
    assert (y.double() - want).abs().le(bound).all(), float(((y.double() - want).abs() - bound).max())


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype, wdtype", [(BF16, BF16), (F16, F32), (F32, F32), (BF16, F32), (F16, F16)])
def test_rows(device, shape, dtype, wdtype):
    x, w, r = _inputs(device, *shape, dtype, wdtype)
    _assert_y(rms_norm(x, w, eps=1e-5), _plain(x, w, 1e-5), dtype)
    y, h = rms_norm(x, w, eps=1e-5, residual=r)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    _assert_y(y, _plain(h, w, 1e-5), dtype)


def _value(codes):
    return codes.view(torch.float8_e4m3fn).double()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block", [0, 128])
@pytest.mark.parametrize("pow2", [False, True])
def test_codes(device, shape, dtype, block, pow2):
    x, w, r = _inputs(device, *shape, dtype, seed=9)
    codes, scale, h = rms_norm_fp8(x, w, eps=1e-6, residual=r, scale_block=block, pow2_scales=pow2)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    want = _plain(h, w, 1e-6)
    n, size = shape[1], block or shape[1]
    per = (scale if block else scale[:, None]).double()
    amax = torch.stack([want[:, i:i + size].abs().amax(1) for i in range(0, n, size)], 1)
    if pow2:
        exact = torch.exp2(torch.ceil(torch.log2(amax / 448)))
        near = ((torch.log2(amax / 448) - torch.log2(amax / 448).round()).abs() < 1e-4)      # amax at a border of two scales: either is right to rounding
        assert ((per == exact) | near).all() and torch.equal(torch.exp2(torch.log2(per).round()), per)
    else:
        assert ((per - amax / 448).abs() <= amax / 448 * 37 * U).all()
    # the code is the nearest one to y / scale: half a step is 2^-4 of the value, or 2^-10 below 2^-6
    spread = per.repeat_interleave(size, 1)[:, :n]
    v = want / spread
    assert ((_value(codes) - v).abs() <= torch.maximum(v.abs() / 16, torch.tensor(2.0 ** -10, device=device, dtype=torch.float64)) + v.abs() * 40 * U).all()


def test_rows_of_zeros_large_and_non_finite_values(device):
    n = 640
    x = torch.randn(6, n, device=device)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 5] = float("inf")
    x[3] *= 1e17
    x[4] *= 1e-30
    w = torch.ones(n, device=device)
    y = rms_norm(x, w, eps=1e-6)
    assert (y[0] == 0).all() and y[1].isnan().all() and y[2, 5].isnan() and (y[2, :5] == 0).all()
    _assert_y(y[3:], _plain(x[3:], w, 1e-6), F32)
    for block in (0, 128):
        codes, scale = rms_norm_fp8(x, w, eps=1e-6, scale_block=block)
        assert (codes[0] == 0).all() and (scale[0] == torch.tensor(1e-12)).all()
        assert _value(codes[1]).isnan().all() and _value(codes[2, 5:6]).isnan().all()
        assert _value(codes[3:]).isfinite().all()
    _, scale = rms_norm_fp8(x, w, pow2_scales=True)
    assert scale[0] == 1
    # an infinite weight makes one block's scale infinite: its finite values have no code but 0
    w[130] = float("inf")
    codes, scale = rms_norm_fp8(x[5:], w, scale_block=128)
    assert scale[0, 1].isinf() and scale[0, 0].isfinite() and _value(codes[0, 130:131]).isnan().all() and (_value(codes[0, 131:256]) == 0).all()


def test_views_pitches_and_places_in_use(device):
    """Rows inside wider rows, odd starts, broadcast inputs, results in the inputs' own place; what lies beside stays."""
    for n in (96, 101, 2050):
        wide = _normal(device, 5, n + 13, dtype=BF16, seed=n)
        x, w = wide[:, 3:3 + n], (1 + 0.1 * torch.randn(n, device=device)).to(BF16)
        want = _plain(x, w, 1e-6)
        y = torch.full((5, n + 7), 7.0, dtype=BF16, device=device)
        assert rms_norm(x, w, out=y[:, 1:1 + n]).data_ptr() == y[:, 1:].data_ptr()
        _assert_y(y[:, 1:1 + n], want, BF16)
        assert (y[:, 0] == 7).all() and (y[:, 1 + n:] == 7).all()
        codes = torch.full((5, n + 5), 99, dtype=torch.uint8, device=device)
        got, scale = rms_norm_fp8(x, w, scale_block=128, codes=codes[:, 2:2 + n])
        again, scale2 = rms_norm_fp8(x.contiguous(), w, scale_block=128)
        assert torch.equal(got, again) and torch.equal(scale, scale2) and (codes[:, :2] == 99).all() and (codes[:, 2 + n:] == 99).all()
        row = x[:1].expand(4, n)
        y, h = rms_norm(row, w, residual=row)
        assert torch.equal(h, (2 * row.float()).to(BF16)) and torch.equal(y[0], y[3])
        # in place: the stream takes the sum, the rows take the result
        a, r = x.contiguous(), _normal(device, 5, n, dtype=BF16, seed=n + 1)
        y, h = rms_norm(a.clone(), w, residual=r)
        stream = r.clone()
        got = rms_norm(a, w, residual=stream, out=a, residual_out=stream)
        assert got[0] is a and got[1] is stream and torch.equal(a, y) and torch.equal(stream, h)
    t = _normal(device, 2, 3, 4, 64, dtype=F16, seed=5)
    assert rms_norm(t, torch.ones(64, dtype=F16, device=device)).shape == t.shape
    assert rms_norm(t[:, :0], torch.ones(64, dtype=F16, device=device)).shape == (2, 0, 4, 64)
    assert rms_norm_fp8(t, torch.ones(64, dtype=F16, device=device), scale_block=128)[1].shape == (2, 3, 4, 1)


def test_more_rows_than_a_32_bit_offset_reaches(device):
    """2^31 elements and more: the last rows are the ones of a small call."""
    rows, n = (1 << 31) // 4096 + 5, 4096
    x = torch.zeros(rows, n, dtype=BF16, device=device)
    x[-7:] = _normal(device, 7, n, dtype=BF16, seed=3)
    w = (1 + 0.1 * torch.randn(n, device=device)).to(BF16)
    y = rms_norm(x, w)
    assert torch.equal(y[-7:], rms_norm(x[-7:].clone(), w)) and (y[:5] == 0).all()
    del y
    codes, scale = rms_norm_fp8(x, w, scale_block=128)
    small = rms_norm_fp8(x[-7:].clone(), w, scale_block=128)
    assert torch.equal(codes[-7:], small[0]) and torch.equal(scale[-7:], small[1])


@pytest.mark.parametrize("n", [8, 520])
def test_more_rows_than_one_launch_has(device, n):
    rows = (1 << 21) + 6
    x, w = _normal(device, rows, n, dtype=BF16, seed=4), (1 + 0.1 * _normal(device, n, dtype=F32, seed=5)).to(BF16)
    y, h = rms_norm(x, w, residual=x)
    codes, scale = rms_norm_fp8(x, w)
    for part in (slice(0, 9), slice((1 << 21) - 9, (1 << 21) + 2), slice(rows - 7, rows)):
        small = rms_norm(x[part], w, residual=x[part]), rms_norm_fp8(x[part], w)
        assert torch.equal(y[part], small[0][0]) and torch.equal(h[part], small[0][1])
        assert torch.equal(codes[part], small[1][0]) and torch.equal(scale[part], small[1][1])


# ---- gradients ------------------------------------------------------------------------------
def _plain_bwd(g, h, w, eps, dh=None):
    g, h, w = g.double(), h.double(), w.double()
    n = h.shape[-1]
    s = 1.0 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    c = (g * w * h).mean(-1, keepdim=True)
    dx = s * g * w - s ** 3 * c * h
    size = (s * g * w).abs() + s ** 3 * (g * w * h).abs().mean(-1, keepdim=True) * h.abs()
    if dh is not None:
        dx, size = dx + dh.double(), size + dh.double().abs()
    return dx, (g * h * s).sum(0), size, (g * h * s).abs().sum(0)


@pytest.mark.parametrize("shape", SHAPES + [(513, 96), (2500, 64), (1027, 5000), (5001, 1030), (9001, 40), (2101, 9000), (2049, 1000)])
@pytest.mark.parametrize("dtype, wdtype", [(BF16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("past", [False, True])
def test_gradients(device, shape, dtype, wdtype, past):
    h, w, g = _inputs(device, *shape, dtype, wdtype, seed=21)
    dh = _normal(device, *shape, dtype=dtype, seed=30) if past else None
    dx, dw = rms_norm_bwd(g, h, w, eps=1e-5, dh=dh)
    want_x, want_w, size_x, size_w = _plain_bwd(g, h, w, 1e-5, dh)
    assert dx.dtype == dtype and dw.dtype == F32
    # 54 roundings of each sum, s three times (32 each), 8 products: below 256 in all
    bound = want_x.abs() * _half(dtype) + size_x * 256 * U + TINY[dtype]
    assert ((dx.double() - want_x).abs() <= bound).all()
    # a group's rows (256 groups at least: up to rows / 256 + 1), groups in 16 runs (up to 2048 / 16), 16 runs, s
    assert ((dw.double() - want_w).abs() <= size_w * (shape[0] / 256 + 1 + 128 + 16 + 40) * U + 1e-40).all()
    again = rms_norm_bwd(g, h, w, eps=1e-5, dh=dh)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def test_gradients_against_differences(device):
    """Directional differences of the formula in 64 bits, along the inputs and along the weight."""
    h, w, g = _inputs(device, 3, 200, F32, seed=40)
    dx, dw = rms_norm_bwd(g, h, w, eps=1e-3)
    _, _, size_x, size_w = _plain_bwd(g, h, w, 1e-3)
    loss = lambda a, b: (_plain(a, b, 1e-3) * g.double()).sum()
    for seed in range(3):
        d, e = _normal(device, 3, 200, dtype=F32, seed=50 + seed).double(), _normal(device, 200, dtype=F32, seed=60 + seed).double()
        step = 1e-5
        by_x = (loss(h.double() + step * d, w.double()) - loss(h.double() - step * d, w.double())) / (2 * step)
        by_w = (loss(h.double(), w.double() + step * e) - loss(h.double(), w.double() - step * e)) / (2 * step)
        # the gradients' own bounds, and the differences' third order: below 1e-9 of the sums of magnitudes
        assert abs(float((dx.double() * d).sum() - by_x)) <= (256 * U + 1e-8) * float((size_x * d.abs()).sum())
        assert abs(float((dw.double() * e).sum() - by_w)) <= (256 * U + 1e-8) * float((size_w * e.abs()).sum())


def test_gradient_views_no_rows_and_results_in_place(device):
    h, w, g = _inputs(device, 6, 101, BF16, seed=70)
    dx, dw = rms_norm_bwd(g, h, w)
    wide = torch.full((6, 130), 5.0, dtype=BF16, device=device)
    wide[:, 7:108] = g
    got = rms_norm_bwd(wide[:, 7:108], h, w, dx=wide[:, 7:108])
    assert torch.equal(got[0], dx) and torch.equal(got[1], dw) and (wide[:, :7] == 5).all() and (wide[:, 108:] == 5).all()
    past = rms_norm_bwd(g, h, w, dh=g)
    mine = g.clone()
    assert torch.equal(rms_norm_bwd(g, h, w, dh=mine, dx=mine)[0], past[0]) and torch.equal(mine, past[0])
    got = rms_norm_bwd(g[:0], h[:0], w, dweight=torch.full((101,), 3.0, device=device))
    assert got[0].shape == (0, 101) and (got[1] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_differentiable_form(device, dtype):
    x, w, r = (t.requires_grad_() for t in _inputs(device, 2 * 3, 320, dtype, seed=80))
    g, d = _normal(device, 6, 320, dtype=dtype, seed=90), _normal(device, 6, 320, dtype=dtype, seed=91)
    y, h = rms_norm_apply(x, w, r, eps=1e-5)
    torch.autograd.backward([y, h], [g, d])
    dx, dw = rms_norm_bwd(g, h.detach(), w.detach(), eps=1e-5, dh=d)
    assert torch.equal(x.grad, dx) and torch.equal(r.grad, dx) and torch.equal(w.grad, dw.to(dtype)) and x.grad.data_ptr() != r.grad.data_ptr()
    # the same tensor twice, a broadcast cotangent, one output only
    x2 = x.detach().clone().requires_grad_()
    y, h = rms_norm_apply(x2, w.detach(), x2, eps=1e-5)
    y.sum().backward()
    dx, _ = rms_norm_bwd(torch.ones_like(h), h.detach(), w.detach(), eps=1e-5)
    assert torch.equal(x2.grad, (2 * dx.float()).to(dtype))
    x3 = x.detach().clone().requires_grad_()
    rms_norm_apply(x3, w.detach(), r.detach())[1].backward(d)
    assert torch.equal(x3.grad, d)
    x4 = x.detach().clone().requires_grad_()
    rms_norm_apply(x4.t().contiguous().t(), w.detach(), eps=1e-5).backward(g)
    assert torch.equal(x4.grad, rms_norm_bwd(g, x.detach(), w.detach(), eps=1e-5)[0])


def test_captured_calls_replay_on_new_values(device):
    x, w, r = _inputs(device, 40, 1536, BF16, seed=100)
    g = _normal(device, 40, 1536, dtype=BF16, seed=101)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            rms_norm(x, w, residual=r), rms_norm_fp8(x, w, scale_block=128), rms_norm_bwd(g, x, w)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = (*rms_norm(x, w, residual=r), *rms_norm_fp8(x, w, scale_block=128), *rms_norm_bwd(g, x, w))
    for k in range(3):
        for t, s in ((x, 110), (r, 120), (g, 130)):
            t.copy_(_normal(device, 40, 1536, dtype=BF16, seed=s + k))
        want = (*rms_norm(x, w, residual=r), *rms_norm_fp8(x, w, scale_block=128), *rms_norm_bwd(g, x, w))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_graphs_of_one_stream_side_by_side(device):
    """Two captures on one stream, replayed on two: neither uses the other's scratch."""
    sets = [(_normal(device, 4096, 1024, dtype=BF16, seed=70 + i), _normal(device, 4096, 1024, dtype=BF16, seed=80 + i), torch.ones(1024, dtype=BF16, device=device)) for i in range(2)]
    want = [rms_norm_bwd(*s) for s in sets]
    side, graphs, got = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            got.append(rms_norm_bwd(*s))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            a[1].zero_()
        torch.cuda.synchronize()


def test_second_derivatives_are_refused(device):
    x, w = _normal(device, 4, 64, dtype=F32, seed=1).requires_grad_(), torch.ones(64, device=device, requires_grad=True)
    (g,) = torch.autograd.grad(rms_norm_apply(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# (the workspace is the call's own, so one per stream at least)
def test_two_streams_at_once(device):
    """The gradient's workspace is one per stream."""
    sets = [(_normal(device, 3000, 2048, dtype=BF16, seed=140 + i), _inputs(device, 3000, 2048, BF16, seed=150 + i)) for i in range(2)]
    want = [rms_norm_bwd(g, h, w) for g, (h, w, _) in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for st, (g, (h, w, _)) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(rms_norm_bwd(g, h, w))
    torch.cuda.synchronize()
    for i, (dx, dw) in enumerate(got):
        assert torch.equal(dx, want[i % 2][0]) and torch.equal(dw, want[i % 2][1])


def test_refusals(device):
    x, y, w = torch.zeros(4, 64, dtype=BF16, device=device), torch.zeros(4, 64, dtype=BF16, device=device), torch.ones(64, dtype=BF16, device=device)
    bad = [
        (ValueError, lambda: rms_norm(x, w[:60])), (TypeError, lambda: rms_norm(x, w.half())), (TypeError, lambda: rms_norm(x.double(), w.double())),
        (ValueError, lambda: rms_norm(x.t(), w[:4].contiguous())), (ValueError, lambda: rms_norm(x, w, residual=x[:2])), (ValueError, lambda: rms_norm(x, w, residual=x.float())),
        (ValueError, lambda: rms_norm(x, w, residual_out=x)), (TypeError, lambda: rms_norm(x, w, out=x.float())), (ValueError, lambda: rms_norm(x, w, out=x[:2])),
        (ValueError, lambda: rms_norm(x, w, out=x[:1].expand(4, 64))), (ValueError, lambda: rms_norm(x, w, eps=-1.0)), (ValueError, lambda: rms_norm(x, w[:1].expand(64))),
        (ValueError, lambda: rms_norm_fp8(x, w, scale_block=32)), (ValueError, lambda: rms_norm_fp8(x, w, scale=torch.zeros(3, device=device))),
        (ValueError, lambda: rms_norm_bwd(x[:3], x, w)), (ValueError, lambda: rms_norm_bwd(x.half(), x, w)), (ValueError, lambda: rms_norm_bwd(x, x, w, dweight=torch.zeros(64, dtype=BF16, device=device))),
        (ValueError, lambda: rms_norm(torch.zeros(1, _lib.NORM_MAX_WIDTH + 1, device=device), torch.zeros(_lib.NORM_MAX_WIDTH + 1, device=device))),
        (_lib.NativeCallError, lambda: rms_norm(x, w.cpu())), (TypeError, lambda: rms_norm(x, w, residual=1.0)), (ValueError, lambda: rms_norm(x, w, residual=x, out=y, residual_out=y)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            print("not refused:", i)


def test_native_launch_path_and_helpers_agree(device, monkeypatch):
    x, w, r = _inputs(device, 6, 320, BF16, seed=160)
    g = _normal(device, 6, 320, dtype=BF16, seed=170)
    host = ops.host
    assert host.rms_norm(x[:, :300], w[:300].contiguous(), None, 1e-6, False, 0, False) is None and host.rms_norm(x, w, None, -1.0, False, 0, False) is None
    assert host.rms_norm(x, w.half(), None, 1e-6, False, 0, False) is None and host.rms_norm(x, w, None, 1e-6, True, 64, False) is None
    assert host.rms_norm_bwd(g[:, :319], x, w, 1e-6, None) is None and host.rms_norm_bwd(g, x, w, 1e-6, g.float()) is None
    calls = [lambda: (rms_norm(x, w),), lambda: rms_norm(x.view(2, 3, 320), w, residual=r.view(2, 3, 320)), lambda: rms_norm_fp8(x, w, scale_block=128, pow2_scales=True),
             lambda: rms_norm_fp8(x.view(2, 3, 320), w, residual=r.view(2, 3, 320)), lambda: rms_norm_bwd(g, x, w), lambda: rms_norm_bwd(g, x, w, dh=r)]
    native = [c() for c in calls]

    class Declines:
        def __getattr__(self, name):
            return getattr(host, name) if "workspace" in name else (lambda *args: None)

    monkeypatch.setattr(ops, "host", Declines())
    for a, b in zip(native, [c() for c in calls]):
        assert len(a) == len(b) and all(s.shape == t.shape and s.dtype == t.dtype and torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block", [0, 128])
def test_power_of_two_scales_at_the_ends_of_float32(device, dtype, block):
    """Blocks (rows) whose largest value is next to float32's least numbers, beside ordinary ones: 448 * scale reaches it with the smallest
    power of two, 2^-149 at least.  y = (h w) s has an absolute error of at most 2^-149 there (two roundings of 2^-150, s <= 1) beside the relative one."""
    sizes = [1.0, 1e-30, 1e-35, 3e-36, 1e-36, 1e-37, 1e-38, 1e-40, 1e-42, 3e-44, 3e-45, 0.0]
    for widths in ([sizes] if block else [[c] for c in sizes]):
        x, w, _ = _inputs(device, 5, 128 * len(widths) if block else 333, dtype, F32, seed=200)
        for i, c in enumerate(widths):
            w[(slice(128 * i, 128 * (i + 1)) if block else slice(None))] *= c
        codes, scale = rms_norm_fp8(x, w, scale_block=block, pow2_scales=True)
        want, size = _plain(x, w, 1e-6), block or x.shape[1]
        per = (scale if block else scale[:, None]).double()
        amax = torch.stack([want[:, i:i + size].abs().amax(1) for i in range(0, x.shape[1], size)], 1)
        least = lambda a: torch.where(a > 0, torch.exp2(torch.ceil(torch.log2(a / 448)).clamp_min(-149)), torch.ones_like(a))
        off = amax * 40 * U + 2.0 ** -149 * (amax > 0)
        assert ((per >= least((amax - off).clamp_min(2.0 ** -150) * (amax > 0))) & (per <= least(amax + off))).all()
        spread = per.repeat_interleave(size, 1)[:, :x.shape[1]]
        v, off = want / spread, 2.0 ** -149 / spread
        slack = (v.abs() * 40 * U + off) * (1 + 1 / 16)
        assert ((_value(codes) - v).abs() <= torch.maximum(v.abs() / 16, torch.tensor(2.0 ** -10, device=device, dtype=torch.float64)) + slack).all()
    # no power of two reaches an infinite value: like the other scales, an infinite one, codes of 0, and NaN in its place
    w = torch.ones(256, device=device)
    w[130] = float("inf")
    codes, scale = rms_norm_fp8(x[:, :256].contiguous(), w, scale_block=block, pow2_scales=True)
    assert scale.reshape(5, -1)[:, -1].isinf().all() and _value(codes[:, 130]).isnan().all() and (_value(codes[:, 131:]) == 0).all()


def test_caller_owned_results_count_as_changed(device):
    """autograd refuses a backward pass whose saved rows were overwritten, as it does after a torch operation."""
    x, w, r = _inputs(device, 4, 96, BF16, seed=210)
    x.requires_grad_()
    y, h = rms_norm_apply(x, w, r)
    rms_norm(r, w, residual=r, residual_out=h.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    a, codes, scale, dx, dw = (torch.zeros(s, dtype=t, device=device) for s, t in (((4, 96), BF16), ((4, 96), torch.uint8), ((4,), F32), ((4, 96), BF16), ((96,), F32)))
    before = [t._version for t in (a, codes, scale, dx, dw)]
    rms_norm(r, w, out=a), rms_norm_fp8(r, w, codes=codes, scale=scale), rms_norm_bwd(r, r, w, dx=dx, dweight=dw)
    assert all(t._version > v for t, v in zip((a, codes, scale, dx, dw), before))
    with torch.inference_mode():
        assert rms_norm(r, w, out=torch.zeros_like(r)).shape == r.shape


def test_widths_beyond_32_bits_are_refused(device):
    x = torch.empty(1, (1 << 32) + 64, dtype=BF16, device=device)
    for call in (lambda: rms_norm(x, x[0]), lambda: rms_norm_fp8(x, x[0], scale_block=128), lambda: rms_norm_bwd(x, x, x[0])):
        with pytest.raises(ValueError, match="width"):
            call()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype, wdtype", [(F16, F16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("block", [0, 128])
@pytest.mark.parametrize("pow2", [False, True])
def test_codes_of_every_type(device, shape, dtype, wdtype, block, pow2):
    """float16 rows, and 16-bit rows with a float32 weight: the bounds of bfloat16 and float32 rows (h is exact in the comparison, the rest is float32)."""
    x, w, r = _inputs(device, *shape, dtype, wdtype, seed=9)
    codes, scale, h = rms_norm_fp8(x, w, eps=1e-6, residual=r, scale_block=block, pow2_scales=pow2)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    alone = rms_norm_fp8(h, w, eps=1e-6, scale_block=block, pow2_scales=pow2)
    assert torch.equal(alone[0], codes) and torch.equal(alone[1], scale)
    want, n, size = _plain(h, w, 1e-6), shape[1], block or shape[1]
    per = (scale if block else scale[:, None]).double()
    amax = torch.stack([want[:, i:i + size].abs().amax(1) for i in range(0, n, size)], 1)
    if pow2:
        least = lambda a: torch.exp2(torch.ceil(torch.log2(a / 448)))
        assert ((per >= least(amax * (1 - 40 * U))) & (per <= least(amax * (1 + 40 * U)))).all()
    else:
        assert ((per - amax / 448).abs() <= amax / 448 * 37 * U).all()
    v = want / per.repeat_interleave(size, 1)[:, :n]
    assert ((_value(codes) - v).abs() <= torch.maximum(v.abs() / 16, torch.tensor(2.0 ** -10, device=device, dtype=torch.float64)) + v.abs() * 43 * U).all()


@pytest.mark.parametrize("shape", SHAPES + [(513, 96), (2500, 64), (1027, 5000), (2049, 1000)])
@pytest.mark.parametrize("dtype, wdtype", [(BF16, F32), (F16, F16)])
@pytest.mark.parametrize("past", [False, True])
def test_gradients_of_every_type(device, shape, dtype, wdtype, past):
    test_gradients(device, shape, dtype, wdtype, past)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block", [0, 128])
def test_codes_in_the_middle_between_two_go_to_the_even_one(device, dtype, block):
    """y / scale = 448 h / max |h| whatever the row's factor: 3 / 64 of the largest are 21, between the codes 20 and 22, and 3 / 32 are 42."""
    top = torch.arange(1, 86, 2, device=device).float()[:, None]
    for n in (128, 640, 2048):
        x = torch.zeros(top.shape[0], n, device=device)
        x[:, 0::128], x[:, 1::128], x[:, 2::128] = top, top * (3 / 64), -top * (3 / 32)
        codes, scale = rms_norm_fp8(x.to(dtype), torch.ones(n, dtype=dtype, device=device), eps=1e-6, scale_block=block)
        v = _value(codes)
        assert (v[:, 0::128] == 448).all() and (v[:, 1::128] == 20).all() and (v[:, 2::128] == -40).all() and (v[:, 3:128] == 0).all()
