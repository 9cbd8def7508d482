"""GPU parity of the gated feed-forward block (16 bits with its gradients, e4m3) against the formulas in 64 bits.

Tolerances, U = 2^-24.  g and u are sums of K exact products in float32: off by at most K U of the sums of magnitudes (e4m3: three roundings of
scales more, and where the matrix instruction for e4m3 may run, into bfloat16, 7 * 2^-13 of the magnitudes: it drops what lies below 2^-13
of the largest of eight products).  s = 1 / (1 + 2^(-z log2 e)): z has up to four roundings, its product with log2 e two, so the
exponential is off by 6 |z| U and its own 2 U of itself, which reaches s as its share 1 - s; the sum and the reciprocal add 3 U: s is off
by e = (6 |z| (1 - s) + 5) U of itself.  y = g s u adds two products; an error of g reaches act(g) by its slope, at most 1.13.  The slope
s + g s (1 - s) z' has 1 - s, off by e s + U, and five roundings more of either term.  A result is rounded once, by eps(type) / 2 of itself
(float16 below 6e-5 by 2^-25); below 2^-126 the exponential's reciprocal is nothing.  float16 ends at 65504 = 2^16 - 2^5: from half a step further,
65520, values round to infinity, so an infinite result is right where the value may be that far."""

import math

import pytest
import torch

from cppmega_mlx_amd import _lib, ops
from cppmega_mlx_amd.nn.gated_ffn import fp8_gated_gemm, gated_gemm, gated_gemm_apply, gated_gemm_bwd
from cppmega_mlx_amd.nn.grouped_gemm import grouped_gemm, grouped_gemm_apply, grouped_gemm_bwd
from cppmega_mlx_amd.nn.rms_norm import rms_norm, rms_norm_fp8

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
TINY = {BF16: 2.0 ** -126, F16: 2.0 ** -25, F32: 2.0 ** -126}
DROPPED = 7 * 2.0 ** -13 / U
ACTIVATIONS = ["silu", "gelu_tanh"]


def _normal(device, *shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=device).manual_seed(seed), device=device).to(dtype)


def _offsets(counts, device, dtype=torch.int32):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=dtype, device=device)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _assert_within(got, want, bound, what=""):
    wide = got.double()
    if got.dtype == F16:
        far = wide.isinf() & (wide.sign() == want.sign()) & (want.abs() + bound >= 65520)
        wide = torch.where(far, want, wide)
    over = (wide - want).abs() - bound
    assert not got.isnan().any() and float(over.max() if over.numel() else 0.0) <= 0, (what, float(over.max()))


def _share(g, name):
    """(z, z', s, 1 - s) in 64 bits."""
    if name == "silu":
        z, dz = g, torch.ones_like(g)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        z, dz = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2)
    return z, dz, torch.sigmoid(z), torch.sigmoid(-z)


def _gated(p, size, terms, name):
    """y and its bound before the last rounding, from the products [T, 2 F] and their magnitudes."""
    n = p.shape[-1] // 2
    g, u, eg, eu = p[:, :n], p[:, n:], size[:, :n] * terms * U, size[:, n:] * terms * U
    z, _, s, r = _share(g, name)
    y = g * s * u
    # (the exponential is taken at the g of the kernel: |z| there is at most eg z' further on)
    share = (6 * (z.abs() + 8 * eg) * r + 7) * U
    return y, 1.13 * eg * (u.abs() + eu) + (g * s).abs() * eu + y.abs() * share * 1.01


def _products(x, w, offsets):
    p = torch.zeros(x.shape[0], w.shape[-2], dtype=torch.float64, device=x.device)
    size = torch.zeros_like(p)
    b = [0, x.shape[0]] if offsets is None else offsets.tolist()
    for e, (lo, hi) in enumerate(zip(b, b[1:])):
        m = (w if offsets is None else w[e]).double()
        p[lo:hi], size[lo:hi] = x[lo:hi].double() @ m.T, x[lo:hi].double().abs() @ m.abs().T
    return p, size


def _grads(dy, pre, x, w, offsets, name):
    """(dx, its bound, dw, its bound) from the products that were kept, before the last rounding."""
    n = dy.shape[1]
    g, u, d = pre[:, :n].double(), pre[:, n:].double(), dy.double()
    z, dz, s, r = _share(g, name)
    e = (6 * z.abs() * r + 5) * U
    slope = s + g * s * r * dz
    eslope = s * (e + U) + (g * dz).abs() * s * (r * (e + 6 * U) + e * s + 2 * U)
    grad = torch.cat([d * u * slope, d * g * s], 1)
    bound = torch.cat([(d * u).abs() * (eslope + 2 * U * slope.abs()), (d * g).abs() * s * (e + 3 * U)], 1) * 1.01
    bound += grad.abs() * _half(dy.dtype) * 1.01 + TINY[dy.dtype]
    b = [0, x.shape[0]] if offsets is None else offsets.tolist()
    dx, ex = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dw, ew = torch.zeros(w.shape, dtype=torch.float64, device=x.device), torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for i, (lo, hi) in enumerate(zip(b, b[1:])):
        if lo == hi:
            continue
        m, v = (w if offsets is None else w[i]).double(), x[lo:hi].double()
        at = (slice(None),) if offsets is None else (i,)
        dx[lo:hi], dw[at] = grad[lo:hi] @ m, grad[lo:hi].T @ v
        ex[lo:hi] = bound[lo:hi] @ m.abs() + 2 * n * U * ((grad[lo:hi].abs() + bound[lo:hi]) @ m.abs())
        ew[at] = bound[lo:hi].T @ v.abs() + (hi - lo) * U * ((grad[lo:hi].abs() + bound[lo:hi]).T @ v.abs())
    return dx, ex, dw, ew


def _rounded(want, bound, dtype):
    return bound + (want.abs() + bound) * _half(dtype) + TINY[dtype]


# counts of rows (None: one matrix), outputs, channels: one of everything, empty experts, tiles that end everywhere, odd and unaligned sizes, long sums
CASES = [
    ([1], 1, 1), ([1], 64, 8), ([3], 33, 7), ([0, 5, 0, 0, 2, 0], 40, 24), ([1] * 8, 256, 128), ([64], 128, 64), ([65, 0, 63], 129, 136), ([17, 128, 1, 129], 100, 200),
    ([300, 3, 0, 511], 192, 320), ([100, 7], 250, 333), ([256, 512], 132, 256), ([40] * 3 + [0] * 90 + [33] * 5, 68, 72), ([2, 0, 1], 500, 4096),
    ([600, 1, 257], 768, 1024), ([0, 0, 0], 64, 64), ([16, 32, 48, 15, 33, 1, 64], 260, 1536), ([9] * 130, 32, 40), (None, 1001, 520), (None, 36, 24), ([2600, 0, 900, 37], 1300, 144),
]


def _rows(counts):
    return 333 if counts is None else sum(counts)


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{_rows(c[0])}x{len(c[0]) if c[0] else 0}x{c[1]}x{c[2]}")
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("name", ACTIVATIONS)
def test_block_and_gradients(device, case, dtype, name):
    _check_block(device, case, dtype, name)


def _check_block(device, case, dtype, name):
    counts, n, k = case
    rows = _rows(counts)
    offsets = None if counts is None else _offsets(counts, device)
    lead = () if counts is None else (len(counts),)
    x, w = _normal(device, rows, k, dtype=dtype, seed=1), (_normal(device, *lead, 2 * n, k, seed=2) * (2.0 * k ** -0.5)).to(dtype)
    dy = _normal(device, rows, n, dtype=dtype, seed=3)
    y = gated_gemm(x, w, offsets, activation=name)
    assert y.dtype == dtype and y.shape == (rows, n)
    p, size = _products(x, w, offsets)
    want, bound = _gated(p, size, k, name)
    _assert_within(y, want, _rounded(want, bound, dtype))
    # keeping the products changes nothing; float32 results hold the same values, from int64 offsets
    pre = torch.empty(rows, 2 * n, dtype=dtype, device=device)
    assert torch.equal(gated_gemm(x, w, offsets, activation=name, pre=pre), y)
    _assert_within(pre, p, p.abs() * _half(dtype) + size * (k * U) * 1.01 + TINY[dtype])
    wide, wide_pre = torch.empty(rows, n, device=device), torch.empty(rows, 2 * n, device=device)
    again = None if offsets is None else offsets.long()
    assert gated_gemm(x, w, again, activation=name, out=wide, pre=wide_pre) is wide
    assert torch.equal(wide.to(dtype), y) and torch.equal(wide_pre.to(dtype), pre)
    _assert_within(wide, want, _rounded(want, bound, F32))
    # gradients, from kept products of either type
    for kept in (pre, wide_pre):
        dx, dw = gated_gemm_bwd(dy, kept, x, w, offsets, activation=name)
        wx, ex, ww, ew = _grads(dy, kept, x, w, offsets, name)
        assert dx.dtype == dw.dtype == dtype and dw.shape == w.shape
        _assert_within(dx, wx, _rounded(wx, ex, dtype), "dx")
        _assert_within(dw, ww, _rounded(ww, ew, dtype), "dw")
    for e, c in enumerate(counts or ()):
        assert c or (dw[e] == 0).all()
    fx, fw = gated_gemm_bwd(dy, kept, x, w, again, activation=name, dx=torch.empty(rows, k, device=device), dw=torch.empty(w.shape, device=device))
    assert torch.equal(fx.to(dtype), dx) and torch.equal(fw.to(dtype), dw)
    assert torch.equal(gated_gemm_bwd(dy, kept, x, w, offsets, activation=name, need_dw=False)[0], dx)
    assert torch.equal(gated_gemm_bwd(dy, kept, x, w, offsets, activation=name, need_dx=False)[1], dw)


# outputs in more than one block of the gradients' kernel, one expert's weights in several passes, few tiles with a long contraction
MORE_CASES = [([5, 0, 30], 2100, 64), ([3], 4099, 24), ([200], 512, 2048), ([700, 0, 300], 520, 1544), ([129], 1000, 776), ([1, 640], 1111, 512)]


@pytest.mark.parametrize("case", MORE_CASES, ids=lambda c: f"{_rows(c[0])}x{len(c[0])}x{c[1]}x{c[2]}")
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_wide_blocks_and_few_tiles(device, case, dtype):
    _check_block(device, case, dtype, "silu" if dtype == BF16 else "gelu_tanh")


FP8_CASES = [([1], 5, 16), ([1] * 8, 256, 128), ([3, 0, 2], 100, 384), ([17, 128, 1, 129], 200, 272), ([300, 3, 0, 511], 192, 640), (None, 130, 200), (None, 257, 129),
             ([40] * 3 + [0] * 90 + [33] * 5, 68, 144), ([600, 1, 257], 384, 1024), ([700, 260], 129, 2048), ([2600, 0, 900, 37], 1300, 256)]
MORE_FP8_CASES = [([1000], 1000, 1040), ([100], 1100, 784), ([60], 500, 2048), ([333, 0, 64], 300, 1552)]


@pytest.mark.parametrize("case", FP8_CASES, ids=lambda c: f"{_rows(c[0])}x{len(c[0]) if c[0] else 0}x{c[1]}x{c[2]}")
@pytest.mark.parametrize("block", [0, 128])
def test_fp8_block(device, case, block):
    _check_fp8_block(device, case, block)


@pytest.mark.parametrize("case", MORE_FP8_CASES, ids=lambda c: f"{_rows(c[0])}x{len(c[0])}x{c[1]}x{c[2]}")
@pytest.mark.parametrize("block", [0, 128])
def test_fp8_few_tiles(device, case, block):
    _check_fp8_block(device, case, block)


def _check_fp8_block(device, case, block):
    counts, n, k = case
    rows = _rows(counts)
    offsets = None if counts is None else _offsets(counts, device)
    lead = () if counts is None else (len(counts),)
    bn, bk = (n + 127) // 128, (k + 127) // 128

    def codes(*shape, seed):
        return (_normal(device, *shape, seed=seed) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)

    x, w = codes(rows, k, seed=1), codes(*lead, 2 * n, k, seed=2)
    xs = torch.exp(_normal(device, *((rows, bk) if block else (rows,)), seed=3))
    ws = torch.exp(_normal(device, *lead, 2, bn, bk, seed=4)) * (2.0 / 3600 / k ** 0.5)
    wide_x = x.view(torch.float8_e4m3fn).double() * (xs.double().repeat_interleave(128, 1)[:, :k] if block else xs.double()[:, None])
    scale = ws.double().repeat_interleave(128, -2)[..., :n, :].flatten(-3, -2).repeat_interleave(128, -1)[..., :k]
    p, size = _products(wide_x, w.view(torch.float8_e4m3fn).double() * scale, offsets)
    for name in ACTIVATIONS:
        for dtype in (BF16, F16, F32):
            out = torch.empty(rows, n, dtype=dtype, device=device)
            assert fp8_gated_gemm(x, xs, w, ws, offsets, activation=name, out=out) is out
            want, bound = _gated(p, size, k + 3 + (DROPPED if dtype == BF16 else 0), name)
            _assert_within(out, want, _rounded(want, bound, dtype), (name, dtype))
            if dtype == BF16:
                assert torch.equal(fp8_gated_gemm(x, xs, w, ws, offsets, activation=name), out)
                if offsets is not None:
                    assert torch.equal(fp8_gated_gemm(x, xs, w, ws, offsets.long(), activation=name), out)


@pytest.mark.parametrize("shape", [(9, 24, 40), (700, 160, 192), (300, 33, 65)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_views_tails_and_experts_without_rows(device, shape, dtype):
    """Rows of a pitch of their own, NaN in every place that no row owns, an empty expert's weights and rows behind the last expert."""
    rows, n, k = shape
    counts, tail = [rows // 2, 0, rows - rows // 2], 70
    offsets = _offsets(counts, device)
    clean = [_normal(device, rows, k, dtype=dtype, seed=1), (_normal(device, 3, 2 * n, k, seed=2) * k ** -0.5).to(dtype), _normal(device, rows, n, dtype=dtype, seed=3)]
    pre = torch.empty(rows, 2 * n, dtype=dtype, device=device)
    y = gated_gemm(clean[0], clean[1], offsets, pre=pre)
    dx, dw = gated_gemm_bwd(clean[2], pre, clean[0], clean[1], offsets)
    w = clean[1].clone()
    w[1] = float("nan")
    for shift in (0, 1, 8):
        def held(t, value=float("nan")):
            big = torch.full((rows + tail, t.shape[1] + 17), value, dtype=t.dtype, device=device)
            view = big[:, shift:shift + t.shape[1]]
            view[:rows] = t
            return big, view

        _, xv = held(clean[0])
        _, dv = held(clean[2])
        big_y, yv = held(torch.zeros_like(y), 7.0)
        big_p, pv = held(torch.zeros_like(pre), 7.0)
        big_x, gv = held(torch.zeros_like(dx), 7.0)
        got = gated_gemm(xv, w, offsets, out=yv, pre=pv)
        assert got is yv
        gw = torch.empty_like(w)
        gated_gemm_bwd(dv, pv, xv, w, offsets, dx=gv, dw=gw)
        for big, view, want in ((big_y, yv, y), (big_p, pv, pre), (big_x, gv, dx)):
            assert torch.isfinite(view).all()
            # (another kernel may add in another order: the types' rounding and K sums of order one)
            assert (view[:rows].double() - want.double()).abs().max() <= (2 * _half(dtype) + 4 * 2 * max(n, k) * U) * max(1.0, float(want.double().abs().max())) * 4
            view[:rows] = 7.0
            assert (big == 7.0).all()
        assert torch.isfinite(gw).all() and (gw[1] == 0).all()
        fresh = gated_gemm(xv, w, offsets)
        assert (fresh[rows:] == 0).all() and torch.isfinite(fresh).all()
        fresh_x, fresh_w = gated_gemm_bwd(dv, torch.cat([pre, torch.full((tail, 2 * n), float("nan"), dtype=dtype, device=device)]), xv, w, offsets)
        assert (fresh_x[rows:] == 0).all() and torch.isfinite(fresh_x).all() and torch.isfinite(fresh_w).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("name", ACTIVATIONS)
def test_far_gates(device, dtype, name):
    """Gates from far below to far above zero: no NaN, shares of nothing and of everything."""
    big = 3e4 if dtype == F16 else 1e18
    g = torch.tensor([-big, -100.0, -88.0, -20.0, -1.5, -1.28, -1e-4, 0.0, 1e-4, 1.0, 17.0, 90.0, big], dtype=dtype, device=device)
    n = g.numel()
    x = torch.eye(n, dtype=dtype, device=device)                   # row i: gate g[i] for every output, up 1
    w = torch.cat([g.repeat(n, 1), torch.ones(n, n, dtype=dtype, device=device)])
    pre = torch.empty(n, 2 * n, dtype=dtype, device=device)
    y = torch.empty(n, n, device=device)
    gated_gemm(x, w, activation=name, out=y, pre=pre)
    p, size = _products(x, w, None)
    want, bound = _gated(p, size, 0, name)                         # (one product and zeros: exact)
    _assert_within(y, want, _rounded(want, bound, F32) + p[:, :n].abs() * 2.0 ** -120)
    assert torch.equal(pre.double(), p)
    dy = torch.ones(n, n, dtype=dtype, device=device)
    dx, dw = gated_gemm_bwd(dy, pre, x, w, activation=name, dw=torch.empty(w.shape, device=device))
    assert torch.isfinite(dw).all()
    _, _, ww, ew = _grads(dy, pre, x, w, None, name)
    _assert_within(dw, ww, _rounded(ww, ew, F32) + pre[:, :n].double().abs().T.repeat(2, 1) * 2.0 ** -120)


def test_gradients_are_those_of_differences(device):
    rows, n, k = 14, 24, 16
    offsets = _offsets([9, 0, 5], device)
    x, w = _normal(device, rows, k, dtype=F16, seed=5) * 0.5, _normal(device, 3, 2 * n, k, dtype=F16, seed=6) * 0.5
    dy = _normal(device, rows, n, dtype=F16, seed=7)
    pre = torch.empty(rows, 2 * n, device=device)
    gated_gemm(x, w, offsets, activation="gelu_tanh", pre=pre)
    dx, dw = gated_gemm_bwd(dy, pre, x, w, offsets, activation="gelu_tanh", dx=torch.empty(rows, k, device=device), dw=torch.empty(w.shape, device=device))

    def loss(a, b):
        p, _ = _products(a, b, offsets)
        return float((_gated(p, p, 0, "gelu_tanh")[0] * dy.double()).sum())

    # central differences of the formula in 64 bits: their own error is h^2 times a third derivative of order |x|^3, below 1e-6
    h = 1e-4
    for t, grad, at in ((x, dx, (3, 5)), (x, dx, (13, 0)), (w, dw, (0, 4, 7)), (w, dw, (2, n + 3, 2)), (w, dw, (1, 0, 0))):
        up, down = t.double().clone(), t.double().clone()
        up[at] += h
        down[at] -= h
        other = (lambda v: (v, w.double())) if t is x else (lambda v: (x.double(), v))
        slope = (loss(*other(up)) - loss(*other(down))) / (2 * h)
        # dg and du are rounded to float16: each of the 2 n (or 9) terms by half a step, of magnitude below 8
        assert abs(slope - float(grad[at])) <= 8 * 2 * n * 2.0 ** -11 * 0.25 + 1e-6


def _check_autograd(device, y, x, w, offsets, act, kept):
    assert torch.equal(y, gated_gemm(x.detach(), w.detach(), offsets, activation=act)) and (y[42:] == 0).all()
    g = _normal(device, *y.shape, dtype=BF16, seed=3)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    pre = torch.empty(y.shape[0], 2 * y.shape[1], dtype=kept, device=device)
    gated_gemm(x.detach(), w.detach(), offsets, activation=act, pre=pre)
    want = gated_gemm_bwd(g, pre, x.detach(), w.detach(), offsets, activation=act)
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])


def test_autograd(device):
    rows, n, k = 50, 40, 48
    offsets = _offsets([20, 0, 22], device)
    x, w = _normal(device, rows, k, dtype=BF16, seed=1).requires_grad_(), (_normal(device, 3, 2 * n, k, seed=2) * 0.2).to(BF16).requires_grad_()
    for act in ACTIVATIONS:
        for kept in (F32, BF16):
            y = gated_gemm_apply(x, w, offsets, activation=act, pre_dtype=kept)
            _check_autograd(device, y, x, w, offsets, act, kept)
    d = w.detach()[0].contiguous()
    gated_gemm_apply(x, d).sum().backward()                        # (a broadcast cotangent, one matrix, no gradient of the weight)
    pre = torch.empty(rows, 2 * n, device=device)
    gated_gemm(x.detach(), d, pre=pre)
    assert torch.equal(x.grad, gated_gemm_bwd(torch.ones(rows, n, dtype=BF16, device=device), pre, x.detach(), d, need_dw=False)[0])
    (g,) = torch.autograd.grad(gated_gemm_apply(x, d).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_nothing_is_kept_without_gradients(device):
    x, w = _normal(device, 70, 64, dtype=BF16, seed=1), (_normal(device, 96, 64, seed=2) * 0.2).to(BF16).requires_grad_()
    want = gated_gemm(x, w.detach())
    base = torch.cuda.memory_allocated(device)
    with torch.no_grad():
        y = gated_gemm_apply(x, w)
    z = gated_gemm_apply(x, w.detach())
    assert torch.equal(y, want) and torch.equal(z, want) and not y.requires_grad and not z.requires_grad
    kept = torch.cuda.memory_allocated(device) - base
    assert kept <= 2 * 70 * 48 * 2 + 2 * 512                       # (two results, in units of 512 bytes)
    assert torch.equal(gated_gemm_apply(x, w), want) and gated_gemm_apply(x, w).requires_grad


def test_one_matrix_is_one_expert(device):
    x, w, dy = _normal(device, 200, 64, dtype=BF16, seed=1), (_normal(device, 96, 64, seed=2) * 0.2).to(BF16), _normal(device, 200, 48, dtype=BF16, seed=3)
    offsets = _offsets([200], device)
    pre = torch.empty(200, 96, dtype=BF16, device=device)
    assert torch.equal(gated_gemm(x, w, pre=pre), gated_gemm(x, w[None], offsets))
    a, b = gated_gemm_bwd(dy, pre, x, w), gated_gemm_bwd(dy, pre, x, w[None], offsets)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1][0])


@pytest.mark.parametrize("values", [[0, 9, 4, 60], [0, 3, 2 ** 30, 5], [5, -7, 40, 40], [40, 40, 40, 40], [0, 0, 0, -1]], ids=str)
def test_offsets_that_break_the_rules_stay_inside(device, values):
    """Unspecified values, no access outside: the places around the outputs keep theirs."""
    rows, n, k = 40, 48, 64
    x, w, dy = _normal(device, rows, k, dtype=BF16, seed=1), _normal(device, 3, 2 * n, k, dtype=BF16, seed=2), _normal(device, rows, n, dtype=BF16, seed=3)
    off = torch.tensor(values, dtype=torch.int64, device=device)
    y, pre = torch.full((rows + 2, n), 7.0, dtype=BF16, device=device), torch.full((rows + 2, 2 * n), 7.0, dtype=BF16, device=device)
    gated_gemm(x, w, off, out=y[1:-1], pre=pre[1:-1])
    dx, dw = torch.full((rows + 2, k), 7.0, dtype=BF16, device=device), torch.full((5, 2 * n, k), 7.0, dtype=BF16, device=device)
    gated_gemm_bwd(dy, pre[1:-1], x, w, off, dx=dx[1:-1], dw=dw[1:-1])
    for t in (y, pre, dx, dw):
        assert (t[0] == 7).all() and (t[-1] == 7).all()


def test_graphs_replay_with_other_rows(device):
    """Captured calls read their operands and offsets at replay; graphs that share a stream have scratch of their own."""
    rows, n, k = 96, 64, 128
    x, w, dy = _normal(device, rows, k, dtype=BF16, seed=1), (_normal(device, 4, 2 * n, k, seed=2) * 0.1).to(BF16), _normal(device, rows, n, dtype=BF16, seed=3)
    x8 = _normal(device, rows, k, seed=4).to(torch.float8_e4m3fn).view(torch.uint8)
    w8 = _normal(device, 4, 2 * n, k, seed=5).to(torch.float8_e4m3fn).view(torch.uint8)
    xs, ws = torch.ones(rows, device=device), torch.full((4, 2, 1, 1), 0.1, device=device)
    off = _offsets([30, 0, 40, 26], device)

    def call():
        pre = torch.empty(rows, 2 * n, dtype=BF16, device=device)
        y = gated_gemm(x, w, off, pre=pre)
        return (y, *gated_gemm_bwd(dy, pre, x, w, off), fp8_gated_gemm(x8, xs, w8, ws, off))

    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for i, counts in enumerate([[30, 0, 40, 26], [96, 0, 0, 0], [1, 2, 3, 4], [0, 0, 0, 0]]):
        off.copy_(_offsets(counts, device))
        x.copy_(_normal(device, rows, k, dtype=BF16, seed=20 + i))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = call()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_streams(device):
    """Calls on several streams at once, operands made on another one."""
    sets = []
    for i in range(3):
        x, w = _normal(device, 300, 256, dtype=BF16, seed=i), (_normal(device, 2, 512, 256, seed=9 + i) * 0.1).to(BF16)
        sets.append((x, w, _offsets([100, 200], device), _normal(device, 300, 256, dtype=BF16, seed=30 + i)))

    def step(x, w, off, dy):
        pre = torch.empty(300, 512, dtype=BF16, device=device)
        return (gated_gemm(x, w, off, pre=pre), *gated_gemm_bwd(dy, pre, x, w, off))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in sets]
    for _ in range(3):
        got = []
        for stream, s in zip(streams, sets):
            stream.wait_stream(torch.cuda.current_stream(device))
            with torch.cuda.stream(stream):
                got.append(step(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_the_native_path_and_the_helpers_agree(device, monkeypatch):
    x, w, dy = _normal(device, 60, 128, dtype=F16, seed=1), (_normal(device, 2, 192, 128, seed=2) * 0.1).to(F16), _normal(device, 60, 96, dtype=F16, seed=3)
    x8, w8 = x.float().to(torch.float8_e4m3fn).view(torch.uint8), w.float().to(torch.float8_e4m3fn).view(torch.uint8)
    xs, ws = torch.ones(60, 1, device=device), torch.ones(2, 2, 1, 1, device=device)
    off = _offsets([33, 27], device)

    def call():
        pre = torch.empty(60, 192, dtype=F16, device=device)
        y = gated_gemm(x, w, off, activation="gelu_tanh", pre=pre)
        wide = torch.empty(60, 192, device=device)
        kept = (gated_gemm(x, w, off, activation="gelu_tanh", pre=wide), wide, *gated_gemm_bwd(dy, wide, x, w, off, activation="gelu_tanh"))
        return (y, pre, *gated_gemm_bwd(dy, pre, x, w, off, activation="gelu_tanh"), fp8_gated_gemm(x8, xs, w8, ws, off), fp8_gated_gemm(x8, xs[:, 0].contiguous(), w8[0], ws[0]), *kept)

    native = call()
    host = ops.host
    assert host.gated_gemm(x[:, ::2], w, off, 0, None) is None and host.gated_gemm(x, w.bfloat16(), off, 0, None) is None and host.gated_gemm(x, w, None, 0, None) is None
    wide = native[7]
    assert wide.dtype == F32 and host.gated_gemm(x, w, off, 0, wide) is not None and host.gated_gemm_bwd(dy, wide, x, w, off, 0) is not None
    assert host.gated_gemm(x, w, off, 0, wide.double()) is None and host.gated_gemm_bwd(dy.float(), wide, x, w, off, 0) is None
    assert host.gated_gemm(x, w, off, 5, None) is None and host.gated_gemm_bwd(dy[:9], native[1], x, w, off, 0) is None and host.fp8_gated_gemm(x8, xs, w8, ws[:1], off, 0) is None
    monkeypatch.setattr(ops, "host", type("Declines", (), {"__getattr__": lambda self, name: lambda *a: None})())
    for a, b in zip(native, call()):
        assert torch.equal(a, b)


def test_versions(device):
    x, w, off = _normal(device, 9, 16, dtype=BF16, seed=1), _normal(device, 2, 32, 16, dtype=BF16, seed=2), _offsets([4, 5], device)
    pre, out = torch.empty(9, 32, dtype=BF16, device=device), torch.empty(9, 16, dtype=BF16, device=device)
    before = pre._version
    gated_gemm(x, w, off, pre=pre)
    assert pre._version > before
    versions = pre._version, out._version
    gated_gemm(x, w, off, out=out, pre=pre)
    assert pre._version > versions[0] and out._version > versions[1]
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    gated_gemm_bwd(out, pre, x, w, off, dx=dx, dw=dw)
    assert dx._version == 1 and dw._version == 1
    # a graph that has saved a tensor which a later call overwrites refuses its backward pass
    y = gated_gemm_apply(x, w.requires_grad_(), off)
    grouped_gemm(torch.ones_like(x), torch.ones(2, 16, 16, dtype=BF16, device=device), off, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals(device):
    x, w, dy = _normal(device, 8, 32, dtype=BF16), _normal(device, 2, 32, 32, dtype=BF16), _normal(device, 8, 16, dtype=BF16)
    off, pre = _offsets([3, 5], device), torch.empty(8, 32, dtype=BF16, device=device)
    x8, w8 = torch.zeros(8, 32, dtype=torch.uint8, device=device), torch.zeros(2, 32, 32, dtype=torch.uint8, device=device)
    xs, ws = torch.ones(8, device=device), torch.ones(2, 2, 1, 1, device=device)
    for error, call in [
        (ValueError, lambda: gated_gemm(x, w, off, activation="relu")), (ValueError, lambda: gated_gemm(x, w)), (ValueError, lambda: gated_gemm(x, w[0], off)),
        (ValueError, lambda: gated_gemm(x, w[:, :31].contiguous(), off)), (TypeError, lambda: gated_gemm(x.float(), w.float(), off)), (TypeError, lambda: gated_gemm(x, w.half(), off)),
        (ValueError, lambda: gated_gemm(x, w[:, :, :30], off)), (ValueError, lambda: gated_gemm(x[:, :30], w, off)), (ValueError, lambda: gated_gemm(x, w, off[:2])), (TypeError, lambda: gated_gemm(x, w, off.float())),
        (_lib.NativeCallError, lambda: gated_gemm(x, w, off.cpu())), (TypeError, lambda: gated_gemm(x, w, off, out=dy.half())), (ValueError, lambda: gated_gemm(x, w, off, out=pre)),
        (ValueError, lambda: gated_gemm(x, w, off, out=dy[:1].expand(8, 16))), (ValueError, lambda: gated_gemm(x, w, off, pre=dy)), (TypeError, lambda: gated_gemm(x, w, off, pre=pre.half())),
        (ValueError, lambda: gated_gemm(x, w, off, pre=pre[:1].expand(8, 32))), (ValueError, lambda: gated_gemm_bwd(dy[:4], pre, x, w, off)), (TypeError, lambda: gated_gemm_bwd(dy.half(), pre, x, w, off)),
        (ValueError, lambda: gated_gemm_bwd(dy, pre[:, :16], x, w, off)), (TypeError, lambda: gated_gemm_bwd(dy, pre.half(), x, w, off)), (ValueError, lambda: gated_gemm_bwd(dy, pre, x, w, off, dw=w[0])),
        (ValueError, lambda: gated_gemm_bwd(dy, pre, x, w, off, dx=dy)), (ValueError, lambda: gated_gemm_bwd(dy, pre, x, w, off, activation="tanh")),
        (TypeError, lambda: fp8_gated_gemm(x, xs, w8, ws, off)), (TypeError, lambda: fp8_gated_gemm(x8, xs, w, ws, off)), (ValueError, lambda: fp8_gated_gemm(x8, xs[:4], w8, ws, off)),
        (ValueError, lambda: fp8_gated_gemm(x8, xs, w8, ws[:, :1], off)), (TypeError, lambda: fp8_gated_gemm(x8, xs.double(), w8, ws, off)), (TypeError, lambda: ops.gated_gemm(x8, w8, off, activation="silu", out=dy, pre=pre, x_scale=xs, w_scale=ws)),
        (_lib.NativeCallError, lambda: gated_gemm(x, torch.zeros(513, 4, 32, dtype=BF16, device=device), torch.zeros(514, dtype=torch.int32, device=device))),
    ]:
        with pytest.raises(error):
            call()
    assert gated_gemm(x[:0], w, off * 0).shape == (0, 16)
    dx, dw = gated_gemm_bwd(dy[:0], pre[:0], x[:0], w, off * 0)
    assert dx.shape == (0, 32) and (dw == 0).all()
    assert gated_gemm_bwd(dy, pre, x, w, off, need_dx=False, need_dw=False) == (None, None)


def test_a_layer_runs_through(device):
    """Norm, gated block and down projection of a training step, forward and backward, against 64 bits; the same by expert in 8 bits."""
    rows, k, f = 120, 64, 96
    offsets = _offsets([50, 0, 70], device)
    h, gain = _normal(device, rows, k, dtype=BF16, seed=1), (1 + 0.1 * _normal(device, k, seed=2)).to(BF16)
    up, down = (_normal(device, 3, 2 * f, k, seed=3) * 0.2).to(BF16), (_normal(device, 3, k, f, seed=4) * 0.2).to(BF16)
    x = rms_norm(h, gain)
    x.requires_grad_()
    up.requires_grad_()
    down.requires_grad_()
    mid = gated_gemm_apply(x, up, offsets)
    out = grouped_gemm_apply(mid, down, offsets)
    g = _normal(device, rows, k, dtype=BF16, seed=5)
    out.backward(g)
    # the formulas over the values that the launches hand on
    p, size = _products(x.detach(), up.detach(), offsets)
    want, bound = _gated(p, size, k, "silu")
    _assert_within(mid.detach(), want, _rounded(want, bound, BF16))
    dmid = grouped_gemm_bwd(g, mid.detach(), down.detach(), offsets, need_dw=False)[0]
    pre = torch.empty(rows, 2 * f, dtype=BF16, device=device)
    gated_gemm(x.detach(), up.detach(), offsets, pre=pre)
    wx, ex, ww, ew = _grads(dmid, pre, x.detach(), up.detach(), offsets, "silu")
    _assert_within(x.grad, wx, _rounded(wx, ex, BF16))
    _assert_within(up.grad, ww, _rounded(ww, ew, BF16))
    # 8 bits
    codes, scale = rms_norm_fp8(h, gain)
    w8, ws = up.detach().float().mul(64).to(torch.float8_e4m3fn).view(torch.uint8), torch.full((3, 2, 1, 1), 1 / 64, device=device)
    y8 = fp8_gated_gemm(codes, scale, w8, ws, offsets)
    wide = codes.view(torch.float8_e4m3fn).double() * (scale.double()[:, None] if scale.ndim == 1 else scale.double().repeat_interleave(128, 1)[:, :k])
    p, size = _products(wide, w8.view(torch.float8_e4m3fn).double() / 64, offsets)
    want, bound = _gated(p, size, k + 3 + DROPPED, "silu")
    _assert_within(y8, want, _rounded(want, bound, BF16))


def test_products_beyond_32_bits(device):
    """Kept products and gradients of more than 2^32 bytes: rows repeat, and their results with them."""
    rows, n, k = 270336, 2048, 64
    x, dy = _normal(device, 1024, k, dtype=BF16, seed=1), _normal(device, 1024, n, dtype=BF16, seed=2)
    w = (_normal(device, 2 * n, k, seed=3) * 0.2).to(BF16)
    pre = torch.empty(rows, 2 * n, device=device)
    many = x.repeat(rows // 1024, 1)
    y = gated_gemm(many, w, pre=pre)
    p, size = _products(x, w, None)
    want, bound = _gated(p, size, k, "silu")
    _assert_within(y[:1024], want, _rounded(want, bound, BF16))
    _assert_within(pre[:1024], p, _rounded(p, size * (k * U) * 1.01, F32))
    dx, _ = gated_gemm_bwd(dy.repeat(rows // 1024, 1), pre, many, w, need_dw=False)
    wx, ex, _, _ = _grads(dy, pre[:1024], x, w, None, "silu")
    _assert_within(dx[:1024], wx, _rounded(wx, ex, BF16))
    for t in (y, pre, dx):
        assert all(torch.equal(t[at:at + 1024], t[:1024]) for at in range(1024, rows, 1024))
