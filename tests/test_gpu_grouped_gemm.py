"""GPU parity of the products grouped by expert (rows, both gradients, 8 bits) against the formulas in 64 bits.

Tolerances.  A product of two 16-bit or e4m3 values is exact in float32; a sum of K of them in any order is off by at most K * 2^-24 of
the sum of their magnitudes (the scales of e4m3 blocks: three roundings more); the result is rounded once, by eps(type) / 2 of
itself (float16 below 6e-5 by 2^-25).  bfloat16 results of e4m3 operands may come from the matrix instruction for e4m3: it aligns eight
products to the largest and drops what lies below 2^-13 of it (one product of 2^8 and one of 2^-5 add up, one of 2^-6 is lost; the
largest itself has 8 bits), so eight products are off by less than 7 * 2^-13 of the largest, which is at most their magnitudes' sum."""

import pytest
import torch

from cppmega_mlx_amd import _lib, ops
from cppmega_mlx_amd.nn.grouped_gemm import grouped_fp8_gemm, grouped_gemm, grouped_gemm_apply, grouped_gemm_bwd
from cppmega_mlx_amd.nn.rms_norm import rms_norm, rms_norm_apply, rms_norm_bwd, rms_norm_fp8

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
TINY = {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0}
DROPPED = 7 * 2.0 ** -13 / U                # the same as a number of roundings


def _normal(device, *shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=device).manual_seed(seed), device=device).to(dtype)


def _offsets(counts, device, dtype=torch.int32):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=dtype, device=device)


def _assert_near(got, want, size, terms):
    bound = want.abs() * (torch.finfo(got.dtype).eps / 2) + size * terms * U + TINY[got.dtype]
    over = (got.double() - want).abs() - bound
    assert not got.isnan().any() and float(over.max() if over.numel() else 0.0) <= 0, float(over.max())


def _plain(x, w, offsets):
    """(y, sums of magnitudes) per row of the experts; rows behind them are zeros."""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    b = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(b, b[1:])):
        y[lo:hi], size[lo:hi] = x[lo:hi].double() @ w[e].double().T, x[lo:hi].double().abs() @ w[e].double().abs().T
    return y, size


# counts of rows, n, k: one row, empty experts, tiles that end everywhere, odd and unaligned sizes, long sums, many experts
CASES = [
    ([1], 1, 1), ([1], 64, 8), ([3], 33, 7), ([0, 5, 0, 0, 2, 0], 40, 24), ([1, 1, 1, 1, 1, 1, 1, 1], 256, 128), ([64], 128, 64), ([65, 0, 63], 129, 136),
    ([17, 128, 1, 129], 257, 200), ([300, 3, 0, 511], 384, 320), ([100, 7], 501, 333), ([256, 512], 512, 256), ([40] * 3 + [0] * 90 + [33] * 5, 130, 72),
    ([2, 0, 1], 1000, 4096), ([600, 1, 257], 1536, 1024), ([0, 0, 0], 64, 64), ([16, 32, 48, 15, 33, 1, 64], 520, 1536), ([9] * 130, 64, 40), ([31, 250], 72, 2056),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{sum(c[0])}x{len(c[0])}x{c[1]}x{c[2]}")
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_and_gradients(device, case, dtype):
    counts, n, k = case
    offsets = _offsets(counts, device)
    rows = sum(counts)
    x, w, dy = _normal(device, rows, k, dtype=dtype, seed=1), _normal(device, len(counts), n, k, dtype=dtype, seed=2), _normal(device, rows, n, dtype=dtype, seed=3)
    y = grouped_gemm(x, w, offsets)
    assert y.dtype == dtype and y.shape == (rows, n)
    _assert_near(y, *_plain(x, w, offsets), k)
    dx, dw = grouped_gemm_bwd(dy, x, w, offsets)
    assert dx.dtype == dw.dtype == dtype
    _assert_near(dx, *_plain(dy, w.transpose(1, 2), offsets), n)
    b = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(b, b[1:])):
        g, v = dy[lo:hi].double().T, x[lo:hi].double()
        _assert_near(dw[e], g @ v, g.abs() @ v.abs(), hi - lo)
        if lo == hi:
            assert (dw[e] == 0).all()
    # the same values into float32, from int64 offsets
    wide = torch.empty(rows, n, device=device)
    assert grouped_gemm(x, w, offsets.long(), out=wide) is wide and torch.equal(wide.to(dtype), y)
    wx, ww = grouped_gemm_bwd(dy, x, w, offsets.long(), dx=torch.empty(rows, k, device=device), dw=torch.empty(len(counts), n, k, device=device))
    assert torch.equal(wx.to(dtype), dx) and torch.equal(ww.to(dtype), dw)


# Many rows, whose results (or, of the second numbers, gradients) come in large tiles: a last round of whole tiles, halves and quarters, experts of
# one row and none, rows and outputs that end inside a tile, short and odd contractions, and rows that only the kernel for any alignment takes.
MANY = [
    ([4200], 4104, 64), ([5000, 1, 0, 250], 4104, 80), ([3300, 0, 700, 37], 2600, 144), ([5120, 700, 65, 0, 1, 3], 2056, 128),
    ([257] * 20 + [0] * 12 + [100] * 10, 1032, 272), ([4700], 4104, 528), ([2900, 0, 1400], 2600, 208), ([1900, 5], 1501, 131),
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{sum(c[0])}x{len(c[0])}x{c[1]}x{c[2]}")
def test_many_rows(device, case):
    counts, n, k = case
    rows, tail = sum(counts), 300
    offsets = _offsets(counts, device)
    for dtype in (BF16, F16):
        wide = torch.full((rows + tail, k + 8), float("nan"), dtype=dtype, device=device)
        x, w = wide[:, :k], _normal(device, len(counts), n, k, dtype=dtype, seed=2)
        x[:rows] = _normal(device, rows, k, dtype=dtype, seed=1)
        for e, c in enumerate(counts):
            if c == 0:
                w[e] = float("nan")
        want, size = _plain(x[:rows], w, offsets)
        out = torch.full((rows + tail, n + 8), 7.0, dtype=dtype, device=device)
        y = grouped_gemm(x, w, offsets, out=out[:, :n])
        _assert_near(y[:rows], want, size, k)
        assert (out[rows:] == 7).all() and (out[:, n:] == 7).all()
        fresh = grouped_gemm(x, w, offsets)
        assert torch.equal(fresh[:rows], y[:rows]) and (fresh[rows:] == 0).all()
        # the same products as a gradient of rows: outputs and inputs change places
        turned = w.transpose(1, 2).contiguous()
        dx = torch.full((rows + tail, n), 5.0, dtype=dtype, device=device)
        grouped_gemm_bwd(x, fresh, turned, offsets, dx=dx, need_dw=False)
        _assert_near(dx[:rows], want, size, k)
        assert (dx[rows:] == 5).all()
        fresh = grouped_gemm_bwd(x, fresh, turned, offsets, need_dw=False)[0]
        assert torch.equal(fresh[:rows], dx[:rows]) and (fresh[rows:] == 0).all()


@pytest.mark.parametrize("case", MANY + [([30, 0, 90, 1], 200, 4104), ([600] * 4, 264, 1032), ([30] * 20 + [0] * 6 + [61] * 6, 1008, 1016), ([900, 0, 1, 700] + [250] * 12, 1288, 1016), ([0, 0], 40, 48)], ids=lambda c: f"{sum(c[0])}x{len(c[0])}x{c[1]}x{c[2]}")
def test_both_gradients_are_the_ones_of_separate_calls(device, case):
    counts, k, n = case                                            # (the rows' gradient has the many columns)
    rows, tail = sum(counts), 300
    offsets = _offsets(counts, device)
    dy, x, w = (_normal(device, *s, dtype=BF16, seed=60 + i) for i, s in enumerate(((rows + tail, n), (rows + tail, k), (len(counts), n, k))))
    dx, dw = grouped_gemm_bwd(dy, x, w, offsets)
    assert torch.equal(dx, grouped_gemm_bwd(dy, x, w, offsets, need_dw=False)[0]) and torch.equal(dw, grouped_gemm_bwd(dy, x, w, offsets, need_dx=False)[1])
    _assert_near(dx[:rows], *_plain(dy[:rows], w.transpose(1, 2), offsets), n)
    assert (dx[rows:] == 0).all()
    b = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(b, b[1:])):
        g, v = dy[lo:hi].double().T, x[lo:hi].double()
        _assert_near(dw[e], g @ v, g.abs() @ v.abs(), hi - lo)
    held = torch.full((rows + tail, k), 5.0, dtype=BF16, device=device), torch.full((len(counts), n, k), 5.0, device=device)
    grouped_gemm_bwd(dy, x, w, offsets, dx=held[0], dw=held[1])
    assert torch.equal(held[0][:rows], dx[:rows]) and (held[0][rows:] == 5).all() and torch.equal(held[1].to(BF16), dw)


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{sum(c[0])}x{len(c[0])}x{c[1]}x{c[2]}")
def test_many_fp8_rows(device, case):
    counts, n, k = case
    rows, tail, e = sum(counts), 300, len(counts)
    offsets = _offsets(counts, device)
    wide = torch.full((rows + tail, k + 16 - k % 16), 0x7F, dtype=torch.uint8, device=device)
    x, xs = wide[:, :k], torch.full((rows + tail, (k + 127) // 128), float("nan"), device=device)
    x[:rows], xs[:rows] = _e4m3(device, rows, k, seed=4), _normal(device, rows, (k + 127) // 128, seed=6).exp() * 1e-2
    w, ws = _e4m3(device, e, n, k, seed=5), _normal(device, e, (n + 127) // 128, (k + 127) // 128, seed=7).exp() * 1e-2
    for i, c in enumerate(counts):
        if c == 0:
            w[i], ws[i] = 0x7F, float("nan")
    for scales in (xs, xs[:, 0].contiguous()):
        want, size = _plain_fp8(x[:rows], scales[:rows], w, ws, offsets)
        for dtype in (BF16, F32):
            out = torch.full((rows + tail, n), 7.0, dtype=dtype, device=device)
            grouped_fp8_gemm(x, scales, w, ws, offsets, out=out)
            _assert_near(out[:rows], want, size, k + 4 + (DROPPED if dtype == BF16 else 0))
            assert (out[rows:] == 7).all()
        fresh = grouped_fp8_gemm(x, scales, w, ws, offsets)
        assert (fresh[rows:] == 0).all()
        _assert_near(fresh[:rows], want, size, k + 4 + DROPPED)


def _e4m3(device, *shape, seed):
    return (_normal(device, *shape, seed=seed) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_fp8(x, xs, w, ws, offsets):
    k, n = x.shape[1], w.shape[1]
    xv, wv = x.view(torch.float8_e4m3fn).double(), w.view(torch.float8_e4m3fn).double()
    xv = xv * (xs.double().repeat_interleave(128, 1)[:, :k] if xs.ndim == 2 else xs.double()[:, None])
    wv = wv * ws.double().repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]
    return _plain(xv, wv, offsets)


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{sum(c[0])}x{len(c[0])}x{c[1]}x{c[2]}")
@pytest.mark.parametrize("block", [0, 128])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_fp8_rows(device, case, block, out_dtype):
    counts, n, k = case
    offsets, rows, e = _offsets(counts, device), sum(counts), len(counts)
    x, w = _e4m3(device, rows, k, seed=4), _e4m3(device, e, n, k, seed=5)
    xs = _normal(device, rows, (k + 127) // 128, seed=6).exp() * 1e-2
    if not block:
        xs = xs[:, 0].contiguous()
    ws = _normal(device, e, (n + 127) // 128, (k + 127) // 128, seed=7).exp() * 1e-2
    out = torch.empty(rows, n, dtype=out_dtype, device=device)
    assert grouped_fp8_gemm(x, xs, w, ws, offsets, out=out) is out
    _assert_near(out, *_plain_fp8(x, xs, w, ws, offsets), k + 4 + (DROPPED if out_dtype == BF16 else 0))
    if out_dtype == BF16:
        assert torch.equal(grouped_fp8_gemm(x, xs, w, ws, offsets.long()), out)


@pytest.mark.parametrize("n, k", [(96, 160), (77, 51), (300, 640)])
@pytest.mark.parametrize("counts", [[3, 0, 2], [40, 0, 90, 200]])
def test_products_of_whole_numbers_are_exact(device, n, k, counts):
    offsets, rows = _offsets(counts, device), sum(counts)
    g = torch.Generator(device=device).manual_seed(8)
    x, w, dy = (torch.randint(-4, 5, s, generator=g, device=device).to(BF16) for s in ((rows, k), (len(counts), n, k), (rows, n)))
    y = torch.empty(rows, n, device=device)
    assert torch.equal(grouped_gemm(x, w, offsets, out=y).double(), _plain(x, w, offsets)[0])
    dx, dw = grouped_gemm_bwd(dy, x, w, offsets, dx=torch.empty(rows, k, device=device), dw=torch.empty(w.shape, device=device))
    assert torch.equal(dx.double(), _plain(dy, w.transpose(1, 2), offsets)[0])
    b = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(b, b[1:])):
        assert torch.equal(dw[e].double(), dy[lo:hi].double().T @ x[lo:hi].double())
    codes = [t.float().to(torch.float8_e4m3fn).view(torch.uint8) for t in (x, w)]
    ones = torch.ones(rows, device=device), torch.ones(len(counts), (n + 127) // 128, (k + 127) // 128, device=device)
    assert torch.equal(grouped_fp8_gemm(codes[0], ones[0], codes[1], ones[1], offsets, out=torch.empty(rows, n, device=device)).double(), _plain(x, w, offsets)[0])


@pytest.mark.parametrize("n, k", [(64, 64), (101, 67), (520, 384), (260, 2048)])
@pytest.mark.parametrize("counts", [[2, 0, 3], [70, 0, 130], [300, 20]])
def test_neighbours_do_not_leak(device, n, k, counts):
    """NaN and infinities in the rows of one expert, in the weights of experts without rows, in the places beside every row and behind
    the last one reach nothing else; rows behind the last expert and places beside the results stay as they were."""
    rows, tail, e = sum(counts), 37, len(counts)
    offsets = _offsets(counts, device)
    nan = float("nan")
    clean = [_normal(device, rows, k, dtype=BF16, seed=9), _normal(device, e, n, k, dtype=BF16, seed=10), _normal(device, rows, n, dtype=BF16, seed=11)]
    want_y = grouped_gemm(clean[0], clean[1], offsets)
    want_dx, want_dw = grouped_gemm_bwd(clean[2], clean[0], clean[1], offsets)
    for shift in (8, 3):                                           # rows that begin on 16 bytes, and rows that do not
        x, dy = (torch.full((rows + tail, m + shift + 8 - (m + shift) % 8), nan, dtype=BF16, device=device) for m in (k, n))
        xv, dv = x[:, shift:shift + k], dy[:, shift:shift + n]
        xv[:rows], dv[:rows] = clean[0], clean[2]
        w = clean[1].clone()
        for i, c in enumerate(counts):
            if c == 0:
                w[i] = nan
        y = torch.full((rows + tail, n + 11), 7.0, dtype=BF16, device=device)
        out = grouped_gemm(xv, w, offsets, out=y[:, 2:2 + n])
        assert torch.equal(out[:rows], want_y) and (out[rows:] == 7).all() and (y[:, :2] == 7).all() and (y[:, 2 + n:] == 7).all()
        fresh = grouped_gemm(xv, w, offsets)
        assert torch.equal(fresh[:rows], want_y) and (fresh[rows:] == 0).all()
        dx, dw = grouped_gemm_bwd(dv, xv, w, offsets)
        assert torch.equal(dx[:rows], want_dx) and (dx[rows:] == 0).all() and torch.equal(dw, want_dw)
        held = torch.full((rows + tail, k), 5.0, dtype=BF16, device=device)
        grouped_gemm_bwd(dv, xv, w, offsets, dx=held, need_dw=False)
        assert torch.equal(held[:rows], want_dx) and (held[rows:] == 5).all()
        # a non-finite row stays within its expert
        first = counts[0]
        xv[0, 0], dv[0, 0] = float("inf"), nan
        assert torch.equal(grouped_gemm(xv, w, offsets)[first:rows], want_y[first:])
        dx, dw = grouped_gemm_bwd(dv, xv, w, offsets)
        assert torch.equal(dx[1:rows], want_dx[1:]) and torch.equal(dw[1:], want_dw[1:]) and dw[0].isnan().any()


@pytest.mark.parametrize("k", [256, 130, 147])
def test_fp8_neighbours_do_not_leak(device, k):
    counts, n, tail = [3, 0, 140], 200, 9
    offsets, rows = _offsets(counts, device), sum(counts)
    w, ws = _e4m3(device, 3, n, k, seed=12), _normal(device, 3, 2, (k + 127) // 128, seed=13).exp()
    x, xs = _e4m3(device, rows, k, seed=14), _normal(device, rows, (k + 127) // 128, seed=15).exp()
    want = grouped_fp8_gemm(x, xs, w, ws, offsets)
    _assert_near(want, *_plain_fp8(x, xs, w, ws, offsets), k + 4 + DROPPED)
    for shift in (16, 5):
        wide = torch.full((rows + tail, k + shift + 16 - (k + shift) % 16), 0x7F, dtype=torch.uint8, device=device)
        wide[:rows, shift:shift + k] = x
        scales = torch.full((rows + tail, xs.shape[1]), float("nan"), device=device)
        scales[:rows] = xs
        bad = w.clone()
        bad[1], s2 = 0x7F, ws.clone()
        s2[1] = float("nan")
        out = torch.full((rows + tail, n), 7.0, dtype=BF16, device=device)
        grouped_fp8_gemm(wide[:, shift:shift + k], scales, bad, s2, offsets, out=out)
        # (rows that do not begin on 16 bytes go through another kernel: its sums differ in their last bits)
        _assert_near(out[:rows], *_plain_fp8(x, xs, w, ws, offsets), k + 4 + DROPPED)
        assert (shift == 5 or k % 16 != 0 or torch.equal(out[:rows], want)) and (out[rows:] == 7).all()


def test_offsets_that_break_the_contract_stay_inside(device):
    """The kernels bring what they read into [0, T]: values are unspecified, but nothing outside the rows is touched."""
    n, k, rows = 72, 64, 50
    x, w, dy = _normal(device, rows, k, dtype=BF16), _normal(device, 3, n, k, dtype=BF16), _normal(device, rows, n, dtype=BF16)
    for bad in ([0, 500, 1000, 2000], [-7, 20, 10, 50], [40, 10, 60, -1], [0, 50, 0, 50]):
        for dtype in (torch.int32, torch.int64):
            off = torch.tensor(bad, dtype=dtype, device=device)
            y = torch.full((rows + 20, n), 7.0, dtype=BF16, device=device)
            grouped_gemm(x, w, off, out=y[:rows])
            grouped_gemm_bwd(dy, x, w, off)
            assert (y[rows:] == 7).all()
    far = torch.tensor([0, 1 << 40, 1 << 41, 1 << 42], dtype=torch.int64, device=device)
    _assert_near(grouped_gemm(x, w, far), *_plain(x, w, torch.tensor([0, rows, rows, rows])), k)


def test_offsets_beyond_32_bits_of_elements(device):
    """Weights of more than 2^31 elements, and rows that end behind 2^31 elements."""
    n, k, e = 4096, 8192, 70
    w = torch.zeros(e, n, k, dtype=BF16, device=device)
    w[-1] = _normal(device, n, k, dtype=BF16, seed=16)
    x = _normal(device, 5, k, dtype=BF16, seed=17)
    off = _offsets([1] + [0] * (e - 2) + [4], device)
    y = grouped_gemm(x, w, off)
    _assert_near(y[1:], *_plain(x[1:], w[-1:], _offsets([4], device)), k)
    dx, _ = grouped_gemm_bwd(y, x, w, off, need_dw=False)
    _assert_near(dx[1:], *_plain(y[1:], w[-1:].transpose(1, 2), _offsets([4], device)), n)
    dw = grouped_gemm_bwd(y, x, w, off, need_dx=False)[1]
    g, v = y[1:].double().T, x[1:].double()
    _assert_near(dw[-1], g @ v, g.abs() @ v.abs(), 4)
    assert (dw[1:-1] == 0).all()
    del w, dw
    rows = (1 << 31) // 8192 + 300
    x = torch.zeros(rows, 8192, dtype=BF16, device=device)
    x[-40:] = _normal(device, 40, 8192, dtype=BF16, seed=18)
    w = _normal(device, 2, 64, 8192, dtype=BF16, seed=19)
    off = _offsets([rows - 40, 40], device)
    y = grouped_gemm(x, w, off)
    _assert_near(y[-40:], *_plain(x[-40:], w[1:], _offsets([40], device)), 8192)
    assert (y[:100] == 0).all()
    dw = grouped_gemm_bwd(y, x, w, off, need_dx=False)[1]
    g, v = y[-40:].double().T, x[-40:].double()
    _assert_near(dw[1], g @ v, g.abs() @ v.abs(), 40)


def test_gradients_against_differences(device):
    """The loss is linear in each operand: whole-number directions give whole-number differences, exact in float32."""
    counts, n, k = [5, 0, 9], 24, 40
    offsets = _offsets(counts, device)
    g = torch.Generator(device=device).manual_seed(20)
    draw = lambda *s: torch.randint(-2, 3, s, generator=g, device=device).to(BF16)
    x, w, dy = draw(14, k), draw(3, n, k), draw(14, n)
    dx, dw = grouped_gemm_bwd(dy, x, w, offsets, dx=torch.empty(14, k, device=device), dw=torch.empty(3, n, k, device=device))
    loss = lambda a, b: float((grouped_gemm(a, b, offsets, out=torch.empty(14, n, device=device)).double() * dy.double()).sum())
    for _ in range(3):
        d, f = draw(14, k), draw(3, n, k)
        assert loss(x + d, w) - loss(x, w) == float((dx.double() * d.double()).sum())
        assert loss(x, w + f) - loss(x, w) == float((dw.double() * f.double()).sum())


def test_differentiable_form(device):
    counts, n, k = [30, 0, 12], 48, 72
    offsets = _offsets(counts, device)
    x, w = _normal(device, 50, k, dtype=BF16, seed=21).requires_grad_(), _normal(device, 3, n, k, dtype=BF16, seed=22).requires_grad_()
    g = _normal(device, 50, n, dtype=BF16, seed=23)
    y = grouped_gemm_apply(x, w, offsets)
    assert torch.equal(y, grouped_gemm(x.detach(), w.detach(), offsets)) and (y[42:] == 0).all()
    y.backward(g)
    dx, dw = grouped_gemm_bwd(g, x.detach(), w.detach(), offsets)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw) and (x.grad[42:] == 0).all()
    x.grad = None
    grouped_gemm_apply(x, w.detach(), offsets).sum().backward()            # (a broadcast cotangent)
    assert torch.equal(x.grad, grouped_gemm_bwd(torch.ones_like(g), x.detach(), w.detach(), offsets, need_dw=False)[0])


def test_second_derivatives_are_refused(device):
    x, w = _normal(device, 8, 16, dtype=BF16, seed=1).requires_grad_(), _normal(device, 2, 8, 16, dtype=BF16, seed=2).requires_grad_()
    (g,) = torch.autograd.grad(grouped_gemm_apply(x, w, _offsets([3, 5], device)).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_captured_calls_replay_on_new_values_and_offsets(device):
    n, k, rows, e = 136, 192, 150, 5
    x, w, dy = _normal(device, rows, k, dtype=BF16), _normal(device, e, n, k, dtype=BF16), _normal(device, rows, n, dtype=BF16)
    x8, w8, ws = _e4m3(device, rows, k, seed=1), _e4m3(device, e, n, k, seed=2), _normal(device, e, 2, 2).exp()
    xs = _normal(device, rows, 2).exp()
    off = _offsets([150, 0, 0, 0, 0], device)
    call = lambda: (grouped_gemm(x, w, off), *grouped_gemm_bwd(dy, x, w, off), grouped_fp8_gemm(x8, xs, w8, ws, off))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for i, counts in enumerate(([30, 30, 30, 30, 30], [0, 149, 0, 0, 1], [1, 2, 3, 4, 5])):
        off.copy_(_offsets(counts, device))
        x.copy_(_normal(device, rows, k, dtype=BF16, seed=30 + i))
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_streams_of_their_own(device):
    sets = [(_normal(device, 300, 512, dtype=BF16, seed=40 + i), _normal(device, 4, 640, 512, dtype=BF16, seed=50 + i), _offsets([i, 100, 0, 200 - i], device)) for i in range(3)]
    want = [grouped_gemm(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(grouped_gemm(*s))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))


def test_native_launch_path_and_helpers_agree(device, monkeypatch):
    n, k, rows, e = 136, 192, 150, 5
    x, w, dy = _normal(device, rows, k, dtype=F16), _normal(device, e, n, k, dtype=F16), _normal(device, rows, n, dtype=F16)
    x8, w8, ws, xs = _e4m3(device, rows, k, seed=1), _e4m3(device, e, n, k, seed=2), _normal(device, e, 2, 2).exp(), _normal(device, rows, 2).exp()
    off = _offsets([50, 0, 60, 1, 30], device)
    host = ops.host
    assert host.grouped_gemm(x[:, :184], w, off) is None and host.grouped_gemm(x, w.bfloat16(), off) is None and host.grouped_gemm(x, w, off[:5]) is None
    assert host.grouped_gemm_bwd(dy[:9], x, w, off) is None and host.grouped_fp8_gemm(x8, xs[:9], w8, ws, off) is None and host.grouped_fp8_gemm(x8, xs, w8, ws[:1], off) is None
    calls = [lambda: (grouped_gemm(x, w, off),), lambda: grouped_gemm_bwd(dy, x, w, off.long()), lambda: (grouped_fp8_gemm(x8, xs, w8, ws, off),),
             lambda: (grouped_fp8_gemm(x8, xs[:, 0].contiguous(), w8, ws, off),)]
    native = [c() for c in calls]

    class Declines:
        def __getattr__(self, name):
            return getattr(host, name) if "workspace" in name else (lambda *args: None)

    monkeypatch.setattr(ops, "host", Declines())
    for a, b in zip(native, [c() for c in calls]):
        assert len(a) == len(b) and all(s.shape == t.shape and s.dtype == t.dtype and torch.equal(s, t) for s, t in zip(a, b))


def test_refusals(device):
    x, w, off = torch.zeros(8, 32, dtype=BF16, device=device), torch.zeros(2, 16, 32, dtype=BF16, device=device), _offsets([4, 4], device)
    x8, w8, xs, ws = x.to(torch.uint8), w.to(torch.uint8), torch.ones(8, device=device), torch.ones(2, 1, 1, device=device)
    dy = torch.zeros(8, 16, dtype=BF16, device=device)
    bad = [
        (TypeError, lambda: grouped_gemm(x.float(), w.float(), off)), (TypeError, lambda: grouped_gemm(x, w.half(), off)), (ValueError, lambda: grouped_gemm(x[:, :30], w, off)),
        (ValueError, lambda: grouped_gemm(x, w[:, :, :30], off)), (ValueError, lambda: grouped_gemm(x, w.transpose(1, 2), off)), (ValueError, lambda: grouped_gemm(x, w, off[:2])),
        (TypeError, lambda: grouped_gemm(x, w, off.float())), (_lib.NativeCallError, lambda: grouped_gemm(x, w, off.cpu())), (ValueError, lambda: grouped_gemm(x, w, off, out=dy[:4])),
        (TypeError, lambda: grouped_gemm(x, w, off, out=dy.half())), (ValueError, lambda: grouped_gemm(x, w, off, out=dy[:1].expand(8, 16))), (ValueError, lambda: grouped_gemm(x.t(), w, off)),
        (ValueError, lambda: grouped_gemm_bwd(dy[:4], x, w, off)), (TypeError, lambda: grouped_gemm_bwd(dy.half(), x, w, off)), (ValueError, lambda: grouped_gemm_bwd(dy, x, w, off, dw=w[:1])),
        (TypeError, lambda: grouped_fp8_gemm(x, xs, w8, ws, off)), (TypeError, lambda: grouped_fp8_gemm(x8, xs, w, ws, off)), (ValueError, lambda: grouped_fp8_gemm(x8, xs[:4], w8, ws, off)),
        (ValueError, lambda: grouped_fp8_gemm(x8, xs, w8, ws[:1], off)), (TypeError, lambda: grouped_fp8_gemm(x8, xs.double(), w8, ws, off)), (TypeError, lambda: grouped_fp8_gemm(x8, xs, w8, ws, off, out=x8[:, :16])),
        (_lib.NativeCallError, lambda: grouped_gemm(x, torch.zeros(513, 16, 32, dtype=BF16, device=device), torch.zeros(514, dtype=torch.int32, device=device))),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            print("not refused:", i)
    assert grouped_gemm(x[:0], w, off * 0).shape == (0, 16)
    assert (grouped_gemm_bwd(dy[:0], x[:0], w, off * 0)[1] == 0).all()


# ---- the operators as a layer uses them -----------------------------------------------------------
def _routed(device, tokens, experts, topk, seed):
    """Rows sorted by expert: offsets, and of every row its token."""
    ids = _normal(device, tokens, experts, seed=seed).topk(topk, 1).indices.reshape(-1)
    order = ids.argsort(stable=True)
    counts = torch.bincount(ids, minlength=experts)
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]), order // topk


@pytest.mark.parametrize("tokens", [1, 5, 200])
def test_second_half_of_a_layer_in_eight_bits(device, tokens):
    """Attention output + stream -> norm in e4m3 -> experts' up and gate product -> silu and product -> e4m3 rows -> experts' down
    product -> sum per token, each step against 64 bits of its own inputs and the whole against 64 bits throughout."""
    d, inner, e, topk = 1024, 512, 16, 4
    x, r, w = _normal(device, tokens, d, dtype=BF16, seed=60), _normal(device, tokens, d, dtype=BF16, seed=61), torch.ones(d, dtype=BF16, device=device)
    up, down = _e4m3(device, e, 2 * inner, d, seed=62), _e4m3(device, e, d, inner, seed=63)
    us, ds = (_normal(device, e, m // 128, c // 128, seed=64).mul(0.2).exp() * (1 / 60) * c ** -0.5 for m, c in ((2 * inner, d), (d, inner)))
    offsets, token = _routed(device, tokens, e, topk, 65)
    codes, scale, h = rms_norm_fp8(x, w, residual=r, scale_block=128)
    rows, row_scale = codes[token], scale[token]
    mid = grouped_fp8_gemm(rows, row_scale, up, us, offsets)
    _assert_near(mid, *_plain_fp8(rows, row_scale, up, us, offsets), d + 4 + DROPPED)
    act = (torch.nn.functional.silu(mid[:, :inner].float()) * mid[:, inner:].float()).contiguous()
    act8, act_scale = torch.empty(act.shape, dtype=torch.uint8, device=device), torch.empty(act.shape[0], device=device)
    ops.fp8_quantize(act, "per_token", codes=act8, scale=act_scale)
    out = grouped_fp8_gemm(act8, act_scale, down, ds, offsets)
    _assert_near(out, *_plain_fp8(act8, act_scale, down, ds, offsets), inner + 4 + DROPPED)
    # 64 bits throughout: e4m3 rounds the rows twice, by 2^-4 of a value at most and by a third of that in the mean
    v = h.double()
    y = v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt()
    one = torch.ones(1, device=device)
    full = lambda t, s: t.view(torch.float8_e4m3fn).double() * s.double().repeat_interleave(128, 1).repeat_interleave(128, 2)
    m = _plain(y[token], full(up, us), offsets)[0]
    want = _plain(torch.nn.functional.silu(m[:, :inner]) * m[:, inner:], full(down, ds), offsets)[0]
    assert one.isfinite().all() and float((out.double() - want).norm() / want.norm()) < 2 * 2.0 ** -4


def test_training_step_of_a_layers_second_half(device):
    """Gradients of norm and experts together, against 64-bit autograd of the same 16-bit inputs."""
    tokens, d, inner, e, topk = 90, 256, 192, 6, 2
    leaves = [_normal(device, tokens, d, dtype=BF16, seed=70), _normal(device, tokens, d, dtype=BF16, seed=71), (1 + 0.1 * _normal(device, d, seed=72)).to(BF16),
              (_normal(device, e, inner, d, seed=73) * d ** -0.5).to(BF16), (_normal(device, e, d, inner, seed=74) * inner ** -0.5).to(BF16)]
    offsets, token = _routed(device, tokens, e, topk, 75)
    cot = _normal(device, tokens, d, seed=76)

    def step(x, r, w, up, down, norm, product):
        y, h = norm(x, w, r)
        out = product(torch.nn.functional.silu(product(y[token], up)), down)
        return h + torch.zeros_like(h).index_add(0, token, out)

    def norm64(x, w, r):
        h = x + r
        return h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w, h

    def product64(x, w):
        b = offsets.tolist()
        return torch.cat([x[lo:hi] @ w[i].T for i, (lo, hi) in enumerate(zip(b, b[1:]))])

    a = [t.clone().requires_grad_() for t in leaves]
    (step(*a, lambda x, w, r: rms_norm_apply(x, w, r), lambda x, w: grouped_gemm_apply(x, w, offsets)).float() * cot).sum().backward()
    b = [t.double().requires_grad_() for t in leaves]
    (step(*b, norm64, product64) * cot.double()).sum().backward()
    for got, want in zip(a, b):
        # a chain of at most ten roundings to bfloat16 (2^-8 each at most, in the 2-norm as well), some of them twice
        assert float((got.grad.double() - want.grad).norm() / want.grad.norm()) < 20 * 2.0 ** -8
    assert torch.equal(rms_norm(leaves[0], leaves[2], residual=leaves[1])[1], (leaves[0].float() + leaves[1].float()).to(BF16))
    assert rms_norm_bwd(leaves[0], leaves[1], leaves[2])[1].dtype == F32


# ---- float16 results of codes: sums of exact products on every kernel ------------------------------
@pytest.mark.parametrize("counts, n, k", [([3, 0, 2], 96, 256), ([40, 0, 90, 200], 300, 640), ([40, 0, 90, 200], 77, 264), ([5000, 1, 0, 250], 520, 128)])
@pytest.mark.parametrize("block", [0, 128])
def test_float16_and_float32_results_of_codes_keep_small_products_beside_large_ones(device, counts, n, k, block):
    """Of every eight products two of 448^2 cancel and six are 14: 84, a whole number on the way and at the end."""
    offsets, rows = _offsets(counts, device), sum(counts)
    encode = lambda v: torch.tensor(v, device=device).repeat(k // 8).to(torch.float8_e4m3fn).view(torch.uint8)
    x = encode([448.0, 448.0, 4.0, 4.0, 4.0, 4.0, 4.0, 4.0]).expand(rows, k).contiguous()
    w = encode([448.0, -448.0, 3.5, 3.5, 3.5, 3.5, 3.5, 3.5]).expand(len(counts), n, k).contiguous()
    xs = torch.ones((rows, (k + 127) // 128) if block else (rows,), device=device)
    ws = torch.full((len(counts), (n + 127) // 128, (k + 127) // 128), 0.125, device=device)
    for dtype in (F16, F32):
        out = torch.empty(rows, n, dtype=dtype, device=device)
        grouped_fp8_gemm(x, xs, w, ws, offsets, out=out)
        assert (out == k // 8 * 84 / 8).all()


@pytest.mark.parametrize("case", CASES + MANY, ids=lambda c: f"{sum(c[0])}x{len(c[0])}x{c[1]}x{c[2]}")
@pytest.mark.parametrize("block", [0, 128])
def test_float16_results_of_codes(device, case, block):
    counts, n, k = case
    offsets, rows, e = _offsets(counts, device), sum(counts), len(counts)
    x, w = _e4m3(device, rows, k, seed=4), _e4m3(device, e, n, k, seed=5)
    xs = _normal(device, rows, (k + 127) // 128, seed=6).exp() * 1e-2
    if not block:
        xs = xs[:, 0].contiguous()
    ws = _normal(device, e, (n + 127) // 128, (k + 127) // 128, seed=7).exp() * 1e-3
    out = torch.empty(rows, n, dtype=F16, device=device)
    assert grouped_fp8_gemm(x, xs, w, ws, offsets, out=out) is out
    _assert_near(out, *_plain_fp8(x, xs, w, ws, offsets), k + 4)


def test_caller_owned_results_count_as_changed(device):
    """autograd refuses a backward pass whose saved operands were overwritten, as it does after a torch operation."""
    x, w, off = _normal(device, 9, 16, dtype=BF16), _normal(device, 2, 16, 16, dtype=BF16), _offsets([4, 5], device)
    y = grouped_gemm_apply(x, w.requires_grad_(), off)
    grouped_gemm(_normal(device, 9, 16, dtype=BF16, seed=1), w.detach(), off, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    w = w.detach()
    dx, dw, other, out = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w), torch.zeros_like(x)
    before = [t._version for t in (dx, dw, other, out)]
    grouped_gemm_bwd(x, x, w, off, dx=dx, dw=dw), grouped_gemm_bwd(x, x, w, off, dw=other, need_dx=False)
    grouped_fp8_gemm(x.to(torch.uint8), torch.ones(9, device=device), w.to(torch.uint8), torch.ones(2, 1, 1, device=device), off, out=out)
    assert all(t._version > v for t, v in zip((dx, dw, other, out), before))


def test_sizes_beyond_the_kernels_counters_are_refused(device):
    x, off = torch.zeros(1, 1, dtype=BF16, device=device), _offsets([1], device)
    wide = torch.empty((1 << 32) + 64, dtype=BF16, device=device)
    codes, one = wide.view(torch.uint8)[:(1 << 32) + 64], torch.ones(1, device=device)
    for call in (lambda: grouped_gemm(x, wide.view(1, -1, 1), off), lambda: grouped_gemm(wide.view(1, -1), wide.view(1, 1, -1), off),
                 lambda: grouped_gemm_bwd(wide.view(1, -1), x, wide.view(1, -1, 1), off), lambda: grouped_gemm_bwd(x, wide.view(1, -1), wide.view(1, 1, -1), off, need_dx=False),
                 lambda: grouped_fp8_gemm(x.to(torch.uint8), one, codes.view(1, -1, 1), torch.ones(1, ((1 << 32) + 64) // 128 + 1, 1, device=device), off)):
        with pytest.raises(ValueError, match="2\\^30"):
            call()
    n, k = (1 << 30) - 64, 8                                        # (the last size of one row that a launch has tiles for)
    w = wide[:n].view(1, n, 1).expand(1, n, k).contiguous()
    w[0, -200:] = _normal(device, 200, k, dtype=BF16, seed=90)
    x = _normal(device, 1, k, dtype=BF16, seed=91)
    y = grouped_gemm(x, w, off)
    _assert_near(y[:, -200:], *_plain(x, w[:, -200:], off), k)
