"""Performance cases of the operators behind the attention call: the norm of the residual stream and the experts' products.

Each case is a dict of plain values; its "kind" names the entry point:

  norm         ``rms_norm``: with or without the residual's addition
  norm_fp8     ``rms_norm_fp8``: the same with e4m3 rows and their scales as the output
  norm_bwd     ``rms_norm_bwd``: gradients of the rows and of the weight
  experts      ``grouped_gemm``: 16-bit rows, sorted by expert, times their expert's weight
  experts_bwd  ``grouped_gemm_bwd``: gradients of the rows and of the weights
  experts_fp8  ``grouped_fp8_gemm``: e4m3 rows and weights with float32 scales per 128 channels

``run`` computes them with torch operations in 32 bits, or, with ``own``, through the framework.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
BLOCK = 128
E4M3_MAX = 448.0


def listed():
    return [
        # the smallest call: the norm in front of a layer's second half, for four sequences' new tokens
        {"name": "norm_decode", "kind": "norm", "dtype": "bf16", "rows": 4, "width": 7168, "residual": True},
        # the same for a whole prefill
        {"name": "norm_prefill", "kind": "norm", "dtype": "bf16", "rows": 8192, "width": 7168, "residual": True},
        # rows for the FP8 products of a decode step of 32 sequences, a scale per 128 channels
        {"name": "norm_fp8_decode", "kind": "norm_fp8", "dtype": "bf16", "rows": 32, "width": 7168, "residual": True, "scale_block": 128},
        # the norm of a low-rank query projection in a ragged prefill chunk, one scale a row
        {"name": "norm_fp8_prefill", "kind": "norm_fp8", "dtype": "f16", "rows": 4099, "width": 1536, "residual": False, "scale_block": 0},
        # a training step's norm, with the gradient of the stream that goes past it
        {"name": "norm_backward", "kind": "norm_bwd", "dtype": "bf16", "rows": 4096, "width": 7168, "residual": True},
        # one token, sent to eight experts
        {"name": "experts_token", "kind": "experts", "dtype": "bf16", "rows": 8, "experts": 64, "active": 8, "n": 4096, "k": 2048},
        # a decode step of 32 sequences in 8 bits: most experts get a few rows
        {"name": "experts_fp8_decode", "kind": "experts_fp8", "rows": 256, "experts": 64, "active": 61, "n": 4096, "k": 7168, "scale_block": 128},
        # a prefill chunk in 16 bits
        {"name": "experts_prefill", "kind": "experts", "dtype": "bf16", "rows": 16384, "experts": 32, "active": 32, "n": 4096, "k": 2048},
        # a prefill chunk in 8 bits: the largest case
        {"name": "experts_fp8_prefill", "kind": "experts_fp8", "rows": 16384, "experts": 32, "active": 32, "n": 4096, "k": 7168, "scale_block": 128},
        # a small model's layer with sizes that fit no tile, and experts without rows
        {"name": "experts_ragged", "kind": "experts", "dtype": "f16", "rows": 1003, "experts": 12, "active": 9, "n": 1001, "k": 520},
        # a training step: both gradients
        {"name": "experts_backward", "kind": "experts_bwd", "dtype": "bf16", "rows": 8192, "experts": 16, "active": 16, "n": 4096, "k": 2048},
        # the same of the small model
        {"name": "experts_backward_ragged", "kind": "experts_bwd", "dtype": "f16", "rows": 777, "experts": 8, "active": 6, "n": 1000, "k": 1544},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_fp8", "norm_bwd", "experts", "experts", "experts_bwd", "experts_fp8", "experts_fp8"])
    if kind.startswith("norm"):
        width = _log(rng, 256, 16384)
        if rng.random() < 0.75:
            width = (width + 127) // 128 * 128
        rows = _log(rng, 1, min(16384, (1 << 26) // width))
        case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "rows": rows, "width": width, "residual": rng.random() < 0.6}
        if kind == "norm_fp8":
            case["scale_block"] = rng.choice([0, 128])
        return case
    n, k = _log(rng, 256, 8192), _log(rng, 256, 8192)
    if rng.random() < 0.75:
        n, k = (n + 127) // 128 * 128, (k + 127) // 128 * 128
    elif rng.random() < 0.75:
        k = (k + 7) // 8 * 8
    experts = _log(rng, 1, min(128, max(1, (1 << 30) // (n * k))))
    rows = _log(rng, 1, min(16384, max(16, int((1.2e11 if kind == "experts_bwd" else 2.4e11) / (n * k)))))
    active = max(1, min(experts, rows, int(round(experts * rng.uniform(0.5, 1.0)))))
    case = {"kind": kind, "rows": rows, "experts": experts, "active": active, "n": n, "k": k}
    if kind == "experts_fp8":
        case["scale_block"] = rng.choice([0, 128])
    else:
        case["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    return case


# --------------------------------------------------------------------------- inputs
def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _routing(case, seed):
    """Rows per expert: the active ones have at least one, and some have several times the rows of others."""
    g = torch.Generator().manual_seed(seed)
    e, a, rows = case["experts"], case["active"], case["rows"]
    ids = torch.randperm(e, generator=g)[:a].sort().values
    share = torch.exp(0.5 * torch.randn(a, generator=g))
    counts = 1 + torch.bincount(torch.multinomial(share, rows - a, replacement=True, generator=g) if rows > a else torch.empty(0, dtype=torch.int64), minlength=a)
    full = torch.zeros(e, dtype=torch.int64)
    full[ids] = counts
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), full.cumsum(0)])
    return offsets, ids, int(counts.max())


def _codes(x, block):
    """e4m3 bytes and float32 scales of the last axis, in blocks or (block 0) rows."""
    n = x.shape[-1]
    if block:
        pad = _blocks(n) * block - n
        amax = torch.nn.functional.pad(x.abs(), (0, pad)).unflatten(-1, (-1, block)).amax(-1)
        scale = (amax * (1.0 / E4M3_MAX)).clamp_min(1e-12)
        per = scale.repeat_interleave(block, -1)[..., :n]
    else:
        scale = (x.abs().amax(-1) * (1.0 / E4M3_MAX)).clamp_min(1e-12)
        per = scale[..., None]
    return (x / per).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s = {"case": dict(case)}
    if kind.startswith("norm"):
        rows, n, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
        # a residual stream: a few channels are many times the others, and rows differ in size
        gain = torch.exp(0.7 * normal(n))
        size = torch.exp(0.5 * normal(rows, 1))
        s["x"] = (normal(rows, n) * gain * size).to(dtype)
        s["weight"] = (1.0 + 0.2 * normal(n)).to(dtype)
        if kind == "norm_bwd":
            s["dy"] = (1e-2 * normal(rows, n)).to(dtype)
            if case["residual"]:
                s["dh"] = (1e-2 * normal(rows, n)).to(dtype)
        elif case["residual"]:
            s["residual"] = (normal(rows, n) * gain).to(dtype)
        return s
    rows, e, n, k = case["rows"], case["experts"], case["n"], case["k"]
    offsets, ids, most = _routing(case, seed)
    s["offsets"], s["ids"], s["most"] = offsets.to(torch.int32).cuda(), ids.cuda(), most
    if kind == "experts_fp8":
        codes, s["x_scale"] = _codes(normal(rows, k), case["scale_block"])
        s["x"] = codes.view(torch.uint8)
        # e4m3 weights with a scale per 128 x 128 block, made an expert at a time
        s["w"] = torch.empty((e, n, k), dtype=torch.uint8, device="cuda")
        for i in range(e):
            s["w"][i] = (normal(n, k) * 100.0).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        s["w_scale"] = torch.exp(0.3 * normal(e, _blocks(n), _blocks(k))) * (1e-2 * k ** -0.5)
        return s
    dtype = DTYPES[case["dtype"]]
    s["x"] = normal(rows, k, dtype=dtype)
    s["w"] = normal(e, n, k, dtype=dtype).mul_(k ** -0.5)
    if kind == "experts_bwd":
        s["dy"] = normal(rows, n, dtype=dtype)
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    return _framework(s) if own else _plain(s)


def _framework(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind.startswith("norm"):
        from cppmega_mlx_amd.nn.rms_norm import rms_norm, rms_norm_bwd, rms_norm_fp8

        if kind == "norm":
            return rms_norm(s["x"], s["weight"], eps=EPS, residual=s.get("residual"))
        if kind == "norm_bwd":
            return rms_norm_bwd(s["dy"], s["x"], s["weight"], eps=EPS, dh=s.get("dh"))
        out = rms_norm_fp8(s["x"], s["weight"], eps=EPS, residual=s.get("residual"), scale_block=case["scale_block"])
        return (out[0].view(torch.float8_e4m3fn),) + tuple(out[1:])
    from cppmega_mlx_amd.nn.grouped_gemm import grouped_fp8_gemm, grouped_gemm, grouped_gemm_bwd

    if kind == "experts":
        return grouped_gemm(s["x"], s["w"], s["offsets"])
    if kind == "experts_bwd":
        return grouped_gemm_bwd(s["dy"], s["x"], s["w"], s["offsets"])
    return grouped_fp8_gemm(s["x"], s["x_scale"], s["w"], s["w_scale"], s["offsets"])


def _places(offsets, rows):
    """Of every row: its expert, and its place among that expert's rows."""
    at = torch.arange(rows, device=offsets.device)
    expert = torch.searchsorted(offsets[1:], at.to(offsets.dtype), right=True)
    return expert, at - offsets[expert]


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind.startswith("norm"):
        h, weight = s["x"], s["weight"].float()
        if s.get("residual") is not None:
            h = (h.float() + s["residual"].float()).to(h.dtype)
        v = h.float()
        rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
        if kind == "norm_bwd":
            gw = s["dy"].float() * weight
            c = (gw * v).mean(-1, keepdim=True)
            dx = rstd * gw - rstd * rstd * rstd * c * v
            if s.get("dh") is not None:
                dx = dx + s["dh"].float()
            return dx.to(h.dtype), (s["dy"].float() * v * rstd).sum(0)
        y = v * rstd * weight
        more = () if s.get("residual") is None else (h,)
        if kind == "norm_fp8":
            return _codes(y, case["scale_block"]) + more
        return (y.to(h.dtype),) + more if more else y.to(h.dtype)
    rows, n, ids = case["rows"], case["n"], s["ids"]
    expert, place = _places(s["offsets"], rows)
    slot = torch.searchsorted(ids, expert)

    def padded(t):
        p = torch.zeros((ids.numel(), s["most"], t.shape[-1]), dtype=torch.float32, device=t.device)
        p[slot, place] = t
        return p

    if kind == "experts_fp8":
        k = case["k"]
        x = s["x"].view(torch.float8_e4m3fn).float()
        x = x * (s["x_scale"].repeat_interleave(BLOCK, 1)[:, :k] if case["scale_block"] else s["x_scale"][:, None])
        w = s["w"][ids].view(torch.float8_e4m3fn).float()
        w = w * s["w_scale"][ids].repeat_interleave(BLOCK, 1)[:, :n].repeat_interleave(BLOCK, 2)[:, :, :k]
        return torch.bmm(padded(x), w.transpose(1, 2))[slot, place].to(torch.bfloat16)
    w = s["w"][ids].float()
    x = padded(s["x"].float())
    if kind == "experts":
        return torch.bmm(x, w.transpose(1, 2))[slot, place].to(s["x"].dtype)
    dy = padded(s["dy"].float())
    dx = torch.bmm(dy, w)[slot, place].to(s["x"].dtype)
    dw = torch.zeros_like(s["w"])
    dw[ids] = torch.bmm(dy.transpose(1, 2), x).to(dw.dtype)
    return dx, dw


# --------------------------------------------------------------------------- work and the definition in 64 bits
def work(case):
    kind = case["kind"]
    if kind.startswith("norm"):
        rows, n, size = case["rows"], case["width"], SIZE[case["dtype"]]
        if kind == "norm_bwd":
            return {"bytes": rows * n * size * (4 if case["residual"] else 3) + n * (size + 4), "flops": 10 * rows * n}
        out = size * rows * n
        if kind == "norm_fp8":
            out = rows * n + 4 * rows * (_blocks(n) if case["scale_block"] else 1)
        return {"bytes": rows * n * size * (3 if case["residual"] else 1) + out + n * size, "flops": 5 * rows * n}
    rows, e, a, n, k = case["rows"], case["experts"], case["active"], case["n"], case["k"]
    if kind == "experts_fp8":
        scales = 4 * (rows * (_blocks(k) if case["scale_block"] else 1) + a * _blocks(n) * _blocks(k))
        return {"bytes": rows * k + a * n * k + 2 * rows * n + scales + 4 * (e + 1), "flops": 2 * rows * n * k}
    if kind == "experts":
        return {"bytes": 2 * (rows * k + a * n * k + rows * n) + 4 * (e + 1), "flops": 2 * rows * n * k}
    return {"bytes": 2 * (rows * n + 2 * rows * k + a * n * k + e * n * k) + 4 * (e + 1), "flops": 4 * rows * n * k}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind.startswith("norm"):
        h, weight = s["x"], s["weight"].double()
        if kind != "norm_bwd" and case["residual"]:
            h = (h.double() + s["residual"].double()).to(h.dtype)
        v = h.double()
        ms = torch.linalg.vector_norm(v, dim=1, keepdim=True) ** 2 / case["width"] + EPS
        unit = v / ms.sqrt()
        if kind == "norm_bwd":
            g = s["dy"].double()
            dx = (g * weight - unit * (g * weight * unit).mean(1, keepdim=True)) / ms.sqrt()
            return dx + s["dh"].double() if case["residual"] else dx, (g * unit).sum(0)
        y = unit * weight
        more = (h.double(),) if case["residual"] else ()
        if kind == "norm_fp8":
            n, block = case["width"], case["scale_block"] or case["width"]
            scale = torch.stack([(y[:, i:i + block].abs().amax(1) / E4M3_MAX).clamp_min(1e-12) for i in range(0, n, block)], 1)
            values = [(y[:, b * block:(b + 1) * block] / scale[:, b:b + 1]).float().clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).double() for b in range(scale.shape[1])]
            return (torch.cat(values, 1), scale if case["scale_block"] else scale[:, 0]) + more
        return (y,) + more if more else y
    rows, n, k = case["rows"], case["n"], case["k"]
    bounds = s["offsets"].tolist()
    out = torch.zeros((rows, n if kind != "experts_bwd" else k), dtype=torch.float64, device="cuda")
    dw = torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda") if kind == "experts_bwd" else None
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo == hi:
            continue
        if kind == "experts_fp8":
            for b in range(_blocks(k)):
                c = slice(b * BLOCK, (b + 1) * BLOCK)
                part = s["x"][lo:hi, c].view(torch.float8_e4m3fn).double() @ s["w"][e][:, c].view(torch.float8_e4m3fn).double().T
                sx = s["x_scale"][lo:hi, b] if case["scale_block"] else s["x_scale"][lo:hi]
                sw = s["w_scale"][e, :, b].double().repeat_interleave(BLOCK)[:n]
                out[lo:hi] += part * sx.double()[:, None] * sw
        elif kind == "experts":
            out[lo:hi] = s["x"][lo:hi].double() @ s["w"][e].double().T
        else:
            out[lo:hi] = s["dy"][lo:hi].double() @ s["w"][e].double()
            dw[e] = s["dy"][lo:hi].double().T @ s["x"][lo:hi].double()
    return out if dw is None else (out, dw)
