"""Performance cases of the feed-forward layer: the gated block in 16 and 8 bits, and products with 4-bit weights.

Each case is a dict of plain values; its "kind" names the entry point:

  gated      ``gated_gemm``: act(x w_gate^T) * (x w_up^T) of 16-bit rows, sorted by expert or of one matrix
  gated_fp8  ``fp8_gated_gemm``: the same of e4m3 rows and weights with float32 scales per 128 channels
  step       ``gated_gemm`` that keeps its two products, then ``gated_gemm_bwd``: the block in a training step
  w4         ``w4_gemm``: 16-bit rows times weights of 4 bits with a scale (and a bias) per group of channels
  w4_gated   ``w4_gated_gemm``: the gated block over such weights

A case with "experts" 0 is one matrix that all rows take.  ``run`` computes them with torch operations in 32 bits, or, with ``own``,
through the framework.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 128
E4M3_MAX = 448.0


def listed():
    return [
        # one token, sent to eight experts
        {"name": "gated_token", "kind": "gated", "dtype": "bf16", "activation": "silu", "rows": 8, "experts": 64, "active": 8, "n": 2048, "k": 2048},
        # a decode step of 32 sequences in 8 bits: most experts get a few rows
        {"name": "gated_fp8_decode", "kind": "gated_fp8", "activation": "silu", "rows": 256, "experts": 64, "active": 61, "n": 2048, "k": 7168, "scale_block": 128},
        # a prefill chunk in 16 bits
        {"name": "gated_prefill", "kind": "gated", "dtype": "bf16", "activation": "silu", "rows": 16384, "experts": 32, "active": 32, "n": 2048, "k": 2048},
        # a prefill chunk in 8 bits: the largest case
        {"name": "gated_fp8_prefill", "kind": "gated_fp8", "activation": "silu", "rows": 16384, "experts": 32, "active": 32, "n": 2048, "k": 7168, "scale_block": 128},
        # a small model's dense layer, ragged in every size
        {"name": "gated_dense_ragged", "kind": "gated", "dtype": "f16", "activation": "gelu_tanh", "rows": 1003, "experts": 0, "n": 1001, "k": 520},
        # a training step of the experts
        {"name": "step_experts", "kind": "step", "dtype": "bf16", "activation": "silu", "rows": 8192, "experts": 16, "active": 16, "n": 2048, "k": 2048},
        # a training step of the small model's dense layer
        {"name": "step_dense_ragged", "kind": "step", "dtype": "f16", "activation": "gelu_tanh", "rows": 777, "experts": 0, "n": 500, "k": 1544},
        # the smallest call: one sequence's new token through a low-rank projection
        {"name": "w4_token", "kind": "w4", "dtype": "bf16", "rows": 1, "experts": 0, "n": 2048, "k": 7168, "group": 64, "bias": True},
        # a decode step of 16 sequences through a wide projection, no biases
        {"name": "w4_decode", "kind": "w4", "dtype": "f16", "rows": 16, "experts": 0, "n": 16384, "k": 7168, "group": 128, "bias": False},
        # a few tokens of the small model, the smallest groups
        {"name": "w4_ragged", "kind": "w4", "dtype": "f16", "rows": 5, "experts": 0, "n": 1001, "k": 1056, "group": 32, "bias": True},
        # a step of 64 sequences, or of fewer with several guessed tokens each
        {"name": "w4_rows", "kind": "w4", "dtype": "bf16", "rows": 64, "experts": 0, "n": 8192, "k": 8192, "group": 128, "bias": True},
        # a decode step of 32 sequences over 4-bit experts
        {"name": "w4_experts", "kind": "w4_gated", "dtype": "bf16", "activation": "silu", "rows": 256, "experts": 64, "active": 61, "n": 2048, "k": 7168, "group": 64, "bias": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["gated", "gated", "gated_fp8", "gated_fp8", "step", "w4", "w4", "w4", "w4_gated"])
    four = kind.startswith("w4")
    halves = 1 if kind == "w4" else 2
    n, k = _log(rng, 128, 4096 if halves == 2 else 16384), _log(rng, 256, 8192)
    if rng.random() < 0.75:
        n, k = (n + 127) // 128 * 128, (k + 127) // 128 * 128
    elif rng.random() < 0.75:
        k = (k + 7) // 8 * 8
    case = {"kind": kind, "experts": 0 if rng.random() < (0.7 if kind == "w4" else 0.3) else _log(rng, 1, min(128, max(1, (1 << 30) // (halves * n * k)))), "n": n, "k": k}
    if four:
        case["group"] = rng.choice([32, 64, 128])
        case["k"] = k = (k + case["group"] - 1) // case["group"] * case["group"]
        case["bias"] = rng.random() < 0.6
        case["rows"] = _log(rng, 1, 256 if case["experts"] else 64)
    else:
        case["rows"] = _log(rng, 1, min(16384, max(16, int((0.7e11 if kind == "step" else 2.2e11) / (halves * n * k)))))
    if case["experts"]:
        case["active"] = max(1, min(case["experts"], case["rows"], int(round(case["experts"] * rng.uniform(0.5, 1.0)))))
    if kind == "gated_fp8":
        case["scale_block"] = rng.choice([0, 128])
    else:
        case["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    if halves == 2:
        case["activation"] = rng.choice(["silu", "silu", "gelu_tanh"])
    return case


# --------------------------------------------------------------------------- inputs
def _blocks(n, block=BLOCK):
    return (n + block - 1) // block


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
    """e4m3 codes and float32 scales of the last axis, in blocks or (block 0) rows."""
    n = x.shape[-1]
    if block:
        amax = torch.nn.functional.pad(x.abs(), (0, _blocks(n) * block - n)).unflatten(-1, (-1, block)).amax(-1)
        scale = (amax * (1.0 / E4M3_MAX)).clamp_min(1e-12)
        per = scale.repeat_interleave(block, -1)[..., :n]
    else:
        scale = (x.abs().amax(-1) * (1.0 / E4M3_MAX)).clamp_min(1e-12)
        per = scale[..., None]
    return (x / per).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _four_bits(w, group, bias, dtype):
    """Codes of 4 bits, two to a byte (the even channel low), scales and biases of every group of channels."""
    g = w.unflatten(-1, (-1, group))
    if bias:
        lo = g.amin(-1).to(dtype)
        scale = ((g.amax(-1) - lo.float()) / 15.0).clamp_min(1e-6).to(dtype)
        q = (g - lo.float()[..., None]) / scale.float()[..., None]
    else:
        lo = None
        scale = (g.abs().amax(-1) / 7.0).clamp_min(1e-6).to(dtype)
        q = g / scale.float()[..., None] + 8.0
    q = q.round().clamp(0.0, 15.0).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale, lo


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, e, n, k = case["kind"], case["rows"], case["experts"], case["n"], case["k"]
    out = n if kind == "w4" else 2 * n                             # rows of a weight: the gate's, then the up projection's

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s = {"case": dict(case), "offsets": None}
    if e:
        offsets, ids, most = _routing(case, seed)
        s["offsets"], s["ids"], s["most"] = offsets.to(torch.int32).cuda(), ids.cuda(), most
    lead = (e,) if e else ()
    if kind == "gated_fp8":
        codes, s["x_scale"] = _codes(normal(rows, k), case["scale_block"])
        s["x"] = codes.view(torch.uint8)
        # e4m3 weights with a scale per 128 x 128 block of either half, made an expert at a time
        s["w"] = torch.empty((*lead, out, k), dtype=torch.uint8, device="cuda")
        for w in s["w"] if e else [s["w"]]:
            w.copy_((normal(out, k) * 100.0).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8))
        s["w_scale"] = torch.exp(0.3 * normal(*lead, 2, _blocks(n), _blocks(k))) * (1e-2 * k ** -0.5)
        return s
    dtype = DTYPES[case["dtype"]]
    s["x"] = normal(rows, k, dtype=dtype)
    if kind.startswith("w4"):
        parts = [_four_bits(normal(out, k) * k ** -0.5, case["group"], case["bias"], dtype) for _ in range(e or 1)]
        s["w"], s["scale"] = (torch.stack([p[i] for p in parts]) if e else parts[0][i] for i in (0, 1))
        s["bias"] = None if not case["bias"] else torch.stack([p[2] for p in parts]) if e else parts[0][2]
        return s
    s["w"] = normal(*lead, out, k, dtype=dtype).mul_(k ** -0.5)
    if kind == "step":
        s["dy"] = normal(rows, n, dtype=dtype)
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    return _framework(s) if own else _plain(s)


def _framework(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "w4":
        from cppmega_mlx_amd.nn.w4_gemm import w4_gemm

        return w4_gemm(s["x"], s["w"], s["scale"], s["bias"], s["offsets"])
    if kind == "w4_gated":
        from cppmega_mlx_amd.nn.w4_gemm import w4_gated_gemm

        return w4_gated_gemm(s["x"], s["w"], s["scale"], s["bias"], s["offsets"], activation=case["activation"])
    from cppmega_mlx_amd.nn.gated_ffn import fp8_gated_gemm, gated_gemm, gated_gemm_bwd

    if kind == "gated":
        return gated_gemm(s["x"], s["w"], s["offsets"], activation=case["activation"])
    if kind == "gated_fp8":
        return fp8_gated_gemm(s["x"], s["x_scale"], s["w"], s["w_scale"], s["offsets"], activation=case["activation"])
    pre = torch.empty((case["rows"], 2 * case["n"]), dtype=torch.float32, device=s["x"].device)
    y = gated_gemm(s["x"], s["w"], s["offsets"], activation=case["activation"], pre=pre)
    return (y,) + tuple(gated_gemm_bwd(s["dy"], pre, s["x"], s["w"], s["offsets"], activation=case["activation"]))


def _gate(g, name):
    """The activation of the gate and its derivative."""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def _wide(s, ids):
    """The weights (of the experts `ids`) in float32."""
    case, w = s["case"], s["w"]

    def of(t):
        return t if ids is None else t[ids]

    if case["kind"] == "gated_fp8":
        n, k = case["n"], case["k"]
        scale = of(s["w_scale"]).repeat_interleave(BLOCK, -2)[..., :n, :].flatten(-3, -2).repeat_interleave(BLOCK, -1)[..., :k]
        return of(w).view(torch.float8_e4m3fn).float() * scale
    if case["kind"].startswith("w4"):
        b = of(w)
        q = torch.stack([b & 15, b >> 4], -1).flatten(-2).float().unflatten(-1, (-1, case["group"]))
        scale = of(s["scale"]).float()[..., None]
        return (q * scale + of(s["bias"]).float()[..., None] if s["bias"] is not None else (q - 8.0) * scale).flatten(-2)
    return of(w).float()


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    rows, n, k, e = case["rows"], case["n"], case["k"], case["experts"]
    dtype = torch.bfloat16 if kind == "gated_fp8" else s["x"].dtype
    if kind == "gated_fp8":
        x = s["x"].view(torch.float8_e4m3fn).float()
        x = x * (s["x_scale"].repeat_interleave(BLOCK, 1)[:, :k] if case["scale_block"] else s["x_scale"][:, None])
    else:
        x = s["x"].float()
    if e:
        # the experts that have rows, each with room for the most rows that one has
        at = torch.arange(rows, device=x.device)
        expert = torch.searchsorted(s["offsets"][1:], at.to(s["offsets"].dtype), right=True)
        place, slot = at - s["offsets"][expert], torch.searchsorted(s["ids"], expert)

        def spread(t):
            p = torch.zeros((s["ids"].numel(), s["most"], t.shape[-1]), dtype=torch.float32, device=t.device)
            p[slot, place] = t
            return p

        def gather(t):
            return t[slot, place].to(dtype)

        w, product, x = _wide(s, s["ids"]), torch.bmm, spread(x)
    else:
        spread, gather = torch.Tensor.float, lambda t: t.to(dtype)
        w, product = _wide(s, None), torch.matmul
    both = product(x, w.transpose(-2, -1))
    if kind == "w4":
        return gather(both)
    g, u = both[..., :n], both[..., n:]
    act, slope = _gate(g, case["activation"])
    y = gather(act * u)
    if kind != "step":
        return y
    dy = spread(s["dy"].float())
    grad = torch.cat([dy * u * slope, dy * act], -1)
    dw = product(grad.transpose(-2, -1), x).to(dtype)
    if e:
        full = torch.zeros_like(s["w"])
        full[s["ids"]] = dw
        dw = full
    return y, gather(product(grad, w)), dw


# --------------------------------------------------------------------------- work and the definition in 64 bits
def work(case):
    kind, rows, e, n, k = case["kind"], case["rows"], case["experts"], case["n"], case["k"]
    a = case["active"] if e else 1
    out = n if kind == "w4" else 2 * n
    offsets = 4 * (e + 1) if e else 0
    if kind == "gated_fp8":
        scales = 4 * (rows * (_blocks(k) if case["scale_block"] else 1) + a * 2 * _blocks(n) * _blocks(k))
        return {"bytes": rows * k + a * out * k + 2 * rows * n + scales + offsets, "flops": 2 * rows * out * k}
    if kind.startswith("w4"):
        weights = a * out * (k // 2 + (4 if case["bias"] else 2) * (k // case["group"]))
        return {"bytes": 2 * rows * (k + n) + weights + offsets, "flops": 2 * rows * out * k}
    if kind == "gated":
        return {"bytes": 2 * (rows * (k + n) + a * out * k) + offsets, "flops": 2 * rows * out * k}
    return {"bytes": 2 * (2 * rows * (k + n) + (a + (e or 1)) * out * k) + offsets, "flops": 6 * rows * out * k}


def exact(case, seed):
    s = prepare(case, seed)
    kind, rows, e, n, k = case["kind"], case["rows"], case["experts"], case["n"], case["k"]

    def weight(i):
        def of(t):
            return t[i] if e else t

        w = of(s["w"])
        if kind == "gated_fp8":
            w, scale = w.view(torch.float8_e4m3fn).double(), of(s["w_scale"]).double()
            for h in range(2):
                for j in range(_blocks(n)):
                    r = slice(h * n + j * BLOCK, h * n + min(n, (j + 1) * BLOCK))
                    w[r] *= scale[h, j].repeat_interleave(BLOCK)[:k]
            return w
        if kind.startswith("w4"):
            wide = torch.empty((w.shape[0], k), dtype=torch.float64, device="cuda")
            wide[:, 0::2], wide[:, 1::2] = (w % 16).double(), (w // 16).double()
            scale = of(s["scale"]).double().repeat_interleave(case["group"], 1)
            return wide * scale + (of(s["bias"]).double().repeat_interleave(case["group"], 1) if s["bias"] is not None else -8.0 * scale)
        return w.double()

    x = s["x"]
    if kind == "gated_fp8":
        x = x.view(torch.float8_e4m3fn).double()
        for b in range(_blocks(k)):
            x[:, b * BLOCK:(b + 1) * BLOCK] *= (s["x_scale"][:, b] if case["scale_block"] else s["x_scale"]).double()[:, None]
    x = x.double()
    bounds = s["offsets"].tolist() if e else [0, rows]
    y = torch.zeros((rows, n), dtype=torch.float64, device="cuda")
    if kind == "step":
        dx, dw = torch.zeros((rows, k), dtype=torch.float64, device="cuda"), torch.zeros((max(e, 1), 2 * n, k), dtype=torch.float64, device="cuda")
    for i, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo == hi:
            continue
        w = weight(i)
        p = x[lo:hi] @ w.T
        if kind == "w4":
            y[lo:hi] = p
            continue
        g, u = p[:, :n], p[:, n:]
        if case["activation"] == "silu":
            share = torch.sigmoid(g)
            slope = share + g * share * torch.sigmoid(-g)
        else:
            c = 2.0 * math.sqrt(2.0 / math.pi)
            share = torch.sigmoid(c * (g + 0.044715 * g ** 3))
            slope = share + g * share * torch.sigmoid(-c * (g + 0.044715 * g ** 3)) * c * (1.0 + 0.134145 * g ** 2)
        y[lo:hi] = g * share * u
        if kind == "step":
            dy = s["dy"][lo:hi].double()
            grad = torch.cat([dy * u * slope, dy * g * share], 1)
            dx[lo:hi] = grad @ w
            dw[i] = grad.T @ x[lo:hi]
    return y if kind != "step" else (y, dx, dw if e else dw[0])
