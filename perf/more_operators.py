"""A decoder layer's projections in 8-bit floating point, as timed calls.

Values are e4m3 with one scale for 128 of them: of a row of activations
128 columns, of a weight 128 x 128.  Six kinds of case:

  rows     rows of activations into e4m3 (cev_hip.fp8_rows);
  blocks   a weight into e4m3 (cev_hip.fp8_blocks);
  linear   rows times a weight (cev_hip.linear_fp8), from rows of the model's
           type or rows in e4m3;
  norm     the residual add and RMS norm that make a projection's rows
           (cev_hip.rms_norm_fp8);
  gate_up  gate and up projection with SwiGLU, which make the down
           projection's rows (cev_hip.gate_up_fp8);
  mlp      norm, gate_up and the down projection in a row, as a layer runs them.

A scale that is made here is the least power of two 2^e, e >= -127, that
holds the block's largest value within 448, e4m3's largest; weights may bring
scales of their own in f32.  A host program keeps its weights laid out for
the products, so prepare() does that.
"""
import math
import os
import random
import sys

import torch

own = False  # False: run() computes the plain forms; True: the framework's operators

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust-cev_amd")
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LARGEST = 448.0
EPS = 1e-6


def _cev_hip():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import cev_hip
    return cev_hip


# ---------------------------------------------------------------------------
# The cases


def _rows(t, k, bf16):
    return dict(kind="rows", t=t, k=k, bf16=bf16)


def _blocks(n, k, bf16):
    return dict(kind="blocks", n=n, k=k, bf16=bf16)


def _linear(t, n, k, bf16, given, own_scales):
    """given: whether the rows come in e4m3 already; own_scales: the weight's are powers of two, otherwise any f32."""
    return dict(kind="linear", t=t, n=n, k=k, bf16=bf16, given=given, own_scales=own_scales)


def _norm(t, k, bf16, add, plus_one):
    return dict(kind="norm", t=t, k=k, bf16=bf16, add=add, plus_one=plus_one)


def _gate_up(t, n, k, given, own_scales, bf16=True):
    return dict(kind="gate_up", t=t, n=n, k=k, bf16=bf16, given=given, own_scales=own_scales)


def _mlp(t, n, k, own_scales):
    return dict(kind="mlp", t=t, n=n, k=k, bf16=True, own_scales=own_scales)


def listed():
    return [
        # one token's attention output before its projection: the smallest call, all latency
        dict(_rows(1, 2048, True), name="rows_one_token"),
        # a prefill's attention output
        dict(_rows(8192, 4096, True), name="rows_prefill"),
        # an f32 model's odd-sized weight as it is loaded
        dict(_blocks(1021, 2056, False), name="blocks_odd_f32"),
        # a wide model's down projection as it is loaded
        dict(_blocks(4096, 12288, True), name="blocks_down"),
        # one token through a small model's fused q, k, v projection: streaming the weight
        dict(_linear(1, 4096, 2048, True, True, True), name="linear_one_token"),
        # a decoding batch's attention output through its projection, with a checkpoint's scales
        dict(_linear(64, 4096, 4096, True, False, False), name="linear_decode"),
        # an f32 model's questions, ragged in every direction
        dict(_linear(333, 1000, 2056, False, False, False), name="linear_odd_f32"),
        # a prefill's down projection: the largest product
        dict(_linear(8192, 4096, 12288, True, True, True), name="linear_prefill"),
        # the norm before a decoding batch's projections, the residual add with it
        dict(_norm(64, 4096, True, True, False), name="norm_decode"),
        # the same of a prefill
        dict(_norm(8192, 4096, True, True, False), name="norm_prefill"),
        # a decoding batch's gate and up projections
        dict(_gate_up(16, 6144, 2048, True, True), name="gate_up_decode"),
        # a chunk of 1021 question tokens through a wide model's MLP, with a checkpoint's scales
        dict(_mlp(1021, 12288, 4096, False), name="mlp_chunk"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "blocks", "linear", "linear", "linear", "norm", "gate_up", "mlp"])
    bf16, own_scales = rng.random() < 0.75, rng.random() < 0.5
    width = lambda lo, hi: rng.choice([8 * _log(rng, lo // 8, hi // 8), 128 * _log(rng, max(1, lo // 128), hi // 128)])  # noqa: E731
    if kind == "rows":
        return _rows(_log(rng, 1, 8192), width(16, 12288), bf16)
    if kind == "blocks":
        return _blocks(_log(rng, 16, 12288), width(16, 8192), bf16)
    if kind == "norm":
        return _norm(_log(rng, 1, 8192), width(64, 8192), bf16, rng.random() < 0.7, rng.random() < 0.3)
    t, k = _log(rng, 1, 8192), width(64, 8192)
    if kind == "linear":
        return _linear(t, rng.choice([_log(rng, 1, 8192), 128 * _log(rng, 1, 64)]), k, bf16, rng.random() < 0.5, own_scales)
    n = rng.choice([_log(rng, 16, 6144), 128 * _log(rng, 1, 48)])
    if kind == "gate_up":
        return _gate_up(t, n, k, rng.random() < 0.5, own_scales, bf16)
    return _mlp(min(t, 4096), n, k, own_scales)


def _wide(k):
    """k up to whole blocks."""
    return -(-k // 128) * 128


def work(case):
    e = 2 if case["bf16"] else 4
    kind, t, n, k = case["kind"], case.get("t", 0), case.get("n", 0), case["k"]
    packed = lambda width: t * (_wide(width) + _wide(width) / 128)  # noqa: E731
    weight = lambda rows, cols: rows * cols + (1 if case.get("own_scales") else 4) * _wide(rows) * _wide(cols) / 16384  # noqa: E731
    if kind == "rows":
        return dict(bytes=t * k * e + packed(k), flops=2.0 * t * k)
    if kind == "blocks":
        return dict(bytes=n * k * (e + 1) + _wide(n) * _wide(k) / 16384, flops=2.0 * n * k)
    if kind == "norm":
        return dict(bytes=t * k * e * (3 if case["add"] else 1) + k * e + packed(k), flops=6.0 * t * k)
    if kind == "linear":
        return dict(bytes=(packed(k) if case["given"] else t * k * e) + weight(n, k) + t * n * e, flops=2.0 * t * n * k)
    if kind == "gate_up":
        return dict(bytes=(packed(k) if case["given"] else t * k * e) + 2 * weight(n, k) + packed(n), flops=4.0 * t * n * k)
    return dict(bytes=t * k * e * 4 + k * e + 2 * weight(n, k) + weight(k, n), flops=6.0 * t * n * k)


# ---------------------------------------------------------------------------
# Inputs


def _dtype(case):
    return torch.bfloat16 if case["bf16"] else torch.float32


def _activations(g, dev, t, k, dtype):
    """Rows whose columns differ in size, a few of them much larger than the others."""
    size = torch.exp(0.5 * torch.randn(k, generator=g, device=dev))
    size = torch.where(torch.rand(k, generator=g, device=dev) < 0.002, 20 * size, size)
    return (torch.randn(t, k, generator=g, device=dev) * size).to(dtype)


def _weight(g, dev, n, k, own_scales):
    """An e4m3 weight (n, k) and its scales."""
    w = 0.02 * torch.randn(n, k, generator=g, device=dev)
    if own_scales:
        return _plain_blocks(w)
    top = _tiles(w).abs().amax((1, 3))
    scale = top / LARGEST
    return (w / _spread(scale, n, k)).to(E4M3), scale


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case)
    kind, t, n, k, dt = case["kind"], case.get("t"), case.get("n"), case["k"], _dtype(case)
    if kind == "blocks":
        s["w"] = (0.02 * torch.randn(n, k, generator=g, device=dev)).to(dt)
        return s
    s["x"] = _activations(g, dev, t, k, dt)
    if kind in ("norm", "mlp"):
        s["gamma"] = ((0.0 if case.get("plus_one") else 1.0) + 0.1 * torch.randn(k, generator=g, device=dev)).to(dt)
        if kind == "mlp" or case["add"]:
            s["h"] = _activations(g, dev, t, k, dt)
            s["x_out"] = torch.zeros_like(s["x"])
    weights = {"linear": ["w"], "gate_up": ["gate", "up"], "mlp": ["gate", "up", "down"]}.get(kind, [])
    for name in weights:
        s[name] = _weight(g, dev, *((k, n) if name == "down" else (n, k)), case["own_scales"])
    if case.get("given"):
        s["rows"] = _plain_rows(s.pop("x").float())
    if own:  # the weights laid out for the products, the rows as the operators hand them on
        cev = _cev_hip()
        for name in set(weights) & {"w", "down"}:
            s[name] = cev.Fp8Weight(*s[name])
        if "gate" in weights:
            s["gate_up"] = cev.Fp8Weight.gate_up(s.pop("gate"), s.pop("up"))
        if "rows" in s:
            s["rows"] = cev.Fp8Rows(*s["rows"], k)
    return s


# ---------------------------------------------------------------------------
# The operators in their plain form


def _exponent(top):
    """The least e >= -127 with top <= 448 * 2^e: 448 is 0.875 * 2^9."""
    m, e = torch.frexp(top)
    return torch.where(top > 0, (e - 9 + (m > 0.875)).clamp(min=-127), -127)


def _power(e):
    """2^e in f32."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[1], 0, rows - x.shape[0]))


def _tiles(w):
    """w (n, k) as (n / 128, 128, k / 128, 128), zeros behind its ends."""
    n, k = _wide(w.shape[0]), _wide(w.shape[1])
    return _padded(w, n, k).view(n // 128, 128, k // 128, 128)


def _spread(scale, n, k):
    """The scale of each value of a weight (n, k)."""
    return scale.float().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _plain_rows(x):
    """f32 rows in e4m3, and their scales."""
    t, k = x.shape
    x = _padded(x, t, _wide(k)).view(t, -1, 128)
    e = _exponent(x.abs().amax(-1))
    return (x * _power(-e)[..., None]).to(E4M3).view(t, -1), _power(e).to(E8M0)


def _plain_blocks(w):
    n, k = w.shape
    tiles = _tiles(w.float())
    e = _exponent(tiles.abs().amax((1, 3)))
    q = (tiles * _power(-e)[:, None, :, None]).to(E4M3)
    return q.view(_wide(n), _wide(k))[:n, :k].contiguous(), _power(e).to(E8M0)


def _values(rows):
    """What rows in e4m3 stand for."""
    q, s = rows
    return (q.float().view(q.shape[0], -1, 128) * s.float()[..., None]).flatten(1)


def _plain_product(rows, weight):
    """f32 rows times an e4m3 weight."""
    q, scale = weight
    w = q.float() * _spread(scale, *q.shape)
    return _values(rows)[:, : q.shape[1]] @ w.t()


def _plain_norm(s):
    case, x = s["case"], s["x"]
    if "h" in s:
        x = (x.float() + s["h"].float()).to(x.dtype)
        s["x_out"].copy_(x)
    x = x.float()
    gamma = s["gamma"].float() + (1.0 if case.get("plus_one") else 0.0)
    return _plain_rows(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma)


def _plain_gate_up(rows, s):
    g, u = _plain_product(rows, s["gate"]), _plain_product(rows, s["up"])
    return _plain_rows(g / (1 + torch.exp(-g)) * u)


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        cev = _cev_hip()
        x = s.get("rows", s.get("x"))
        if kind == "blocks":
            q, scale = cev.fp8_blocks(s["w"])
            return {"q": q, "s": scale}
        if kind == "linear":
            return cev.linear_fp8(x, s["w"], out_dtype=_dtype(case))
        if kind == "rows":
            rows = cev.fp8_rows(x)
        if kind in ("norm", "mlp"):
            rows = cev.rms_norm_fp8(x, s["gamma"], EPS, h=s.get("h"), x_out=s.get("x_out"), plus_one=case.get("plus_one", False))
        if kind == "gate_up":
            rows = cev.gate_up_fp8(x, s["gate_up"])
        if kind == "mlp":
            return {"x_out": s["x_out"], "out": cev.linear_fp8(cev.gate_up_fp8(rows, s["gate_up"]), s["down"], out_dtype=_dtype(case))}
        rows = (rows.q, rows.s)
    else:
        if kind == "blocks":
            q, scale = _plain_blocks(s["w"])
            return {"q": q, "s": scale}
        rows = _plain_norm(s) if kind in ("norm", "mlp") else s["rows"] if "rows" in s else _plain_rows(s["x"].float())
        if kind == "linear":
            return _plain_product(rows, s["w"]).to(_dtype(case))
        if kind in ("gate_up", "mlp"):
            rows = _plain_gate_up(rows, s)
        if kind == "mlp":
            return {"x_out": s["x_out"], "out": _plain_product(rows, s["down"]).to(_dtype(case))}
    out = {"q": rows[0], "s": rows[1]}
    return dict(out, x_out=s["x_out"]) if "x_out" in s else out


# ---------------------------------------------------------------------------
# The operators from their definitions in 64 bits


def _exact_scale(top):
    """The least power of two from 2^-127 on that 448 times is not below top."""
    e = torch.full_like(top, -127.0)
    some = top > 0
    e[some] = torch.ceil(torch.log2(top[some] / LARGEST)).clamp(min=-127)
    e = torch.where(LARGEST * torch.exp2(e) < top, e + 1, e)  # where the logarithm was rounded
    return torch.where((e > -127) & (LARGEST * torch.exp2(e - 1) >= top), e - 1, e).exp2()


def _exact_round(x):
    """To the nearest value of 4 significant bits and at least 2^-9 apart, the even one of two."""
    low = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    low = torch.where(torch.exp2(low) > x.abs().clamp(min=2.0 ** -6), low - 1, low)
    step = torch.exp2(low - 3)
    return torch.round(x / step) * step


def _exact_groups(x):
    """Column groups of a row, one after the other."""
    q, s = torch.zeros(x.shape[0], _wide(x.shape[1]), dtype=torch.float64, device=x.device), []
    for c in range(0, x.shape[1], 128):
        part = x[:, c: c + 128]
        scale = _exact_scale(part.abs().amax(1))
        q[:, c: c + part.shape[1]] = _exact_round(part / scale[:, None])
        s.append(scale)
    return q, torch.stack(s, 1)


def _exact_product(rows, weight):
    """The sum over column groups, each with its scales."""
    (q, s), (w, scale) = rows, weight
    w, y = w.double(), torch.zeros(q.shape[0], w.shape[0], dtype=torch.float64, device=q.device)
    of_row = torch.arange(w.shape[0], device=q.device) // 128
    for b in range(s.shape[1]):
        at = slice(128 * b, min(128 * b + 128, w.shape[1]))
        y += (q[:, at].double() @ w[:, at].t().contiguous()) * s[:, b, None].double() * scale.double()[of_row, b]
    return y


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "blocks":
        w = s["w"].double()
        q, scale = torch.zeros_like(w), []
        for r in range(0, w.shape[0], 128):
            row = []
            for c in range(0, w.shape[1], 128):
                part = w[r: r + 128, c: c + 128]
                row.append(_exact_scale(part.abs().amax()[None])[0])
                q[r: r + 128, c: c + 128] = _exact_round(part / row[-1])
            scale.append(torch.stack(row))
        return {"q": q, "s": torch.stack(scale)}
    out = {}
    if "rows" in s:
        rows = s["rows"]
    elif kind in ("norm", "mlp"):
        x = s["x"].double()
        if "h" in s:
            x = (x + s["h"].double()).to(_dtype(case)).double()
            out["x_out"] = x
        size = torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / case["k"]
        rows = _exact_groups(x / torch.sqrt(size + EPS) * (s["gamma"].double() + (1 if case.get("plus_one") else 0)))
    else:
        rows = _exact_groups(s["x"].double())
    if kind == "linear":
        return _exact_product(rows, s["w"])
    if kind in ("gate_up", "mlp"):
        g = _exact_product(rows, s["gate"])
        rows = _exact_groups(g * torch.sigmoid(g) * _exact_product(rows, s["up"]))
    if kind == "mlp":
        return dict(out, out=_exact_product(rows, s["down"]))
    return dict(out, q=rows[0], s=rows[1])
