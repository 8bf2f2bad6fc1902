"""Projections in 8-bit floating point: values in e4m3 with one scale for 128
of them (of a row of activations 128 columns, of a weight 128 x 128).

    w = Fp8Weight(*fp8_blocks(weight))                 # once; or a checkpoint's e4m3 values and scales
    gu = Fp8Weight.gate_up(fp8_blocks(gate), fp8_blocks(up))
    rows = rms_norm_fp8(x, norm, eps, h=h, x_out=x)    # the residual add, the norm, into e4m3
    y = linear_fp8(rows, w)                            # or linear_fp8(x, w): into e4m3 on the way
    y = linear_fp8(gate_up_fp8(rows, gu), down)

Scales that are made here are powers of two (cev_hip.h says which), so that
they cost no significant bit, and every result is rounded once.  f32 outputs
of linear_fp8, and gate_up_fp8 of few rows, come from f32 sums.  For bfloat16
outputs, and gate_up_fp8 of many rows, the matrix cores cut each product to
2^-13 of the largest of eight: 4.5e-5 of a result on normal data, and about one
e4m3 value of gate_up_fp8 in a thousand is the nearest but one, which ones
depending on how many rows the call has.  f32 sums for any number of rows:

    rows = fp8_rows(swiglu(linear_fp8(x, gate, out_dtype=float32), linear_fp8(x, up, out_dtype=float32)))

The calls record nothing for autograd.  An output has memory of its own: one that
lies over a part of an input is refused.
"""
from __future__ import annotations

from ._abi import CEV_BF16, CEV_F32, CEV_FP8_SCALES_E8M0, CEV_FP8_SCALES_F32, CevError, calls
from .paged import _on


def _call(name: str, stream, *args):
    """The native call, its allocations for work on `stream`."""
    f = getattr(calls(), name)
    if stream is None:
        return f(*args, None)
    with _on(stream):
        return f(*args, stream)


class Fp8Rows:
    """Rows of k columns in e4m3: q (t, k up to a multiple of 128), with zeros
    behind column k, and s (t, q's columns / 128), the scales as
    float8_e8m0fnu."""
    __slots__ = ("q", "s", "k")

    def __init__(self, q, s, k: int):
        self.q, self.s, self.k = q, s, k

    @classmethod
    def empty(cls, t: int, k: int, device):
        """Room for t rows of k columns, to be a call's `out`."""
        import torch
        kb = -(-k // 128)
        return cls(torch.empty((t, kb * 128), dtype=torch.float8_e4m3fn, device=device),
                   torch.empty((t, kb), dtype=torch.float8_e8m0fnu, device=device), k)

    def float(self):
        """The values that the rows stand for (t, k), as f32."""
        return (self.q.float() * self.s.float().repeat_interleave(128, 1))[:, : self.k]


class Fp8Weight:
    """A weight (n, k) for linear_fp8: q (n, k) float8_e4m3fn and its scales
    (ceil(n / 128), ceil(k / 128)), float8_e8m0fnu as fp8_blocks makes them or
    a checkpoint's float32 or bfloat16 ones; gate_up() a gate and an up
    projection for gate_up_fp8.  Laid out once, in the order in which the
    products read it (cev_fp8_weight_pack); q is not needed after that."""
    __slots__ = ("n", "k", "is_gate_up", "scale_kind", "data")

    def __init__(self, q, scales, stream=None, _up=(None, None)):
        import torch
        wide = lambda s: s.float() if s is not None and s.dtype == torch.bfloat16 else s  # noqa: E731
        with _on(stream):  # (the wide scales too)
            self.data = calls().fp8_pack(q, wide(scales), _up[0], wide(_up[1]), stream)
        self.n, self.k = q.shape
        self.is_gate_up = _up[0] is not None
        self.scale_kind = CEV_FP8_SCALES_E8M0 if scales.dtype == torch.float8_e8m0fnu else CEV_FP8_SCALES_F32

    @classmethod
    def gate_up(cls, gate, up, stream=None):
        """gate and up: (q, scales) of the same shape."""
        return cls(*gate, stream=stream, _up=tuple(up))


def _room(call: str, out, k: int):
    """The values and scales of `out`, which a call fills with rows of k columns."""
    if out is None:
        return None, None
    if out.k != k:
        raise CevError(-1, f"{call}: out must be Fp8Rows of {k} columns, not of {out.k}")
    return out.q, out.s


def fp8_rows(x, out=None, stream=None):
    """x (t, k) in e4m3 (cev_fp8_rows), for several projections of the same
    rows.  Returns Fp8Rows."""
    q, s = _room("fp8_rows", out, x.shape[-1])
    return Fp8Rows(*_call("fp8_rows", stream, x, q, s), x.shape[1])


def fp8_blocks(w, stream=None):
    """A weight (n, k) in e4m3 with a scale for 128 x 128 values
    (cev_fp8_blocks): (q, scales) for Fp8Weight."""
    return _call("fp8_blocks", stream, w)


def rms_norm_fp8(x, w, eps: float, h=None, x_out=None, out=None, plus_one: bool = False, stream=None):
    """rms_norm into e4m3 (cev_fp8_rms_norm): with h the residual add first,
    x_out = x + h in x's type (x_out defaults to x, and may be h), then the norm, its only
    rounding the one into e4m3.  Returns Fp8Rows."""
    if h is not None and x_out is None:
        x_out = x
    q, s = _room("rms_norm_fp8", out, x.shape[-1])
    return Fp8Rows(*_call("fp8_rms_norm", stream, x, w, eps, h, x_out, plus_one, q, s), x.shape[1])


def _operand(x):
    return (x.q, x.s, x.k) if isinstance(x, Fp8Rows) else (x, None, 0)


def linear_fp8(x, w: Fp8Weight, out=None, out_dtype=None, stream=None):
    """x . w^T (cev_fp8_product) for x (t, k) rows of float32 or bfloat16, or
    Fp8Rows.  out (t, n) is float32 or bfloat16: by default x's type, bfloat16
    for Fp8Rows.  Its workspace comes from torch's allocator for the call's
    stream, so calls on several streams may overlap."""
    import torch
    if w.is_gate_up:
        raise CevError(-1, "linear_fp8: a gate and up weight goes to gate_up_fp8")
    if out is None and out_dtype is None:
        out_dtype = torch.bfloat16 if isinstance(x, Fp8Rows) else x.dtype
    if out_dtype not in (None, torch.float32, torch.bfloat16):
        raise CevError(-2, f"dtype {out_dtype} not supported (float32, bfloat16)")
    code = CEV_F32 if out_dtype == torch.float32 else CEV_BF16
    return _call("fp8_product", stream, *_operand(x), w.data, w.n, w.k, w.scale_kind, False, out, None, code)


def gate_up_fp8(x, w: Fp8Weight, out=None, stream=None):
    """silu(x . gate^T) * (x . up^T) into e4m3 (cev_fp8_product), the rows of
    the down projection: x as for linear_fp8, w from Fp8Weight.gate_up.
    Returns Fp8Rows."""
    if not w.is_gate_up:
        raise CevError(-1, "gate_up_fp8: the weight is no Fp8Weight.gate_up")
    q, s = _room("gate_up_fp8", out, w.n)
    return Fp8Rows(*_call("fp8_product", stream, *_operand(x), w.data, w.n, w.k, w.scale_kind, True, q, s, CEV_BF16), w.n)
