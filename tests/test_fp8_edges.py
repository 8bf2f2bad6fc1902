"""Projections in 8-bit floating point at the ends of their range and in calls
that tests/test_fp8.py does not make; its oracle and tolerances."""
import pytest
import torch

import cev_hip
from cev_hip import Fp8Rows, Fp8Weight
from test_fp8 import (E4M3, E8M0, GATE_UPS, activations, check_product, form_of, half_ulp, oracle_norm, oracle_rows, packed, round_e4m3, up128, values,
                      weight_of, weight_values)


# ---------------------------------------------------------------------------
# Scales far apart

SCALES_APART = [(112, -40, 448.0), (118, -100, 448.0), (112, 10, 2.0 ** -9), (-118, 120, 448.0), (-118, 120, 2.0 ** -9), (-120, 100, 2.0 ** -9),
                (100, -126, 448.0), (119, -149, 448.0), (-100, 127, 448.0), (-60, 127, 2.0 ** -9)]


def far_rows(t, k, m, x_exp, gpu):
    """Rows of m * 2^x_exp whose blocks all have the scale 2^x_exp, by their first columns."""
    x = torch.full((t, k), m, dtype=torch.float64) * 2.0 ** x_exp
    x[:, ::128] = 448 * 2.0 ** x_exp
    return x.float().to(gpu)


def far_weight(n, k, m, w_exp, kind, gpu):
    """(q, scales) of m, but for 0 in each block's first column; 1.5 * 2^w_exp (f32) or 2^w_exp."""
    q = torch.full((n, k), m).to(E4M3)
    q[:, ::128] = 0
    scale = (1.5 if kind == "f32" and w_exp > -140 else 1.0) * 2.0 ** w_exp
    return q.to(gpu), torch.full((up128(n) // 128, up128(k) // 128), scale, dtype=torch.float64).to(torch.float32 if kind == "f32" else E8M0).to(gpu), scale


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,k", [(2, 40, 128), (20, 40, 1032), (130, 4096, 520), (3000, 4100, 1032), (900, 4000, 8200)])
@pytest.mark.parametrize("x_exp,w_exp,m", SCALES_APART)
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_scales_whose_effects_cancel(gpu, t, n, k, x_exp, w_exp, m, kind, out_dtype):
    """A row's scale alone takes a sum out of f32's range, the weight's takes the result back into it: on both ends."""
    if kind == "e8m0" and w_exp < -127:
        pytest.skip("no such e8m0 scale")
    q, s, scale = far_weight(n, k, m, w_exp, kind, gpu)
    want = m * m * 2.0 ** x_exp * scale * (k - len(range(0, k, 128)))
    y = cev_hip.linear_fp8(far_rows(t, k, m, x_exp, gpu), Fp8Weight(q, s), out_dtype=out_dtype).double().cpu()
    # equal products of 49 * 2^12 or 2^-18 (1.5 times that): nothing is cut, and sums of fewer than 2^24 / 147 of them are exact
    assert 2.0 ** -126 < want < 2.0 ** 127 and bool(((y - want).abs() <= half_ulp(out_dtype) * want).all()), (want, y.min(), y.max())


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,k", [(2, 40, 128), (20, 136, 1032), (900, 4000, 1032)])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_gate_up_of_scales_whose_effects_cancel(gpu, t, n, k, kind):
    q, s, scale = far_weight(n, k, 448.0, -110, kind, gpu)
    rows = cev_hip.gate_up_fp8(far_rows(t, k, 448.0, 108, gpu), Fp8Weight.gate_up((q, s), (q, s)))
    g = 448.0 ** 2 * 2.0 ** 108 * scale * (k - len(range(0, k, 128)))  # silu(g) is g
    assert bool(((rows.float().double() / (g * g) - 1).abs() <= 2.0 ** -4 + 2.0 ** -20).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,k", [(2, 40, 128), (20, 40, 1032), (900, 4000, 1032)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_scales_of_zero_infinity_and_nan(gpu, t, n, k, out_dtype):
    """A weight's scale of 0 gives 0 also under rows of the largest scale, and one that is not finite stays in its columns."""
    x = far_rows(t, k, 448.0, 119, gpu)
    q, s, _ = far_weight(n, k, 448.0, -100, "f32", gpu)
    want = cev_hip.linear_fp8(x, Fp8Weight(q, s), out_dtype=out_dtype)
    y = cev_hip.linear_fp8(x, Fp8Weight(q, torch.zeros_like(s)), out_dtype=out_dtype)
    assert bool((y == 0).all())
    for bad in (float("inf"), float("-inf"), float("nan")):
        s2 = s.clone()
        s2[-1, 0] = bad
        y = cev_hip.linear_fp8(x, Fp8Weight(q, s2), out_dtype=out_dtype)
        at = up128(n) - 128
        assert torch.equal(y[:, :at], want[:, :at])
        assert bool((y[:, at:] == bad).all() if bad == bad else torch.isnan(y[:, at:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,k", [(2, 40, 128), (20, 40, 1032), (40, 300, 640), (300, 2048, 256), (900, 4000, 1160)])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_scales_of_rows_that_are_nan_or_at_their_ends(gpu, t, n, k, kind, out_dtype):
    """A NaN scale of a row, in its first, last or some block, makes that row NaN and no other; the largest and least ones are used."""
    rows = cev_hip.fp8_rows(activations(t, k, torch.bfloat16, 80).to(gpu))
    w = packed(weight_of(n, k, kind, 81), gpu)
    clean = cev_hip.linear_fp8(rows, w, out_dtype=out_dtype)
    kb = rows.s.shape[1]
    for row, block in ((0, 0), (t - 1, kb - 1), (t // 2, kb // 2)):
        s = rows.s.view(torch.uint8).clone()
        s[row, block] = 255
        y = cev_hip.linear_fp8(Fp8Rows(rows.q, s.view(E8M0), k), w, out_dtype=out_dtype)
        others = torch.arange(t, device=gpu) != row
        assert bool(torch.isnan(y[row]).all()) and torch.equal(y[others], clean[others])
    # scales of 2^127 and 2^-127 in turn, beside weights of 2^-126 (sums up to 2^25) and 2^126
    for code, w_exp in ((254, -126), (0, 126)):
        q = torch.ones_like(rows.q.float()).to(E4M3)
        q[:, k:] = 0
        y = cev_hip.linear_fp8(Fp8Rows(q, torch.full_like(s, code).view(E8M0), k),
                               Fp8Weight(torch.ones(n, k, device=gpu).to(E4M3), torch.full((up128(n) // 128, kb), 2.0 ** w_exp, device=gpu).to(torch.float32 if kind == "f32" else E8M0)),
                               out_dtype=out_dtype)
        assert bool((y.double() == torch.tensor(k * 2.0 ** (code - 127 + w_exp)).to(out_dtype).double().to(gpu)).all())


# ---------------------------------------------------------------------------
# Overlapping memory


def test_overlapping_rows_by_every_byte(cev):
    """cev_overlap against the sets of bytes, for all small strides, lengths and distances."""
    import ctypes as C
    import itertools

    class Rows(C.Structure):
        _fields_ = [("p", C.c_void_p), ("rows", C.c_int64), ("stride", C.c_int64), ("bytes", C.c_int64)]

    f = cev._abi.lib().cev_overlap
    f.restype, f.argtypes = C.c_bool, [C.POINTER(Rows), C.POINTER(Rows)]
    of = lambda p, rows, stride, n: {p + i * stride + j for i in range(rows) for j in range(n)}  # noqa: E731
    shapes = [(r, s, n) for r in (0, 1, 2, 4) for n in (0, 1, 3) for s in (n, n + 1, n + 4) if r > 1 or s == n] + [(3, 7, 2), (1, -5, 2), (1, 0, 4)]
    n = 0
    for a, b in itertools.product(shapes, repeat=2):
        for at in range(-24, 25):
            want = bool(of(100, *a) & of(100 + at, *b))
            assert f(C.byref(Rows(100, *a)), C.byref(Rows(100 + at, *b))) == want, (a, b, at)
            n += want
    assert n > 1000
    big = 1 << 31
    assert not f(C.byref(Rows(1 << 20, big, 256, 128)), C.byref(Rows((1 << 20) + 128, big, 256, 128)))
    assert f(C.byref(Rows(1 << 20, big, 256, 129)), C.byref(Rows((1 << 20) + 128, big, 256, 128)))


def test_shifted_outputs_are_refused(cev):
    """An output that lies over a part of an input or of another output: refused before the GPU is looked at."""
    import ctypes as C
    L = cev._abi.lib()
    at = lambda x: C.c_void_p((1 << 20) + x)  # noqa: E731

    def refused(rc):
        assert rc == -1 and " own" in L.cev_last_error().decode(), (rc, L.cev_last_error())

    far = 1 << 24
    # rows: x (4, 128) f32 with rows 256 elements apart, (4 * 256 - 128) * 4 bytes
    rows = lambda q, s: L.cev_fp8_rows(0, 4, 128, at(0), 256, at(q), at(s), None)  # noqa: E731
    refused(rows(16, far))
    refused(rows(-16, far))
    refused(rows(3 * 1024 + 496, far))
    refused(rows(far, 511))
    refused(rows(512 - 16, far))
    refused(rows(far, far + 511))
    refused(rows(far, far - 3))
    # the norm: x, h (4, 64) bf16, x_out shifted against them, or over w
    norm = lambda xo=0, so=64, h=far, w=2 * far, q=3 * far, s=4 * far: L.cev_fp8_rms_norm(1, 4, 64, at(0), 64, at(h), 64, at(xo), so, at(w), 1e-6, 0, at(q), at(s), None)  # noqa: E731
    refused(norm(xo=128))
    refused(norm(xo=-384))
    refused(norm(xo=0, so=72))
    refused(norm(xo=far + 16))
    refused(norm(xo=2 * far - 16))
    refused(norm(q=16))
    refused(norm(q=far - 256))
    refused(norm(xo=far, s=far + 511))
    refused(norm(q=2 * far + 112))
    refused(norm(s=2 * far + 127))
    refused(norm(q=3 * far, s=3 * far + 511))
    # blocks: w (130, 136) f32
    blocks = lambda q, s: L.cev_fp8_blocks(0, 130, 136, at(0), 136, at(q), at(s), None)  # noqa: E731
    refused(blocks(130 * 136 * 4 - 16, far))
    refused(blocks(far, 130 * 136 * 4 - 1))
    refused(blocks(far, far + 130 * 136 - 1))
    # pack: q (130, 136), f32 scales (2, 2), 256-byte aligned weight of 2 * 8 * 2 pieces
    pack = lambda w, up=None, ups=None: L.cev_fp8_weight_pack(130, 136, 1, at(0), 136, at(far), 2, up, 136 if up else 0, ups, 2 if up else 0, at(w), 1 << 22, None)  # noqa: E731
    refused(pack(17408))
    refused(pack(-256))
    refused(pack(far))
    refused(pack(2 * far, at(2 * far + 512), at(3 * far)))
    refused(pack(2 * far, at(3 * far), at(2 * far + 512)))
    # products: x (40, 128) bf16 with rows 256 apart, a weight of 8 pieces, out (40, 200)
    desc = cev._abi.Fp8Desc
    size = C.c_size_t()

    def product(x=0, xs=None, w=far, out=2 * far, outs=None, work=4 * far, **kw):
        d = desc(**{**dict(x_dtype=1, out_dtype=1, scales=1, gate_up=0, t=40, n=200, k=128, x_stride=256, out_stride=200), **kw})
        assert L.cev_fp8_work_size(C.byref(d), C.byref(size)) == 0
        return L.cev_fp8_product(C.byref(d), at(x), xs, at(w), 1 << 22, at(out), outs, at(work), size.value, None)

    refused(product(out=16))
    refused(product(out=-40 * 400 + 2))
    refused(product(out=far + 8 * 4100 - 2))
    refused(product(work=512))
    refused(product(work=2 * far + 256))
    refused(product(work=far))
    refused(product(x=16, out=0, out_stride=256))
    refused(product(x_dtype=2, xs=at(3 * far), out=40 * 128 - 2))
    refused(product(x_dtype=2, xs=at(3 * far), out=3 * far + 38))
    gate = dict(x_dtype=2, xs=at(3 * far), gate_up=1, out_dtype=2, n=128)
    refused(product(outs=at(2 * far + 39), **gate))
    refused(product(outs=at(40 * 128 - 1), **gate))
    refused(product(out=16, outs=at(5 * far), **gate))
    refused(product(work=5 * far, outs=at(5 * far + 100), **gate))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_outputs_beside_their_inputs_in_one_buffer(gpu, dtype):
    """Columns of one wide buffer as x and out, the sum of a norm in place of x or of h, and x_out beside both."""
    t, k, n = 40, 256, 200
    g = torch.Generator().manual_seed(1)
    room = torch.randn(t, 1024, generator=g).to(dtype).to(gpu)
    x, h, out, xo = room[:, :k], room[:, 256: 512], room[:, 512: 512 + n], room[:, 768:]
    w = Fp8Weight(*cev_hip.fp8_blocks(torch.randn(n, k, generator=g).to(dtype).to(gpu)))
    gamma = torch.ones(k, dtype=dtype, device=gpu)
    want = cev_hip.linear_fp8(x.contiguous(), w)
    assert torch.equal(cev_hip.linear_fp8(x, w, out=out), want) and torch.equal(out, want)
    total = x + h
    rows = cev_hip.rms_norm_fp8(x.contiguous(), gamma, 1e-6, h=h)
    for place in (xo, h, x):  # (h and x last: they are overwritten)
        a, b = x.clone(), h.clone()
        got = cev_hip.rms_norm_fp8(x, gamma, 1e-6, h=h, x_out=place)
        assert torch.equal(place, total) and torch.equal(got.q.view(torch.uint8), rows.q.view(torch.uint8))
        x.copy_(a), h.copy_(b)
    with pytest.raises(cev_hip.CevError, match="of its own"):
        cev_hip.rms_norm_fp8(room[:, 8: 8 + k], gamma, 1e-6, h=h.clone(), x_out=x)
    with pytest.raises(cev_hip.CevError, match="of its own"):
        cev_hip.linear_fp8(x, w, out=room[:, k - 8: k - 8 + n])


# ---------------------------------------------------------------------------
# The norm at the ends of f32's range


def norm_rows(kind, t, k, dtype):
    """(x, weight) whose normalised values, or what they are made from, are not normal f32 numbers."""
    g = torch.Generator().manual_seed(70)
    x, w = torch.randn(t, k, generator=g).double(), 1 + 0.1 * torch.randn(k, generator=g).double()
    if kind == "subnormal x":  # 1 / root is beyond f32
        x *= 2.0 ** -135
    elif kind == "large x":  # 1 / root is a subnormal f32
        x = (x * 2.0 ** 126).clamp(-2.0 ** 127, 2.0 ** 127)
    elif kind == "one large x":  # all others over the root are subnormal, and normal times w
        x *= 2.0 ** -78
        x[:, 5] = 2.0 ** 60
        w *= 2.0 ** 100
        w[5] = 1.0
    elif kind == "small blocks":  # the same of whole blocks, beside ordinary weights
        x *= 2.0 ** 60
        x[:, 128: 256] *= 2.0 ** -130
        x[:, 5: 9] *= 2.0 ** -130
    elif kind == "small w":  # the results are subnormal
        w *= 2.0 ** -129
    elif kind == "smallest w":
        w *= 2.0 ** -136
    elif kind == "zeros":  # whole chunks of 8, beside others that need f64
        x *= 2.0 ** -135
        x[:, : k // 2] = 0
        x[0] *= torch.rand(k, generator=g) < 0.3
    return x.float().to(dtype), w.float().to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["subnormal x", "large x", "one large x", "small blocks", "small w", "smallest w", "zeros"])
@pytest.mark.parametrize("t,k", [(3, 264), (64, 4096), (600, 2056), (2, 20000)])
def test_norm_is_the_nearest_at_the_ends_of_the_range(gpu, t, k, kind, dtype):
    """Every value and scale is that of 64-bit arithmetic, as for ordinary rows."""
    x, w = norm_rows(kind, t, k, dtype)
    got = cev_hip.rms_norm_fp8(x.to(gpu), w.to(gpu), 0.0)
    q, e = oracle_rows(oracle_norm(x, w, 0.0, None, False)[1])
    assert torch.equal(got.s.view(torch.uint8).cpu().double(), e + 127) and torch.equal(got.q.double().cpu(), q)


@pytest.mark.gpu
def test_norm_of_values_beyond_f32(gpu):
    """A normalised value that f32 does not hold is not finite: NaN, and it counts for no scale."""
    x, w = torch.ones(2, 256), torch.full((256,), 2.0)
    x[:, 7] = 64.0
    w[7] = 2.0 ** 127
    got = cev_hip.rms_norm_fp8(x.to(gpu), w.to(gpu), 1e-6)
    want = oracle_norm(x, w, 1e-6, None, False)[1]
    assert float(want[0, 7]) > 2.0 ** 128
    want[:, 7] = float("inf")
    q, e = oracle_rows(want)
    g = got.q.double().cpu()
    assert torch.equal(got.s.view(torch.uint8).cpu().double(), e + 127)
    assert torch.equal(torch.isnan(g), torch.isnan(q)) and torch.equal(torch.nan_to_num(g), torch.nan_to_num(q))


# ---------------------------------------------------------------------------
# Rows that a call fills


def test_out_of_other_columns_is_refused(cev):
    """Rows of 300 and of 310 columns take the same room; an `out` that says 300 is not filled with 310."""
    z = torch.zeros
    out = Fp8Rows(z(2, 384).to(E4M3), z(2, 3).to(E8M0), 300)
    gate_up = type("W", (), dict(is_gate_up=True, data=z(1 << 16, dtype=torch.uint8), n=310, k=128, scale_kind=0))
    for call in (lambda: cev_hip.fp8_rows(z(2, 310), out=out), lambda: cev_hip.rms_norm_fp8(z(2, 310), z(310), 1e-6, out=out),
                 lambda: cev_hip.gate_up_fp8(z(2, 128), gate_up, out=out)):
        with pytest.raises(cev_hip.CevError, match="310 columns, not of 300") as err:
            call()
        assert err.value.code == -1


# ---------------------------------------------------------------------------
# Zero rows, a checkpoint's bfloat16 scales, f32 sums


@pytest.mark.gpu
def test_no_rows_of_bfloat16(gpu):
    w = packed(weight_of(40, 72, "e8m0", 14), gpu)
    x = torch.zeros(0, 72, dtype=torch.bfloat16, device=gpu)
    assert cev_hip.linear_fp8(x, w).shape == (0, 40) and cev_hip.fp8_rows(x).q.shape == (0, 128)
    assert cev_hip.linear_fp8(cev_hip.fp8_rows(x), w).shape == (0, 40)
    assert cev_hip.rms_norm_fp8(x, torch.ones(72, dtype=torch.bfloat16, device=gpu), 1e-6).s.shape == (0, 1)
    gu = Fp8Weight.gate_up(*[tuple(y.to(gpu) for y in weight_of(40, 72, "e8m0", 14)) for _ in range(2)])
    assert cev_hip.gate_up_fp8(x, gu).q.shape == (0, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("t,n,k", [(3, 300, 520), (300, 136, 1032)])
def test_bfloat16_scales(gpu, side, t, n, k):
    """A weight with bfloat16 scales is the one with the same scales in f32; on a side stream its f32 copies are that stream's."""
    x = activations(t, k, torch.bfloat16, 71).to(gpu)
    pairs = [tuple(y.to(gpu) for y in weight_of(n, k, "bf16", 72 + i)) for i in range(2)]
    wide = [(q, s.float()) for q, s in pairs]
    want = cev_hip.linear_fp8(x, Fp8Weight(*wide[0])), cev_hip.gate_up_fp8(x, Fp8Weight.gate_up(*wide))
    s = torch.cuda.Stream() if side else None
    torch.cuda.synchronize()
    for _ in range(5):
        w, gu = Fp8Weight(*pairs[0], stream=s), Fp8Weight.gate_up(*pairs, stream=s)
        got = cev_hip.linear_fp8(x, w, stream=s), cev_hip.gate_up_fp8(x, gu, stream=s)
        if side:
            s.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].q.view(torch.uint8), want[1].q.view(torch.uint8))
        assert torch.equal(got[1].s.view(torch.uint8), want[1].s.view(torch.uint8))
        check_product(got[0], values(*[y.cpu() for y in (lambda r: (r.q, r.s))(cev_hip.fp8_rows(x))])[:, :k], weight_values(*[y.cpu() for y in wide[0]]), torch.bfloat16)


def check_nearest(got, xv, gate, up):
    """Rows of silu(g) u from sums in f32: the nearest e4m3 values of 64-bit ones, but for those next to a border."""
    k, n = xv.shape[1], gate.shape[0]
    g, u = (xv @ w.t() for w in (gate, up))
    size = [xv.abs() @ w.abs().t() for w in (gate, up)]
    want = g * torch.sigmoid(g) * u
    # each sum within c of its magnitudes; silu's slope is at most 1.1; the exponential within 2^-22 (1 + |g|), the rest some f32 roundings
    c = (k + k / 64 + 16) * 2.0 ** -23
    tol = 1.1 * c * size[0] * (u.abs() + c * size[1]) + g.abs() * c * size[1] + want.abs() * (2.0 ** -22 * (1 + g.abs()) + 2.0 ** -21)
    e = got.s.view(torch.uint8).cpu().double() - 127
    v, slack, q = (torch.zeros(xv.shape[0], up128(n), dtype=torch.float64) for _ in range(3))
    v[:, :n], slack[:, :n] = want, tol
    by = torch.exp2(-e).repeat_interleave(128, 1)
    v, slack, q = v * by, slack * by, got.q.double().cpu()
    step = torch.exp2(torch.floor(torch.log2((v.abs() + slack).clamp(min=2.0 ** -6))) - 3)
    assert bool(((q - v).abs() <= step / 2 + slack + 1e-30).all())
    # Errors are 2^-19 of a value at the root mean square (an order above f32 sums of these lengths); borders are 2^-4 of a
    # value apart or more, so that 2 * 2^-19 / 2^-4 of the values may fall to the other side of one.
    other = q[:, :n] != round_e4m3(v[:, :n].clamp(-448, 448))
    assert int(other.sum()) <= 2.0 ** -14 * other.numel() + 2, int(other.sum())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("t,n,k", GATE_UPS + [(16, 6144, 2048), (16, 2048, 4104)])
def test_gate_up_of_few_rows_has_f32_sums(gpu, t, n, k, kind):
    if form_of(t, n, k, kind, gate_up=True)[0]:
        pytest.skip("the kernel for many rows")
    x = activations(t, k, torch.float32, 15) * (1.5 / k ** 0.5)
    gate, up = weight_of(n, k, kind, 16), weight_of(n, k, kind, 17)
    rows = cev_hip.fp8_rows(x.to(gpu))
    got = cev_hip.gate_up_fp8(rows, Fp8Weight.gate_up(tuple(y.to(gpu) for y in gate), tuple(y.to(gpu) for y in up)))
    check_nearest(got, values(rows.q.cpu(), rows.s.cpu())[:, :k], weight_values(*gate), weight_values(*up))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("t,n,k", [(17, 1000, 520), (300, 384, 2056), (700, 1000, 1032)])
def test_gate_up_of_many_rows_with_f32_sums(gpu, t, n, k, kind):
    """What a caller runs instead of gate_up_fp8 for sums in f32 whatever the number of rows."""
    x = activations(t, k, torch.bfloat16, 15) * (1.5 / k ** 0.5)
    gate, up = weight_of(n, k, kind, 16), weight_of(n, k, kind, 17)
    rows = cev_hip.fp8_rows(x.to(gpu))
    g, u = (cev_hip.linear_fp8(rows, packed(w, gpu), out_dtype=torch.float32) for w in (gate, up))
    got = cev_hip.fp8_rows(cev_hip.swiglu(g, u))
    check_nearest(got, values(rows.q.cpu(), rows.s.cpu())[:, :k], weight_values(*gate), weight_values(*up))
