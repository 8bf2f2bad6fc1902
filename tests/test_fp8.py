"""Projections in 8-bit floating point (cev_hip.fp8): rows and weights into
e4m3, the RMS norm into e4m3, products, gate and up with SwiGLU.

The oracle is 64-bit arithmetic on the CPU.  What goes into e4m3 from the
model's type is compared bit for bit: scales are powers of two, so the values
before the rounding are exact.  Tolerances of products:
  - the sum of a column, K products (each exact: 4 bits by 4 bits) and K / 128
    scalings in f32 in any order, each step off by at most 2^-23 of the sum of
    magnitudes so far (which also covers steps that cut bits off):
    (K + K / 64 + 16) 2^-23 A, A the sum of |x w|;
  - outputs in bf16 or e4m3: the matrix cores cut each of eight neighbouring
    columns' products to a multiple of 2^-13 of the largest one's power of
    two, seven of them at most: 7 2^-13 A more;
  - one rounding to the output type, 2^-8 (bf16) or 2^-24 of it.
Integer-valued operands make every sum exact, and are compared for equality.
"""
import math

import pytest
import torch

import cev_hip
from cev_hip import CevError, Fp8Rows, Fp8Weight

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
F64 = torch.float64
CUT = 7 * 2.0 ** -13


# ---------------------------------------------------------------------------
# The oracle


def up128(k):
    return -(-k // 128) * 128


def round_e4m3(x):
    """x (f64, |x| <= 448) to the nearest e4m3 value, ties to the even one; NaN where it is not finite."""
    a = x.abs()
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -6)))
    e = torch.where(torch.ldexp(torch.ones_like(a), e.to(torch.int32)) > a.clamp(min=2.0 ** -6), e - 1, e)
    step = torch.ldexp(torch.ones_like(a), (e - 3).to(torch.int32))
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, float("nan"))


def scale_of(top):
    """The least 2^e, e >= -127, with top <= 448 2^e, by trying."""
    e = torch.full_like(top, -127.0)
    for i in range(-127, 128):
        e = torch.where(448.0 * 2.0 ** e < top, torch.full_like(e, float(i)), e)
    return e


def finite_top(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dims)


def oracle_rows(x):
    """(q, exponents) of x (t, k), f64."""
    t, k = x.shape
    p = torch.zeros(t, up128(k), dtype=F64)
    p[:, :k] = x.to(F64)
    p = p.view(t, -1, 128)
    e = scale_of(finite_top(p, 2))
    return round_e4m3(torch.ldexp(p, -e[..., None])).view(t, -1), e


def oracle_blocks(w):
    n, k = w.shape
    p = torch.zeros(up128(n), up128(k), dtype=F64)
    p[:n, :k] = w.to(F64)
    p = p.view(up128(n) // 128, 128, up128(k) // 128, 128)
    e = scale_of(finite_top(p, (1, 3)))
    return round_e4m3(torch.ldexp(p, -e[:, None, :, None])).view(up128(n), up128(k))[:n, :k], e


def values(q, s):
    """What e4m3 rows and their scales stand for, f64."""
    return q.double() * s.double().repeat_interleave(128, 1)


def weight_values(q, s):
    n, k = q.shape
    return q.double() * s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def check_product(y, x, w, dtype):
    """y against x (t, k) . w (n, k)^T in 64 bits, under the bound of this file's head."""
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    k = x.shape[1]
    tol = ((k + k / 64 + 16) * 2.0 ** -23 + (0 if dtype == torch.float32 else CUT)) * size
    tol = tol + half_ulp(dtype) * (want.abs() + tol) + 1e-40
    off = (y.double().cpu() - want).abs()
    assert y.dtype == dtype and bool((off <= tol).all()), f"worst {float((off / tol).max()):.3g} of the bound"
    # far below the worst case: the root mean square error, the sums' own part 2^-21 of the magnitudes (2^-13 with the cut)
    rms = float((off.square().mean() / size.square().mean()).sqrt())
    assert rms <= half_ulp(dtype) * float((want.square().mean() / size.square().mean()).sqrt()) + (2.0 ** -21 if dtype == torch.float32 else 2.0 ** -13), rms


def gen(seed):
    return torch.Generator().manual_seed(seed)


def activations(t, k, dtype, seed, spread=0.5):
    g = gen(seed)
    x = torch.randn(t, k, generator=g) * torch.exp(spread * torch.randn(k, generator=g))
    return x.to(dtype)


def weight_of(n, k, kind, seed):
    """(q, scales) on the CPU; kind "e8m0", "f32" or "bf16"."""
    g = gen(seed)
    nb, kb = up128(n) // 128, up128(k) // 128
    q = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(E4M3)
    if kind == "e8m0":
        return q, torch.randint(112, 124, (nb, kb), generator=g).to(torch.uint8).view(E8M0)
    s = 0.002 * (0.3 + torch.rand(nb, kb, generator=g))
    return q, s.to(torch.bfloat16) if kind == "bf16" else s


def packed(w, gpu):
    return Fp8Weight(w[0].to(gpu), w[1].to(gpu))


# ---------------------------------------------------------------------------
# Rows and blocks

SIZES = [(1, 1), (1, 8), (3, 127), (5, 128), (2, 129), (7, 200), (64, 2048), (33, 2056), (4, 8200), (2, 20000), (300, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,k", SIZES)
def test_rows(gpu, t, k, dtype):
    vec = 8 if dtype == torch.bfloat16 else 4
    pitch = -(-k // vec) * vec + vec
    x = activations(t, pitch, dtype, 1, spread=2.0)[:, :k]
    x[:, ::5] *= 2.0 ** -12
    got = cev_hip.fp8_rows(_strided(x, pitch, gpu))
    q, e = oracle_rows(x)
    assert got.k == k and got.q.shape == (t, up128(k)) and got.s.shape == (t, up128(k) // 128)
    assert torch.equal(got.s.view(torch.uint8).cpu().double(), e + 127)
    assert torch.equal(got.q.double().cpu(), q)
    assert torch.equal(got.float().double().cpu(), (q * torch.exp2(e).repeat_interleave(128, 1))[:, :k])


def _strided(x, pitch, gpu):
    """x (t, k) on the GPU with rows `pitch` apart and NaN between them."""
    t, k = x.shape
    room = torch.full((t, pitch), float("nan"), dtype=x.dtype, device=gpu)
    room[:, :k] = x.to(gpu)
    return room[:, :k]


@pytest.mark.gpu
def test_every_bf16_value_rounds_as_e4m3(gpu):
    """All 65536 bf16 bit patterns beside a block's largest value of 448 and of 2^e more."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(-1, 64)
    for top in (448.0, 449.0, 2.0 ** -110, 3.0e38, 0.0):
        keep = torch.where(bits.float().abs() <= top, bits, torch.zeros_like(bits)) if top else torch.where(torch.isfinite(bits), torch.zeros_like(bits), bits)
        keep = torch.where(torch.isfinite(bits), keep, bits)
        x = torch.cat([keep, torch.full((keep.shape[0], 64), top).bfloat16()], 1)
        q, e = oracle_rows(x)
        for dtype in (torch.bfloat16, torch.float32):
            got = cev_hip.fp8_rows(x.to(dtype).to(gpu))
            assert torch.equal(got.s.view(torch.uint8).cpu().double(), e + 127), (top, dtype)
            g = got.q.double().cpu()
            assert torch.equal(torch.isnan(g), torch.isnan(q)) and torch.equal(torch.nan_to_num(g), torch.nan_to_num(q)), (top, dtype)


@pytest.mark.gpu
def test_scales_at_their_borders(gpu):
    """Largest values at, just under and just over 448 * 2^e, subnormal ones and zeros."""
    tops = []
    for e in (-149, -140, -127, -126, -120, -100, -1, 0, 1, 60, 118, 119):
        for m in (1.0, 1.75, 1.75 * (1 - 2.0 ** -23), 1.75 * (1 + 2.0 ** -22), 1.9999):
            tops.append(min(m * 2.0 ** e * 256, 3.4e38))
    x = torch.zeros(len(tops), 128)
    x[:, 3] = torch.tensor(tops, dtype=F64).float()
    x[:, 77] = -x[:, 3] / 3
    got = cev_hip.fp8_rows(x.to(gpu))
    q, e = oracle_rows(x)
    assert torch.equal(got.s.view(torch.uint8).cpu().double(), e + 127)
    assert torch.equal(got.q.double().cpu(), q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 8), (127, 130), (128, 128), (129, 264), (1021, 72), (300, 2056)])
def test_blocks(gpu, n, k, dtype):
    vec = 8 if dtype == torch.bfloat16 else 4
    pitch = -(-k // vec) * vec + vec
    w = activations(n, k, dtype, 2, spread=1.0)
    if n > 2:
        w[1, 0] = float("inf")
        w[2, k - 1] = float("nan")
    q, s = cev_hip.fp8_blocks(_strided(w, pitch, gpu))
    want, e = oracle_blocks(w)
    assert q.shape == (n, k) and q.is_contiguous() and s.shape == e.shape
    assert torch.equal(s.view(torch.uint8).cpu().double(), e + 127)
    g = q.double().cpu()
    assert torch.equal(torch.isnan(g), torch.isnan(want)) and torch.equal(torch.nan_to_num(g), torch.nan_to_num(want))


# ---------------------------------------------------------------------------
# The norm


def oracle_norm(x, w, eps, h, plus_one):
    """(x_out, the rows before they go into e4m3), f64."""
    v = x.double()
    if h is not None:
        v = (v + h.double()).to(x.dtype).double()
    return v, v / torch.sqrt(v.square().mean(1, keepdim=True) + eps) * (w.double() + (1 if plus_one else 0))


def check_rows_near(got, want, rel):
    """Rows in e4m3 against the values before the rounding, known up to a factor 1 +- rel: nearest e4m3 value of
    something that near, under a scale that is right for something that near."""
    k = want.shape[1]
    low, high = scale_of(_tops(want) * (1 - rel)), scale_of(_tops(want) * (1 + rel))
    e = got.s.view(torch.uint8).cpu().double() - 127
    assert bool(((e >= low) & (e <= high)).all())
    v = torch.zeros(want.shape[0], up128(k), dtype=F64)
    v[:, :k] = want
    v = torch.ldexp(v.view(v.shape[0], -1, 128), -e[..., None]).view(v.shape[0], -1)
    q = got.q.double().cpu()
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    assert bool(((q - v).abs() <= step / 2 + 2 * rel * v.abs() + 1e-30).all())
    assert bool((q[:, k:] == 0).all())


def _tops(v):
    p = torch.zeros(v.shape[0], up128(v.shape[1]), dtype=F64)
    p[:, : v.shape[1]] = v
    return p.view(v.shape[0], -1, 128).abs().amax(2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("add,plus_one", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("t,k", [(1, 8), (3, 128), (5, 136), (6, 512), (9, 520), (4, 2048), (3, 2200), (7, 4096), (3, 8192), (2, 8200), (2, 20008)])
def test_norm(gpu, t, k, add, plus_one, dtype):
    x, h = activations(t, k, dtype, 3), activations(t, k, dtype, 4)
    w = ((0 if plus_one else 1) + 0.1 * torch.randn(k, generator=gen(5))).to(dtype)
    pitch = -(-k // 8) * 8 + 8
    xg, hg = _strided(x, pitch, gpu), _strided(h, pitch, gpu) if add else None
    got = cev_hip.rms_norm_fp8(xg, w.to(gpu), 1e-6, h=hg, plus_one=plus_one)
    xo, want = oracle_norm(x, w, 1e-6, h if add else None, plus_one)
    assert torch.equal(xg.double().cpu(), xo)  # with h it is the sum, in place
    # f32: the sum of squares within (k / 64 + 16) 2^-24 of itself (64 lanes or more), halved by the root; five roundings more
    check_rows_near(got, want, (k / 128 + 16) * 2.0 ** -24 + 8 * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("t,k", [(515, 512), (514, 1000), (513, 2056), (600, 4096), (513, 4104), (514, 8200), (513, 17000)])
def test_norm_of_many_rows(gpu, t, k, add, dtype):
    x, h = activations(t, k, dtype, 3), activations(t, k, dtype, 4)
    w = (1 + 0.1 * torch.randn(k, generator=gen(5))).to(dtype)
    xg = x.to(gpu)
    got = cev_hip.rms_norm_fp8(xg, w.to(gpu), 1e-6, h=h.to(gpu) if add else None)
    xo, want = oracle_norm(x, w, 1e-6, h if add else None, False)
    assert torch.equal(xg.double().cpu(), xo)
    check_rows_near(got, want, (k / 128 + 16) * 2.0 ** -24 + 8 * 2.0 ** -24)  # as above


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1.0, 1e25, 1e-25])
@pytest.mark.parametrize("t,k", [(64, 4096), (700, 2056), (5, 296)])
def test_norm_is_the_nearest(gpu, t, k, size, dtype):
    """The norm is f64 up to the rounding into e4m3: every value and scale is that of 64-bit arithmetic, also where f32 squares
    leave its range.  (64-bit sums in another order differ by 2^-50 or so: of 10^6 values one is that near a border once in 10^8.)"""
    x = activations(t, k, torch.float32, 61).mul(size).to(dtype)
    w = (1 + 0.1 * torch.randn(k, generator=gen(62))).to(dtype)
    got = cev_hip.rms_norm_fp8(x.to(gpu), w.to(gpu), 0.0)
    q, e = oracle_rows(oracle_norm(x, w, 0.0, None, False)[1])
    assert torch.equal(got.s.view(torch.uint8).cpu().double(), e + 127) and torch.equal(got.q.double().cpu(), q)


@pytest.mark.gpu
def test_norm_of_rows_that_are_zero_or_not_finite(gpu):
    x = activations(5, 200, torch.float32, 6)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    w = torch.ones(200)
    got = cev_hip.rms_norm_fp8(x.to(gpu), w.to(gpu), 1e-6)
    q = got.q.double().cpu()
    assert bool((q[1] == 0).all()) and bool(torch.isnan(q[2, :200]).all()) and bool((q[2, 200:] == 0).all())
    assert bool(torch.isnan(q[3, 9])) and not bool(torch.isnan(q[[0, 1, 4]]).any())


# ---------------------------------------------------------------------------
# Products


def form_of(t, n, k, kind, out=torch.bfloat16, gate_up=False):
    """(rows of a tile, parts of the columns, teams that share a part) of the kernel that runs it; of the one for few rows (0,
    rows of a workgroup, 0)."""
    import ctypes as C
    from cev_hip import _abi
    d = _abi.Fp8Desc(x_dtype=2, out_dtype=2 if gate_up else 0 if out == torch.float32 else 1, scales=0 if kind == "e8m0" else 1, gate_up=gate_up,
                     t=t, n=n, k=k, x_stride=k, out_stride=n)
    rows, parts, teams = C.c_int32(), C.c_int32(), C.c_int32()
    _abi.check(_abi.lib().cev_fp8_form(C.byref(d), C.byref(rows), C.byref(parts), C.byref(teams)))
    return (rows.value, parts.value, teams.value) if teams.value else (0, rows.value, 0)


def test_every_kernel_is_among_the_tested_products(cev):
    def forms_of(products, **kw):
        f = {(kind,) + form_of(t, n, k, kind, **kw) for kind in ("e8m0", "f32") for t, n, k in products}
        few = {(kind, rows) for kind, tile, rows, _ in f if not tile}
        return few, {(kind, tile, teams) for kind, tile, _, teams in f if tile}, {parts for _, tile, parts, _ in f if tile}

    few, tiles, parts = forms_of(PRODUCTS + LARGE)
    assert few == {(kind, rows) for kind in ("e8m0", "f32") for rows in (16, 32, 64)}, few
    assert tiles == {("e8m0", 64, 1), ("e8m0", 64, 2), ("e8m0", 128, 1), ("e8m0", 256, 1), ("f32", 64, 1), ("f32", 64, 2), ("f32", 128, 1), ("f32", 128, 2)}, tiles
    assert parts >= {1, 2} and max(parts) > 2, parts
    few, tiles, parts = forms_of(PRODUCTS + LARGE_F32, out=torch.float32)
    assert few == {(kind, rows) for kind in ("e8m0", "f32") for rows in (16, 32)}, few
    assert tiles == {(kind, 64, teams) for kind in ("e8m0", "f32") for teams in (1, 2)} and max(parts) > 2, (tiles, parts)
    few, tiles, parts = forms_of(GATE_UPS + LARGE_GATE_UPS, gate_up=True)
    assert few == {(kind, rows) for kind in ("e8m0", "f32") for rows in (16, 32)}, few
    assert tiles == {("e8m0", 64, 1), ("e8m0", 64, 2), ("e8m0", 128, 1), ("e8m0", 256, 1), ("f32", 64, 1), ("f32", 64, 2), ("f32", 128, 1), ("f32", 128, 2)}, tiles
    assert max(parts) > 1, parts


LARGE = [(2048, 4096, 2048), (1030, 8320, 264), (4096, 4000, 4104), (400, 4096, 6144), (900, 4000, 8200), (1536, 4000, 8328), (130, 5000, 8200), (260, 2056, 12296)]
LARGE_F32 = [(700, 4100, 2056), (1021, 2056, 4104), (3000, 4100, 1032), (900, 4000, 8200)]
LARGE_GATE_UPS = [(2048, 12288, 4096), (2048, 12288, 6144), (400, 4096, 6080), (900, 4000, 8200), (1000, 1030, 4360)]
PRODUCTS = [(1, 1, 1), (1, 40, 128), (2, 256, 136), (7, 129, 1000), (16, 300, 520), (31, 64, 2048), (32, 1000, 264), (33, 257, 384), (64, 512, 1280),
            (100, 136, 4104), (129, 520, 640), (257, 1000, 392), (400, 384, 1152), (1, 2048, 6144), (300, 2048, 256), (9, 40, 4104),
            (300, 2000, 6152), (333, 4100, 4104), (190, 4100, 1032), (40, 7000, 1160)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("given", ["rows", torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,n,k", PRODUCTS)
def test_linear(gpu, t, n, k, given, kind):
    dtype = torch.bfloat16 if given == "rows" else given
    k = k if given == "rows" or k % 8 == 0 else 8 * -(-k // 8)
    x, w = activations(t, k, torch.float32 if given == "rows" else dtype, 7), weight_of(n, k, kind, 8)
    q, e = oracle_rows(x)
    xg = x.to(gpu)
    if given == "rows":
        xg = Fp8Rows(q.float().to(E4M3).to(gpu), (e + 127).to(torch.uint8).view(E8M0).to(gpu), k)
    wv = weight_values(*w)
    xv = (q * torch.exp2(e).repeat_interleave(128, 1))[:, :k]
    for out_dtype in (torch.bfloat16, torch.float32):
        check_product(cev_hip.linear_fp8(xg, packed(w, gpu), out_dtype=out_dtype), xv, wv, out_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("t,n,k", LARGE)
def test_linear_large(gpu, t, n, k, kind):
    """Several tiles in each direction, last ones in part: rows and columns drawn from all of them."""
    x, w = activations(t, k, torch.bfloat16, 7), weight_of(n, k, kind, 8)
    q, e = oracle_rows(x)
    at_t = torch.cat([torch.randint(0, t, (60,), generator=gen(1)), torch.tensor([0, t - 1])])
    at_n = torch.cat([torch.randint(0, n, (60,), generator=gen(2)), torch.tensor([0, n - 1])])
    y = cev_hip.linear_fp8(x.to(gpu), packed(w, gpu)).cpu()[at_t][:, at_n]
    xv = (q * torch.exp2(e).repeat_interleave(128, 1))[:, :k]
    check_product(y, xv[at_t], weight_values(*w)[at_n], torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("t,n,k", LARGE_F32)
def test_linear_large_f32(gpu, t, n, k, kind):
    x, w = activations(t, k, torch.float32, 7), weight_of(n, k, kind, 8)
    q, e = oracle_rows(x)
    at_t = torch.cat([torch.randint(0, t, (60,), generator=gen(1)), torch.tensor([0, t - 1])])
    at_n = torch.cat([torch.randint(0, n, (60,), generator=gen(2)), torch.tensor([0, n - 1])])
    y = cev_hip.linear_fp8(x.to(gpu), packed(w, gpu)).cpu()[at_t][:, at_n]
    xv = (q * torch.exp2(e).repeat_interleave(128, 1))[:, :k]
    check_product(y, xv[at_t], weight_values(*w)[at_n], torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,k", [(1, 128, 128), (5, 200, 300), (40, 96, 512), (200, 384, 640), (600, 520, 1032), (1000, 1300, 520), (2048, 4096, 260), (1100, 4096, 520), (64, 256, 4096)])
def test_linear_of_integers_is_exact(gpu, t, n, k):
    g = gen(9)
    x = torch.randint(-8, 9, (t, k), generator=g).float()
    q = torch.randint(-8, 9, (n, k), generator=g).float()
    kb, nb = up128(k) // 128, up128(n) // 128
    s = torch.exp2(torch.randint(-1, 2, (nb, kb), generator=g).float())  # sums below 2^24 in units of 1 / 2
    want = x.double() @ weight_values(q.double(), s).t()
    rows = Fp8Rows(torch.nn.functional.pad(x, (0, kb * 128 - k)).to(E4M3).to(gpu), torch.ones(t, kb).to(E8M0).to(gpu), k)
    for scales in (s, s.to(E8M0)):
        w = packed((q.to(E4M3), scales), gpu)
        for operand in (rows, x.to(gpu) if k % 4 == 0 else rows):
            y = cev_hip.linear_fp8(operand, w, out_dtype=torch.float32)
            assert torch.equal(y.double().cpu(), want)
            # (products of at most 64 within 2^13 of each other: nothing is cut)
            assert torch.equal(cev_hip.linear_fp8(operand, w, out_dtype=torch.bfloat16).cpu(), want.float().bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("t", [1, 20, 70, 300, 700, 5000])
def test_linear_nan_and_infinity_stay_in_their_rows(gpu, t, kind):
    x, w = activations(t, 520, torch.bfloat16, 10), weight_of(300, 520, kind, 11)
    clean = cev_hip.linear_fp8(x.to(gpu), packed(w, gpu)).cpu()
    bad = x.clone()
    bad[0, 5] = float("nan")
    if t > 1:
        bad[t - 1, 519] = float("-inf")
    got = cev_hip.linear_fp8(bad.to(gpu), packed(w, gpu)).cpu()
    rows = sorted({0, t - 1})
    assert bool(torch.isnan(got[rows]).all())
    keep = [r for r in range(t) if r not in rows]
    assert torch.equal(got[keep], clean[keep])
    # a weight's NaN stays in its column, as a NaN scale in its columns
    wq = w[0].clone()
    wq[17, 300] = float("nan")
    y = cev_hip.linear_fp8(x.to(gpu), packed((wq, w[1]), gpu)).cpu()
    assert bool(torch.isnan(y[:, 17]).all()) and torch.equal(y[:, :17], clean[:, :17]) and torch.equal(y[:, 18:], clean[:, 18:])
    ws = w[1].clone()
    ws[1, 2] = float("nan")
    y = cev_hip.linear_fp8(x.to(gpu), packed((w[0], ws), gpu)).cpu()
    assert bool(torch.isnan(y[:, 128:256]).all()) and torch.equal(y[:, :128], clean[:, :128]) and torch.equal(y[:, 256:], clean[:, 256:])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 3, 50, 300])
def test_linear_writes_its_rows_only(gpu, t):
    """Outputs with strides and odd starts: what lies between and behind the rows stays."""
    n, k = 133, 256
    x, w = activations(t, k, torch.bfloat16, 12), weight_of(n, k, "f32", 13)
    for dtype in (torch.bfloat16, torch.float32):
        want = cev_hip.linear_fp8(x.to(gpu), packed(w, gpu), out_dtype=dtype)
        for start, pitch in ((0, 136), (1, 139), (2, 148), (3, 133 + 5)):
            room = torch.full((t + 2, pitch), -7.0, dtype=dtype, device=gpu)
            out = room.flatten()[pitch + start: pitch + start + t * pitch].as_strided((t, n), (pitch, 1), pitch + start)
            assert cev_hip.linear_fp8(x.to(gpu), packed(w, gpu), out=out) is out
            assert torch.equal(out, want)
            mask = torch.zeros(room.numel(), dtype=torch.bool, device=gpu)
            mask.as_strided((t, n), (pitch, 1), pitch + start).fill_(True)
            assert bool((room.flatten()[~mask] == -7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,k", [(530000, 40, 4096), (40, 530000, 4096)])
def test_offsets_past_31_bits(gpu, t, n, k):
    """Rows, or a weight, of more than 2^31 bytes: the last ones as by themselves.  Small integers, whose sums are exact in any order."""
    g = torch.Generator(device=gpu).manual_seed(60)
    x = torch.randint(-2, 3, (t, k), generator=g, device=gpu, dtype=torch.int8).bfloat16()
    q = torch.randint(-2, 3, (n, k), generator=g, device=gpu, dtype=torch.int8).to(E4M3)
    s = torch.ones(up128(n) // 128, up128(k) // 128, device=gpu)
    y = cev_hip.linear_fp8(x, Fp8Weight(q, s))
    rows, cols = min(t, 200), min(n, 128 + n % 128)
    want = (x[-rows:].double() @ q[-cols:].double().t()).to(torch.bfloat16)
    assert torch.equal(y[-rows:, -cols:], want)


@pytest.mark.gpu
def test_no_rows(gpu):
    w = packed(weight_of(40, 72, "e8m0", 14), gpu)
    x = torch.zeros(0, 72, dtype=torch.bfloat16, device=gpu)
    assert cev_hip.linear_fp8(x, w).shape == (0, 40) and cev_hip.fp8_rows(x).q.shape == (0, 128)
    assert cev_hip.linear_fp8(cev_hip.fp8_rows(x), w).shape == (0, 40)
    assert cev_hip.rms_norm_fp8(x, torch.ones(72, dtype=torch.bfloat16, device=gpu), 1e-6).s.shape == (0, 1)
    gu = Fp8Weight.gate_up(*[tuple(y.to(gpu) for y in weight_of(40, 72, "e8m0", 14)) for _ in range(2)])
    assert cev_hip.gate_up_fp8(x, gu).q.shape == (0, 128)


# ---------------------------------------------------------------------------
# Gate and up


GATE_UPS = [(1, 1, 8), (1, 256, 128), (3, 130, 264), (16, 1000, 512), (20, 136, 4104), (33, 128, 1032), (65, 300, 640), (130, 520, 384), (300, 384, 256), (513, 640, 520),
            (260, 5130, 264), (1030, 4100, 200), (11, 136, 4104), (132, 2217, 2104)]


def check_gate_up(got, xv, gate, up):
    """got against silu(x . gate^T) * (x . up^T) in 64 bits, x (t, k), gate and up (n, k)."""
    t, k, n = xv.shape[0], xv.shape[1], gate.shape[0]
    g, u = (xv @ w.t() for w in (gate, up))
    size = [xv.abs() @ w.abs().t() for w in (gate, up)]
    want = g * torch.sigmoid(g) * u
    # each product within c = (K + K / 64 + 16) 2^-23 of its sum of magnitudes; silu's slope is at most 1.1; the exponential of
    # -g within 2^-22 (1 + |g|) of itself, and the rest a few f32 roundings
    c = (k + k / 64 + 16) * 2.0 ** -23 + CUT
    tol = 1.1 * c * size[0] * (u.abs() + c * size[1]) + g.abs() * c * size[1] + want.abs() * (2.0 ** -22 * (1 + g.abs()) + 2.0 ** -21)
    e = got.s.view(torch.uint8).cpu().double() - 127
    low, high = (scale_of(_tops((want.abs() + s * tol).clamp(min=0))) for s in (-1, 1))
    assert bool(((e >= low) & (e <= high)).all())
    v, slack = (torch.zeros(t, up128(n), dtype=F64) for _ in range(2))
    v[:, :n], slack[:, :n] = want, tol
    v, slack = (torch.ldexp(z.view(t, -1, 128), -e[..., None]).view(t, -1) for z in (v, slack))
    q = got.q.double().cpu()
    step = torch.exp2(torch.floor(torch.log2((v.abs() + slack).clamp(min=2.0 ** -6))) - 3)
    assert bool(((q - v).abs() <= step / 2 + slack + 1e-30).all())
    assert bool((q[:, n:] == 0).all())
    # the bound is wide where sums are long: nearly all values are the nearest of the exact ones.  On data like these the
    # cut leaves each product within 2^-13 of itself, so of values 2^-4 of themselves apart at least 2 * 2 * 2^-13 / 2^-4 may fall to the other side
    assert float((q[:, :n] != round_e4m3(v[:, :n].clamp(-448, 448))).double().mean()) <= 2.0 ** -7 + 2 / q.numel()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("given", ["rows", torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,n,k", GATE_UPS)
def test_gate_up(gpu, t, n, k, given, kind):
    x = activations(t, k, torch.float32 if given == "rows" else given, 15)
    x *= 1.5 / math.sqrt(k)
    gate, up = weight_of(n, k, kind, 16), weight_of(n, k, kind, 17)
    rows = oracle_rows(x)
    xv = (rows[0] * torch.exp2(rows[1]).repeat_interleave(128, 1))[:, :k]
    xg = cev_hip.fp8_rows(x.to(gpu)) if given == "rows" else x.to(gpu)
    w = Fp8Weight.gate_up(tuple(y.to(gpu) for y in gate), tuple(y.to(gpu) for y in up))
    got = cev_hip.gate_up_fp8(xg, w)
    check_gate_up(got, xv, weight_values(*gate), weight_values(*up))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("t,n,k", LARGE_GATE_UPS)
def test_gate_up_of_many_tiles(gpu, t, n, k, kind):
    """Rows and blocks of columns drawn from all tiles of a wide layer."""
    g = torch.Generator(device=gpu).manual_seed(36)
    x = torch.randn(t, k, generator=g, device=gpu) * 0.03
    weights = [((torch.randn(n, k, generator=g, device=gpu) * 100).clamp(-448, 448).to(E4M3), weight_of(n, k, kind, 37 + i)[1].to(gpu)) for i in range(2)]
    rows = cev_hip.fp8_rows(x)
    got = cev_hip.gate_up_fp8(rows, Fp8Weight.gate_up(*weights))
    at = torch.tensor([r for r in (0, 1, 127, 128, 255, 256, 300, 1000, 1023, 1024, 2000) if r < t] + [t - 1])
    blocks = [b for b in (0, 1, 31, 64, 95) if b < up128(n) // 128]
    xv = values(rows.q[at.to(gpu)].cpu(), rows.s[at.to(gpu)].cpu())[:, :k]
    for b in blocks:
        cols = slice(128 * b, min(128 * b + 128, n))
        wv = [q[cols].cpu().double() * s[b].cpu().double().repeat_interleave(128)[:k] for q, s in weights]
        gv, uv = xv @ wv[0].t(), xv @ wv[1].t()
        want = gv * torch.sigmoid(gv) * uv
        have = (got.q[:, cols].cpu()[at].double() * got.s[:, b].cpu()[at].double()[:, None])
        # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale), and the sums' 2^-13 of a typical size
        tol = want.abs() * 2.0 ** -4 + want.abs().amax(1, keepdim=True) * (2.0 ** -17 + 2.0 ** -11)
        assert bool(((have - want).abs() <= tol).all()), b


@pytest.mark.gpu
@pytest.mark.parametrize("t", [2, 40, 300])
def test_gate_up_large_and_bad_values(gpu, t):
    """Gates far out on both sides (silu is g, or 0), and rows with NaN."""
    n, k = 200, 128
    q = torch.zeros(n, k)
    q[:, 0] = torch.linspace(-400, 400, n)
    gate = (q.to(E4M3), torch.ones(2, 1))
    q = torch.zeros(n, k)
    q[:, 1] = 1
    up = (q.to(E4M3), torch.ones(2, 1))
    x = torch.zeros(t, k)
    x[:, 0], x[:, 1] = 1, 2
    x[t - 1, 3] = float("nan")
    got = cev_hip.gate_up_fp8(x.to(gpu), Fp8Weight.gate_up(*[tuple(y.to(gpu) for y in w) for w in (gate, up)]))
    g = gate[0][:, 0].double()
    want, e = oracle_rows((g * torch.sigmoid(g) * 2)[None])
    rows = got.q.double().cpu()
    assert torch.equal(got.s.view(torch.uint8).cpu().double()[:-1], (e + 127).expand(t - 1, -1))
    assert torch.equal(rows[:-1], want.expand(t - 1, -1))
    assert bool(torch.isnan(rows[-1, :n]).all()) and bool((rows[-1, n:] == 0).all())


# ---------------------------------------------------------------------------
# Together


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 17, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_calls_together(gpu, t, dtype):
    """A layer's norm, gate and up, down: each call on the one before's rows, against the composition of single results in 64 bits."""
    hidden, inter = 512, 1000
    x, h = activations(t, hidden, dtype, 18), activations(t, hidden, dtype, 19)
    w = (1 + 0.1 * torch.randn(hidden, generator=gen(20))).to(dtype)
    weights = [0.03 * torch.randn(n, k, generator=gen(21 + i)) for i, (n, k) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    blocks = [cev_hip.fp8_blocks(m.to(dtype).to(gpu)) for m in weights]
    gu, down = Fp8Weight.gate_up(blocks[0], blocks[1]), Fp8Weight(*blocks[2])
    xg = x.to(gpu)
    rows = cev_hip.rms_norm_fp8(xg, w.to(gpu), 1e-6, h=h.to(gpu))
    act = cev_hip.gate_up_fp8(rows, gu)
    y = cev_hip.linear_fp8(act, down, out_dtype=dtype)
    assert torch.equal(xg.cpu(), (x.double() + h.double()).to(dtype))
    wv = [weight_values(q.cpu(), s.cpu()) for q, s in blocks]
    r = rows.float().double().cpu()
    check_rows_near(rows, oracle_norm(x, w, 1e-6, h, False)[1], 40 * 2.0 ** -24)
    g, u = r @ wv[0].t(), r @ wv[1].t()
    a = act.float().double().cpu()
    full = g * torch.sigmoid(g) * u
    top = _tops(full).repeat_interleave(128, 1)[:, :inter]
    assert bool(((a - full).abs() <= full.abs() * 2.0 ** -4 * 1.01 + top * 2.0 ** -16).all())
    check_product(y, a, wv[2], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 48, 300])
def test_plain_rows_are_rows_first(gpu, t):
    """A product of rows in the model's type is the product of fp8_rows, bit for bit, and a repeated call gives the same bits."""
    x, w = activations(t, 1032, torch.bfloat16, 24).to(gpu), packed(weight_of(520, 1032, "f32", 25), gpu)
    a = cev_hip.linear_fp8(x, w, out_dtype=torch.float32)
    assert torch.equal(a, cev_hip.linear_fp8(cev_hip.fp8_rows(x), w, out_dtype=torch.float32))
    assert torch.equal(a, cev_hip.linear_fp8(x, w, out_dtype=torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 40, 300])
def test_captured_calls_replay(gpu, t):
    """A layer's calls in a graph, replayed on new values with eager work between."""
    hidden, inter = 512, 640
    w = torch.ones(hidden, dtype=torch.bfloat16, device=gpu)
    blocks = [tuple(y.to(gpu) for y in weight_of(n, k, "f32", 26 + i)) for i, (n, k) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    gu, down = Fp8Weight.gate_up(blocks[0], blocks[1]), Fp8Weight(*blocks[2])
    x, h, xo = (torch.zeros(t, hidden, dtype=torch.bfloat16, device=gpu) for _ in range(3))

    def layer():
        rows = cev_hip.rms_norm_fp8(x, w, 1e-6, h=h, x_out=xo)
        return cev_hip.linear_fp8(cev_hip.gate_up_fp8(rows, gu), down), cev_hip.linear_fp8(xo, down_in)

    down_in = packed(weight_of(264, hidden, "e8m0", 30), gpu)
    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for i in range(4):
        x.copy_(activations(t, hidden, torch.bfloat16, 40 + i))
        h.copy_(activations(t, hidden, torch.bfloat16, 50 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in out]
        for a, b in zip(got, layer()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_calls_on_two_streams(gpu):
    """Calls that overlap on two streams have workspaces and outputs of their own."""
    w = packed(weight_of(520, 1024, "f32", 31), gpu)
    xs = [activations(t, 1024, torch.float32, 32 + i).to(gpu) for i, t in enumerate((300, 65))]
    want = [cev_hip.linear_fp8(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (x, s) in enumerate(zip(xs, streams)):
            got[i].append(cev_hip.linear_fp8(x, w, stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,k", [(2, 40, 128), (20, 40, 1032), (3000, 4100, 1032), (900, 4000, 8200)])
@pytest.mark.parametrize("x_exp,w_exp", [(-110, -40), (-40, -110), (10, 112), (-118, 120)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_scales_far_apart(gpu, t, n, k, x_exp, w_exp, out_dtype):
    """Products of a row's and a weight's scale that leave f32's range, where the result stays within it."""
    m = 2.0 ** -9 if x_exp + w_exp > 100 else 448.0
    x = torch.full((t, k), m * 2.0 ** x_exp, dtype=torch.float32, device=gpu)
    x[:, ::128] = 448 * 2.0 ** x_exp  # each block's scale
    q = torch.full((n, k), m).to(E4M3)
    q[:, ::128] = 0
    w = Fp8Weight(q.to(gpu), torch.full((up128(n) // 128, up128(k) // 128), 2.0 ** w_exp, device=gpu))
    want = m * m * 2.0 ** (x_exp + w_exp) * (k - len(range(0, k, 128)))
    y = cev_hip.linear_fp8(x, w, out_dtype=out_dtype).double().cpu()
    # equal products: nothing is cut, and sums of fewer than 2^24 of them are exact
    assert 2.0 ** -126 < want < 2.0 ** 127 and bool(((y - want).abs() <= half_ulp(out_dtype) * want).all()), (want, y.min(), y.max())


@pytest.mark.gpu
def test_no_rows(gpu):
    w = packed(weight_of(40, 300, "f32", 35), gpu)
    gu = Fp8Weight.gate_up(*[tuple(y.to(gpu) for y in weight_of(40, 300, "e8m0", 35))] * 2)
    x = torch.zeros(0, 300, device=gpu)
    rows = cev_hip.fp8_rows(x)
    assert rows.q.shape == (0, 384) and rows.s.shape == (0, 3) and rows.float().shape == (0, 300)
    assert cev_hip.rms_norm_fp8(x, torch.ones(300, device=gpu), 1e-6, h=torch.zeros_like(x)).q.shape == (0, 384)
    for given in (x, rows):
        assert cev_hip.linear_fp8(given, w).shape == (0, 40)
        assert cev_hip.gate_up_fp8(given, gu).s.shape == (0, 1)


@pytest.mark.gpu
def test_given_outputs(gpu):
    x = activations(20, 300, torch.float32, 34).to(gpu)
    rows = cev_hip.fp8_rows(x)
    other = Fp8Rows(torch.empty_like(rows.q), torch.empty_like(rows.s), 300)
    got = cev_hip.fp8_rows(x, out=other)
    assert got.q.data_ptr() == other.q.data_ptr() and torch.equal(got.q.view(torch.uint8), rows.q.view(torch.uint8))
    assert torch.equal(got.s.view(torch.uint8), rows.s.view(torch.uint8))
    dense = torch.zeros(20, 128, device=gpu)
    with pytest.raises(CevError, match="of their own"):
        cev_hip.fp8_rows(dense, out=Fp8Rows(dense.view(E4M3)[:, :128].as_strided((20, 128), (128, 1)), torch.empty(20, 1, dtype=E8M0, device=gpu), 128))
    square = Fp8Weight.gate_up(*[tuple(y.to(gpu) for y in weight_of(128, 128, "f32", 35))] * 2)
    rows_128 = cev_hip.fp8_rows(dense)
    with pytest.raises(CevError, match="of its own"):
        cev_hip.gate_up_fp8(rows_128, square, out=rows_128)
    with pytest.raises(CevError, match="of its own"):
        cev_hip.linear_fp8(dense, packed(weight_of(128, 128, "f32", 35), gpu), out=dense)
    with pytest.raises(CevError, match="Fp8Rows of 20 rows"):
        cev_hip.fp8_rows(x, out=Fp8Rows(rows.q[:10], rows.s[:10], 300))
    with pytest.raises(CevError, match="contiguous"):
        cev_hip.fp8_rows(x.t())
    w = packed(weight_of(40, 300, "f32", 35), gpu)
    with pytest.raises(CevError, match=r"\(20, 40\)"):
        cev_hip.linear_fp8(rows, w, out=torch.empty(20, 41, device=gpu))
    with pytest.raises(CevError, match="300 columns for a weight"):
        cev_hip.linear_fp8(rows, packed(weight_of(40, 128, "f32", 35), gpu))
    with pytest.raises(CevError, match="multiple of 4"):
        cev_hip.fp8_rows(torch.zeros(3, 9, device=gpu))
    with pytest.raises(CevError, match="aligned"):
        cev_hip.fp8_rows(torch.zeros(400, device=gpu)[1:].as_strided((2, 128), (128, 1)))
    with pytest.raises(CevError, match="gate_up_fp8"):
        cev_hip.linear_fp8(rows, Fp8Weight.gate_up(*[tuple(y.to(gpu) for y in weight_of(40, 300, "f32", 35))] * 2))
    with pytest.raises(CevError, match="no Fp8Weight.gate_up"):
        cev_hip.gate_up_fp8(rows, w)


# ---------------------------------------------------------------------------
# Refusals (CPU)


def test_refusals_before_any_launch(cev):
    z = torch.zeros
    w = type("W", (), dict(is_gate_up=False, data=z(4096 * 8 + 32, dtype=torch.uint8), n=256, k=128, scale_kind=0))
    with pytest.raises(CevError, match="float16") as err:
        cev_hip.fp8_rows(z(2, 64, dtype=torch.float16))
    assert err.value.code == -2
    with pytest.raises(CevError, match="on the GPU"):
        cev_hip.fp8_rows(z(2, 64))
    with pytest.raises(CevError, match="on the GPU"):
        cev_hip.fp8_blocks(z(2, 64))
    with pytest.raises(CevError, match=r"\(t, k\)"):
        cev_hip.fp8_rows(z(64))
    with pytest.raises(CevError, match="share the dtype"):
        cev_hip.rms_norm_fp8(z(2, 64), z(64, dtype=torch.bfloat16), 1e-6)
    with pytest.raises(CevError, match="x's shape"):
        cev_hip.rms_norm_fp8(z(2, 64), z(64), 1e-6, h=z(3, 64))
    with pytest.raises(CevError, match="a value for each column"):
        cev_hip.rms_norm_fp8(z(2, 64), z(63), 1e-6)
    with pytest.raises(CevError, match="goes with h"):
        cev_hip.rms_norm_fp8(z(2, 64), z(64), 1e-6, x_out=z(2, 64))
    with pytest.raises(CevError, match="columns for a weight"):
        cev_hip.linear_fp8(z(2, 64), w)
    with pytest.raises(CevError, match="float64"):
        cev_hip.linear_fp8(z(2, 128), w, out_dtype=torch.float64)
    with pytest.raises(CevError, match="on the GPU"):
        cev_hip.linear_fp8(z(2, 128), w)
    with pytest.raises(CevError, match="what fp8_rows makes"):
        cev_hip.linear_fp8(Fp8Rows(z(2, 128), z(2, 1).to(E8M0), 128), w)
    with pytest.raises(CevError, match="float8_e4m3fn"):
        Fp8Weight(z(128, 128), z(1, 1))
    with pytest.raises(CevError, match="one for 128 x 128 values"):
        Fp8Weight(z(129, 128).to(E4M3), z(1, 1))
    with pytest.raises(CevError, match="scales of"):
        Fp8Weight(z(128, 128).to(E4M3), z(1, 1, dtype=torch.float16))
    with pytest.raises(CevError, match="one shape"):
        Fp8Weight.gate_up((z(128, 128).to(E4M3), z(1, 1)), (z(64, 128).to(E4M3), z(1, 1)))
    with pytest.raises(CevError, match="one type"):
        Fp8Weight.gate_up((z(128, 128).to(E4M3), z(1, 1)), (z(128, 128).to(E4M3), z(1, 1).to(E8M0)))


def test_abi_refusals(cev):
    """The C calls' own checks: all of these return before the GPU is looked at."""
    import ctypes as C
    L = cev._abi.lib()
    desc = cev._abi.Fp8Desc
    size = C.c_size_t()
    p = C.c_void_p(4096)

    def refused(rc, code, text):
        assert rc == code and text in L.cev_last_error().decode(), (rc, L.cev_last_error())

    refused(L.cev_fp8_rows(2, 1, 8, p, 8, p, p, None), -2, "dtype")
    refused(L.cev_fp8_rows(0, -1, 8, p, 8, p, p, None), -1, "rows")
    refused(L.cev_fp8_rows(0, 1, 0, p, 8, p, p, None), -1, "values")
    refused(L.cev_fp8_rows(0, 1, 1 << 31, p, 8, p, p, None), -1, "values")
    refused(L.cev_fp8_rows(0, 2, 8, p, 4, p, p, None), -1, "stride")
    refused(L.cev_fp8_rows(0, 2, 8, p, 10, p, p, None), -1, "stride")
    refused(L.cev_fp8_rows(0, 2, 8, C.c_void_p(4100), 8, p, p, None), -1, "aligned")
    refused(L.cev_fp8_rows(0, 2, 8, p, 8, None, p, None), -1, "output")
    refused(L.cev_fp8_rows(0, 1 << 28, 1 << 30, p, 1 << 30, p, p, None), -2, "too many")
    refused(L.cev_fp8_rows(0, 1 << 25, 1 << 11, p, 1 << 11, C.c_void_p(8192), C.c_void_p(16384), None), -2, "too many")  # 2^33 threads
    assert L.cev_fp8_rows(0, 0, 8, None, 8, None, None, None) == 0
    refused(L.cev_fp8_rms_norm(1, 2, 8, p, 8, None, 0, None, 0, None, 1e-6, 0, p, p, None), -1, "null w")
    refused(L.cev_fp8_rms_norm(1, 2, 8, p, 8, p, 8, None, 0, p, 1e-6, 0, p, p, None), -1, "null x_out")
    refused(L.cev_fp8_rms_norm(1, 2, 8, p, 8, None, 0, None, 0, p, float("nan"), 0, p, p, None), -1, "eps")
    refused(L.cev_fp8_blocks(0, 0, 8, p, 8, p, p, None), -1, "weight of")
    refused(L.cev_fp8_weight_size(0, 8, 0, C.byref(size)), -1, "weight of")
    assert L.cev_fp8_weight_size(1, 1, 0, C.byref(size)) == 0 and size.value == 8 * 4100
    assert L.cev_fp8_weight_size(129, 129, 1, C.byref(size)) == 0 and size.value == 2 * 2 * 8 * 4100
    assert L.cev_fp8_weight_size((1 << 31) - 257, 1 << 30, 0, C.byref(size)) == 0 and size.value > 1 << 60
    refused(L.cev_fp8_weight_pack(128, 128, 2, p, 128, p, 1, None, 0, None, 0, p, 1 << 20, None), -2, "scale kind")
    refused(L.cev_fp8_weight_pack(128, 128, 1, p, 127, p, 1, None, 0, None, 0, p, 1 << 20, None), -1, "stride")
    refused(L.cev_fp8_weight_pack(128, 128, 1, p, 128, p, 1, None, 0, None, 0, p, 100, None), -4, "needed")
    refused(L.cev_fp8_weight_pack(128, 128, 1, p, 128, p, 1, p, 128, None, 0, p, 1 << 20, None), -1, "null")

    def product(d, x=p, xs=None, w=p, wb=1 << 40, out=C.c_void_p(8192), outs=None, work=p, wk=1 << 40):
        return L.cev_fp8_product(C.byref(d), x, xs, w, wb, out, outs, work, wk, None)

    good = dict(x_dtype=1, out_dtype=1, scales=1, gate_up=0, t=4, n=256, k=128, x_stride=128, out_stride=256)
    refused(product(desc(**dict(good, x_dtype=5))), -2, "x dtype")
    refused(product(desc(**dict(good, out_dtype=2))), -2, "out dtype")
    refused(product(desc(**dict(good, gate_up=1))), -2, "out dtype")
    refused(product(desc(**dict(good, scales=3))), -2, "scale kind")
    refused(product(desc(**dict(good, t=-1))), -1, "rows")
    refused(product(desc(**dict(good, n=0))), -1, "weight")
    refused(product(desc(**dict(good, t=1 << 30, n=1 << 30))), -1, "too large")
    refused(product(desc(**dict(good, t=1 << 30, k=1 << 30, x_stride=1 << 30))), -1, "too large")
    refused(product(desc(**good), wb=100), -4, "weight of 100")
    refused(product(desc(**good), x=None), -1, "null")
    refused(product(desc(**good), xs=p), -1, "scales")
    refused(product(desc(**dict(good, x_dtype=2))), -1, "scales")
    refused(product(desc(**dict(good, x_stride=120))), -1, "stride of x")
    refused(product(desc(**dict(good, x_stride=132))), -1, "stride of x")
    refused(product(desc(**dict(good, out_stride=255))), -1, "stride of out")
    refused(product(desc(**good), out=C.c_void_p(4097)), -1, "misaligned")
    refused(product(desc(**good), x=C.c_void_p(4104)), -1, "aligned")
    refused(L.cev_fp8_rows(0, 2, 8, p, 8, p, C.c_void_p(8192), None), -1, "of their own")
    refused(L.cev_fp8_rms_norm(1, 2, 8, p, 8, None, 0, None, 0, C.c_void_p(8192), 1e-6, 0, p, C.c_void_p(16384), None), -1, "of their own")
    refused(product(desc(**good), out=p), -1, "of its own")
    refused(product(desc(**dict(good, x_dtype=2, n=1 << 27, out_stride=1 << 27)), xs=C.c_void_p(16384)), -2, "grid too large")
    big = desc(**dict(good, t=4000))
    assert L.cev_fp8_work_size(C.byref(big), C.byref(size)) == 0 and size.value >= 4000 * 129
    refused(product(big, wk=size.value - 1), -4, "workspace")
    refused(product(big, work=C.c_void_p(4096 + 16)), -1, "workspace")
    assert product(desc(**dict(good, t=0)), x=None, out=None) == 0


def test_oracle_scales_and_roundings():
    """The oracle itself: torch's conversion where it saturates nothing, scales by hand."""
    x = torch.linspace(-448, 448, 100001, dtype=F64).float()
    assert torch.equal(round_e4m3(x.double()), x.to(E4M3).double())
    tiny = torch.ldexp(torch.arange(-600, 601, dtype=F64), torch.tensor(-15))
    assert torch.equal(round_e4m3(tiny), tiny.float().to(E4M3).double())
    tops = torch.tensor([0.0, 448.0, 448.5, 224.0, 224.5, 1.75, 1.76, 2.0 ** -149, 3.0e38], dtype=F64)
    assert scale_of(tops).tolist() == [-127, 0, 1, -1, 0, -8, -7, -127, 120]
