"""Projections in 8-bit floating point at the ends of their range and in calls
that tests/test_fp8.py does not make; its oracle and tolerances."""
import pytest
import torch

import cev_hip
from cev_hip import Fp8Weight
from test_fp8 import E4M3, E8M0, half_ulp, up128


# ---------------------------------------------------------------------------
# Scales far apart

SCALES_APART = [(112, -40, 448.0), (118, -100, 448.0), (112, 10, 2.0 ** -9), (-118, 120, 448.0), (-118, 120, 2.0 ** -9), (-120, 100, 2.0 ** -9),
                (100, -126, 448.0), (119, -149, 448.0)]


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
