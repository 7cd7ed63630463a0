"""Orthogonalisation with polynomials that stretch: the first two steps are one only where their joint matrices fit f16.

Tolerance.  Single steps, with d = 2^-11 / sqrt(3) the root mean square of a rounding to f16, |.|_F the Frobenius and |.| the
spectral norm, F = b G + c G^2 and independent roundings (squares add):
    dG = d |G|_F,   dF = d |F|_F + (|b| + 2 |c| |G|) dG,   dx' = L dx + |x| dF + d |x'|_F
L is the largest |slope| of a s + b s^3 + c s^5 between 0 and the largest singular value, which bounds the divided differences by
which an odd function of the singular values moves.  An fp32 update enters in two halves except as the factor of F: d |x|_F |F|.
A factor 4 covers the tail; the result is rounded to bf16 once, half a step, 2^-8 relative."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 2.0 ** -11 / math.sqrt(3)
STRETCHING = [(1.0, 16.0, -16.0), (0.25, 0.0, 0.0), (1.5, -0.5, 0.0)]       # at s^2 = 1/2, (1 + F)^2 - 1 = 24: beyond f16 at 2^12


def _single_steps64(u, coefficients):
    x = u.double()
    tall = x.shape[0] > x.shape[1]
    x = x.mT if tall else x
    x = x / (x.norm() + 1e-7)
    err2, first = 0.0, (D * float(x.norm())) ** 2 if u.dtype == torch.float32 else 0.0
    for a, b, c in coefficients:
        g = x @ x.mT
        f = b * g + c * (g @ g)
        new = a * x + f @ x
        s = float(torch.linalg.matrix_norm(x, 2))
        z = torch.linspace(0, s, 4097, dtype=torch.float64) ** 2
        slope = float((a + 3 * b * z + 5 * c * z * z).abs().max())
        df = (D * float(f.norm())) ** 2 + ((abs(b) + 2 * abs(c) * s * s) * D * float(g.norm())) ** 2
        top_f = float(torch.linalg.matrix_norm(f, 2))
        err2 = slope ** 2 * err2 + s * s * df + top_f ** 2 * first + (D * float(new.norm())) ** 2
        first, x = 0.0, new
    return (x.mT if tall else x), math.sqrt(err2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(2, 2), (48, 80), (128, 40), (300, 260), (160, 500)])
def test_stretching_polynomials_stay_finite(shape, dtype):
    from bibo_b200 import functional as Fn
    g = torch.Generator().manual_seed(sum(shape))
    u = 1e-3 * torch.randn(shape, generator=g)
    u[0, 1] += 1.0                                       # two equal singular values far above the rest, along the axes
    u[1, 0] -= 1.0
    u = u.to(dtype)
    want, bound = _single_steps64(u, STRETCHING)
    got = Fn.orthogonalize(u.to(DEV), 3, STRETCHING).double().cpu()
    assert bool(got.isfinite().all())
    assert float((got - want).norm()) <= 4 * bound + 2.0 ** -8 * float(want.norm())
