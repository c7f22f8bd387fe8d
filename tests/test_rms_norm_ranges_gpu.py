"""Normalisation over channels where the values are far from 1: against the formula in 64 bits, by the bounds of the ordinary ones."""
import pytest
import torch

from rembrandt_b200.ops import native_ops as K
from test_rms_norm_gpu import EPS, _backward, _formula, _gamma, _sum_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,C,c_valid", [(5, 64, 60), (3, 2048, 2048)])
@pytest.mark.parametrize("size,delta,eps", [(1e16, 1e-4, EPS), (1e17, 1e-7, EPS), (3e17, 1e-8, EPS), (1e-4, 1e3, EPS), (1e-17, 1e-3, 2.0 ** -126),
                                            (1e-25, 1.0, 2.0 ** -126)])
@pytest.mark.parametrize("add", [False, True])
def test_large_and_small_values(rows, C, c_valid, size, delta, eps, add):
    """3e17 squared times 2048 is 1.9e38: within fp32. What an epsilon adds to a mean is one more rounding."""
    gen = torch.Generator(device="cuda").manual_seed(C)
    make = lambda std: torch.randn((rows, C), generator=gen, device="cuda").clamp(-4, 4).mul(std).bfloat16()
    h, dy, gamma = make(size), make(delta), _gamma(gen, C, c_valid)
    if C == 2048:
        h /= 2                    # squares of up to 4 x the size, 2048 of them
    y, dx, rstd, dgamma = torch.empty_like(h), torch.empty_like(h), torch.empty(rows, device="cuda"), torch.zeros(C, device="cuda")
    K.rms_norm_fwd(h, rows, C, c_valid, eps, gamma, y, rstd=rstd)
    want, r = _formula(h, c_valid, gamma, False, eps)
    assert ((rstd - r).abs() <= _sum_error(C) * r).all()
    assert ((y.double() - want).abs() <= (2.0 ** -8 + 2 * _sum_error(C)) * want.abs()).all()
    more = make(delta / max(size, 1e-3)) if add else None
    K.rms_norm_bwd(h, dy, rows, C, c_valid, rstd, gamma, dgamma, dx, K.rms_norm_scratch(C, "cuda"), add=more)
    dh, dg, sizes, dg_sizes = _backward(h, dy, c_valid, rstd, gamma, False, more)
    # half a step of bf16's smallest numbers beside that of the others
    assert ((dx.double() - dh).abs() <= 2.0 ** -8 * dh.abs() + 2 * _sum_error(C) * sizes + 2.0 ** -134).all()
    assert ((dgamma.double() - dg).abs() <= 2 * _sum_error(C) * dg_sizes).all()
