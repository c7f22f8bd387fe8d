"""Clipping where scale, coefficient and gradients are far from 1, against the formula in 64 bits. A factor has two roundings,
what it makes of a value one more to fp32 and one to the value's type."""
import pytest
import torch

from rembrandt_b200.ops import native_ops as K
from rembrandt_b200.optim.sgd import reference_step

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,scale,coef", [(1e30, 2.0 ** -100, 2.0 ** -40), (1e38, 2.0 ** -70, 3e-20), (3e37, 2.0 ** -126, 2.0 ** -13 / 3), (1e36, 1.0, 1e-37),
                                             (1e20, 2.0 ** -10, 1e-30), (1e-20, 1e20, 0.3), (1.0, 2.0 ** -126, 0.7), (1e10, 2.0 ** -120, 1e-30)])
def test_factors_far_from_one(dtype, size, scale, coef):
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = (torch.randn(5003, generator=gen, device="cuda").clamp(-3, 3) * size).to(dtype)
    out = torch.tensor([1.0, coef], device="cuda")
    want = g.double() * (scale * out[1].double())
    K.clip_grads([g], out, scale=scale)
    half = max(U, torch.finfo(dtype).eps / 2) if dtype != torch.float32 else 0.0
    smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    assert ((g.double() - want).abs() <= (half + 4 * U) * want.abs() + 2 * smallest).all()


@pytest.mark.parametrize("size,scale,coef", [(1e30, 2.0 ** -100, 2.0 ** -40), (1e38, 2.0 ** -70, 3e-20), (1e36, 1.0, 1e-37), (1.0, 1.0, 0.3)])
@pytest.mark.parametrize("mode", range(6))
@pytest.mark.parametrize("n", [1025, 4_194_311])
@pytest.mark.parametrize("phases", [(7,), (1, 6)])
def test_updates_with_factors_far_from_one(size, scale, coef, mode, n, phases):
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = torch.randn(n, generator=gen, device="cuda").clamp(-3, 3) * size
    out = torch.tensor([1.0, coef], device="cuda")
    factor = scale * out[1].double().item()
    unit = size * factor        # of a clipped gradient
    w, v = (torch.randn(n, generator=gen, device="cuda").clamp(-3, 3) * unit for _ in range(2))
    w16 = torch.empty(n, device="cuda", dtype=torch.bfloat16)
    ref = [t.double() for t in (w, g, v)]
    for phase in phases:
        reference_step(*ref, 0.1, 0.9, 5e-4, factor, mode, phase)
        K.sgd_fused(w, g, v, w16, n, 0.1, 0.9, 5e-4, scale, mode, phase, clip=out)
    for got, want in zip((w, g, v), ref):
        # at most eight operations on values below 10 units, and the factor's roundings
        assert ((got.double() - want).abs() <= 16 * U * 10 * unit + 2.0 ** -149).all()
    assert torch.equal(w16, w.bfloat16())
