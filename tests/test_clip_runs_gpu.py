"""Clipping of lists so long that a block takes a run of several chunks, which may pass from one tensor and type into the next: every
value against the formula in 64 bits. A norm has at most seven roundings of fp32 between a square and the 64-bit sum (3.5 in the
root) and one of its own, a factor three more."""
import math

import pytest
import torch

from rembrandt_b200.ops import native_ops as K

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
CHUNK_BYTES = 16 * 1024      # of a tensor that a block takes at a time; the kernel starts at most 3552 blocks


def _long_list():
    gen = torch.Generator(device="cuda").manual_seed(3)
    make = lambda n, t: torch.randn(n, generator=gen, device="cuda").to(t)
    types = [torch.float32, torch.bfloat16, torch.float16]
    small = [make(n % 97 + 5000 * (n % 3) + 1, types[n % 3]) for n in range(120)]
    odd = [make(9001 + 7 * n, types[n % 3])[n % 5 + 1:] for n in range(60)]
    return [make(20_000_003, torch.float32), *small[:60], make(20_000_005, torch.bfloat16), *odd, make(9_000_001, torch.float16), *small[60:]]


@pytest.mark.parametrize("share,scale", [(0.31, 1.0), (1.5, 3.0)])
@pytest.mark.parametrize("few", [False, True])
def test_runs_of_chunks_through_many_tensors(share, scale, few):
    """`few`: at most as many tensors as the small table holds."""
    tensors = _long_list()
    if few:
        tensors = tensors[:1] + tensors[30:100] + tensors[121:161]
        assert len(tensors) <= 128
    assert sum(-(-t.numel() * t.element_size() // CHUNK_BYTES) for t in tensors) > 2 * 3552
    before = [t.clone() for t in tensors]
    norm = scale * math.sqrt(sum(t.double().square().sum().item() for t in tensors))
    out = torch.zeros(2, device="cuda")
    K.grad_norm(tensors, share * norm, out, K.grad_norm_scratch("cuda"), scale=scale)
    got, coef = out.tolist()
    assert abs(got - norm) <= 6 * U * norm and abs(coef - min(1.0, share)) <= 9 * U
    K.clip_grads(tensors, out, scale=scale)
    for i, (t, b) in enumerate(zip(tensors, before)):
        want = b.double() * (scale * min(1.0, share))
        half_step = max(U, torch.finfo(t.dtype).eps / 2)
        smallest = torch.finfo(t.dtype).smallest_normal * torch.finfo(t.dtype).eps / 2
        assert ((t.double() - want).abs() <= (half_step + 9 * U) * want.abs() + smallest * 1.001).all(), i


def test_what_lies_around_the_tensors_of_a_run_stays():
    flat = torch.full((40_000_000,), 2.0, device="cuda")
    parts = [flat[5: 15_000_002], *(flat[16_000_000 + 1000 * i + i % 4: 16_000_000 + 1000 * i + 990] for i in range(100)), flat[17_000_001: 39_999_997]]
    K.clip_grads(parts, torch.tensor([1.0, 0.5], device="cuda"))
    want = torch.full_like(flat, 2.0)
    for p in parts:
        at = (p.data_ptr() - flat.data_ptr()) // 4
        want[at: at + p.numel()] = 1.0
    assert torch.equal(flat, want)
