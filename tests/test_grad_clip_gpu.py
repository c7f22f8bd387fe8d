"""The gradients' global norm, clipping by it, and the clipped update, against their formulas in 64 bits.

A norm is rounded to fp32 once (2^-24); groups of at most eight squares may be added in fp32 before that (8 x 2^-24 of their sum,
half of it in the root). The factor of a gradient has that error and two more roundings."""
import math

import pytest
import torch

from rembrandt_b200.ops import native_ops as K
from rembrandt_b200.optim.sgd import reference_step

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NORM = 6 * U
FACTOR = NORM + 3 * U
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _norm(tensors, scale=1.0):
    return scale * math.sqrt(sum(t.double().square().sum().item() for t in tensors))


def _call(tensors, max_norm, scale=1.0):
    out, ws = torch.full((2,), 9.0, device="cuda"), K.grad_norm_scratch("cuda")
    K.grad_norm(tensors, max_norm, out, ws, scale=scale)
    return out


def _lists():
    gen = torch.Generator(device="cuda").manual_seed(0)
    make = lambda n, t, std=1.0: (torch.randn(n, generator=gen, device="cuda") * std).to(t)
    yield "one value", [make(1, torch.float32)]
    yield "each type", [make(n, t) for t in TYPES for n in (1, 7, 8, 9, 4095, 4096, 4097, 100_003)]
    yield "none and empty ones", [make(0, torch.float32), make(5, torch.bfloat16), make(0, torch.float16)]
    yield "many small ones", [make(n % 300 + 1, TYPES[n % 3]) for n in range(1000)]
    yield "more than one table holds", [make(n % 37 if n % 9 else 0, TYPES[n % 3]) for n in range(4000)]
    yield "one large one", [make(9_999_991, torch.float32)]
    yield "large ones of 16 bits", [make(3_000_001, torch.bfloat16), make(2_000_003, torch.float16)]
    flat = make(50_000, torch.float32)
    yield "off the boundaries", [flat[1:2], flat[3:8], flat[9:40_000], flat[40_001:40_003], flat[40_003:]]
    half = make(50_000, torch.bfloat16)
    yield "off the boundaries in 16 bits", [half[1:2], half[3:8], half[9:30_000], half[30_003:]]
    yield "other orders", [make(64 * 48, torch.float32).view(64, 48).t(), make(24 * 12, torch.float32).view(2, 3, 6, 8).permute(0, 3, 1, 2)]


@pytest.mark.parametrize("i", range(10))
@pytest.mark.parametrize("scale,share", [(1.0, 0.37), (0.125, 1.0 + 1e-3), (4.0, 0.9)])
def test_norm_and_clipping(i, scale, share):
    name, tensors = list(_lists())[i]
    before = [t.clone() for t in tensors]
    norm = _norm(tensors, scale)
    out = _call(tensors, share * norm, scale)
    got, coef = out.tolist()
    assert abs(got - norm) <= NORM * norm, name
    assert abs(coef - min(1.0, share)) <= FACTOR * share
    for a, b in zip(tensors, before):
        assert torch.equal(a, b)
    K.clip_grads(tensors, out, scale=scale)
    for t, b in zip(tensors, before):
        want = b.double() * (scale * min(1.0, share))
        half_step = max(U, torch.finfo(t.dtype).eps / 2)
        smallest = torch.finfo(t.dtype).smallest_normal * torch.finfo(t.dtype).eps / 2
        assert ((t.double() - want).abs() <= (half_step + FACTOR) * want.abs() + smallest * 1.001).all(), name


def test_what_lies_between_the_tensors_stays():
    flat = torch.arange(1.0, 10_001.0, device="cuda")
    keep = flat.clone()
    parts = [flat[3:4], flat[7:4099], flat[5000:9999]]
    K.clip_grads(parts, _call(parts, 1.0))
    inside = torch.zeros(10_000, dtype=torch.bool, device="cuda")
    for lo, hi in ((3, 4), (7, 4099), (5000, 9999)):
        inside[lo:hi] = True
    assert torch.equal(flat[~inside], keep[~inside]) and (flat[inside] < keep[inside]).all()


@pytest.mark.parametrize("value", [1e-30, 1e-22, 1e25, 3e37])
def test_squares_neither_overflow_nor_vanish(value):
    t = [torch.full((5,), value, device="cuda"), torch.zeros(1000, device="cuda"), torch.full((11,), -value, device="cuda").bfloat16()]
    norm = _norm(t)
    got, coef = _call(t, norm / 2).tolist()
    assert abs(got - norm) <= NORM * norm and abs(coef - 0.5) <= FACTOR


@pytest.mark.parametrize("dtype", TYPES)
def test_denormal_values(dtype):
    tiny = torch.finfo(dtype).smallest_normal
    t = torch.full((4097,), tiny / 4, device="cuda", dtype=dtype)
    assert (t != 0).all()
    norm = _norm([t])
    assert abs(_call([t], 1.0)[0].item() - norm) <= NORM * norm + 2.0 ** -149


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", [0, 4096, 8191, 12_345])
def test_a_norm_that_is_not_finite_leaves_zeros(bad, dtype, at):
    good, t = torch.ones(100, device="cuda"), torch.ones(12_346, device="cuda", dtype=dtype)
    t[at] = bad
    out = _call([good, t], 1.0)
    assert not out[0].isfinite() and out[0].isnan() == math.isnan(bad) and out[1] == 0
    K.clip_grads([good, t], out)
    assert (good == 0).all() and (t == 0).all()


def test_gradients_of_zeros_and_no_gradients():
    zeros = torch.zeros(10_000, device="cuda")
    assert _call([zeros], 1e-3).tolist() == [0.0, 1.0]
    assert _call([], 1.0).tolist() == [0.0, 1.0]
    assert _call([zeros[:0]], 1.0).tolist() == [0.0, 1.0]
    K.clip_grads([], _call([], 1.0))


def test_a_norm_within_the_bound_leaves_the_bits():
    t = torch.randn(5000, device="cuda").bfloat16()
    before = t.clone()
    out = _call([t], float("inf"))
    assert out[1] == 1
    K.clip_grads([t], out)
    assert torch.equal(t, before)


def test_the_same_norm_every_time_and_with_a_used_scratch():
    gen = torch.Generator(device="cuda").manual_seed(4)
    many = K.grad_list([torch.randn(n, generator=gen, device="cuda") for n in (3, 1_000_000, 77, 500_001)] * 1)
    few = K.grad_list([torch.ones(10, device="cuda")])
    out, ws = torch.zeros(2, device="cuda"), K.grad_norm_scratch("cuda")
    seen = set()
    for _ in range(5):
        K.grad_norm(many, 1.0, out, ws)
        seen.add(out[0].item())
        K.grad_norm(few, 1.0, out, ws)
        assert abs(out[0].item() - math.sqrt(10)) <= NORM * math.sqrt(10)
    assert len(seen) == 1


@pytest.mark.parametrize("n", [300_000, 20_000])      # several launches, and one
def test_another_stream_and_a_captured_call(n):
    t = [torch.randn(n, device="cuda"), torch.randn(301, device="cuda").half()]
    first = [x.clone() for x in t]
    want = _norm(t)
    many, out, ws = K.grad_list(t), torch.zeros(2, device="cuda"), K.grad_norm_scratch("cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        K.grad_norm(many, want / 4, out, ws)
    s.synchronize()
    assert abs(out[0].item() - want) <= NORM * want
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.grad_norm(many, want / 4, out, ws)
        K.clip_grads(many, out)
    for k in (1.0, 3.0):
        for x, f in zip(t, first):
            x.copy_(f * k)
        g.replay()
        assert abs(out[0].item() - k * want) <= (NORM + 2.0 ** -11) * k * want
        assert abs(_norm(t) - want / 4) <= 2.0 ** -11 * want


def test_more_than_two_to_the_31_values():
    n = 2 ** 31 + 4097
    t = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    t[-1], t[0], t[2 ** 31 - 1], t[2 ** 31] = 3.0, 4.0, 12.0, 84.0
    out = _call([t], 42.5)
    assert out.tolist() == [85.0, 0.5]
    K.clip_grads([t], out)
    assert [t[i].item() for i in (-1, 0, 2 ** 31 - 1, 2 ** 31)] == [1.5, 2.0, 6.0, 42.0]
    assert _call([t], 100.0).tolist() == [42.5, 1.0]


@pytest.mark.parametrize("mode", range(6))
@pytest.mark.parametrize("n", [1, 1025, 300_000, 4_194_311])
def test_clipped_update(mode, n):
    gen = torch.Generator(device="cuda").manual_seed(n + mode)
    w, g, v = (torch.randn(n, generator=gen, device="cuda") for _ in range(3))
    w16 = torch.empty(n, device="cuda", dtype=torch.bfloat16)
    norm = _norm([g], 0.5)
    out, ws = torch.zeros(2, device="cuda"), K.grad_norm_scratch("cuda")
    K.grad_norm([g], norm / 4, out, ws, scale=0.5)
    ref = reference_step(w.double(), g.double(), v.double(), 0.1, 0.9, 5e-4, 0.5 * 0.25, mode)
    big = 1.0 + max(t.abs().max().item() for t in (w, g, v))
    K.sgd_fused(w, g, v, w16, n, 0.1, 0.9, 5e-4, 0.5, mode, clip=out)
    for got, want in zip((w, g, v), ref):
        # at most eight operations on values below 2 * big, and the coefficient's error
        assert ((got.double() - want).abs() <= (16 * U + FACTOR) * 2 * big).all()
    assert torch.equal(w16, w.bfloat16())


def test_an_update_whose_gradients_are_not_finite_is_one_with_zeros():
    n = 1027
    w, v = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    g = torch.randn(n, device="cuda")
    g[5], g[-1] = float("inf"), float("nan")
    w16 = torch.empty(n, device="cuda", dtype=torch.bfloat16)
    out = _call([g], 1.0)
    ref = reference_step(w.clone(), torch.zeros_like(g), v.clone(), 0.1, 0.9, 5e-4, 1.0, 1)
    K.sgd_fused(w, g, v, w16, n, 0.1, 0.9, 5e-4, 1.0, 1, clip=out)
    for got, want in zip((w, g, v), ref):
        assert (got - want).abs().max() < 1e-5


def test_refusals_that_need_a_device():
    t, cpu = torch.ones(10, device="cuda"), torch.ones(10)
    out, ws = torch.zeros(2, device="cuda"), K.grad_norm_scratch("cuda")
    with pytest.raises(ValueError, match="overlap"):
        K.grad_list([t, t])
    with pytest.raises(ValueError, match="overlap"):
        K.grad_list([t[:6], torch.ones(3, device="cuda"), t[5:]])
    with pytest.raises(ValueError, match="gradient 1"):
        K.grad_list([t, cpu])
    with pytest.raises(ValueError, match="out"):
        K.grad_norm([t], 1.0, torch.zeros(2), ws)
    with pytest.raises(ValueError, match="scratch"):
        K.grad_norm([t], 1.0, out, ws[1:])
    for bound in (0.0, -1.0, float("nan"), 1e-60):
        with pytest.raises(ValueError, match="norm"):
            K.grad_norm([t], bound, out, ws)
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-60, 1e39):
        with pytest.raises(ValueError, match="scale"):
            K.grad_norm([t], 1.0, out, ws, scale=scale)
        with pytest.raises(ValueError, match="scale"):
            K.clip_grads([t], out, scale=scale)
    with pytest.raises(ValueError, match="clip"):
        K.sgd_fused(t, t, t, None, 10, 0.1, 0.9, 0.0, 1.0, 1, clip=out[:1])
    assert (t == 1).all()
