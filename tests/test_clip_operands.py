"""Operands that the gradient norm, clipping, the clipped update and the normalisation over channels refuse before anything is
launched (no GPU: a launch of the stand-in library fails the test)."""
import pytest
import torch

from rembrandt_b200 import _native
from rembrandt_b200.ops import native_ops as K


@pytest.fixture
def no_launch(monkeypatch):
    class Library:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")
    monkeypatch.setattr(_native, "cuda", Library)


@pytest.fixture
def as_on_a_gpu(monkeypatch, no_launch):
    """Everything on the CPU passes for what is on the current device."""
    class Launched(Exception):
        pass

    class Library:
        def __getattr__(self, name):
            raise Launched
    monkeypatch.setattr(_native, "cuda", Library)
    monkeypatch.setattr(K, "_stream_of", lambda names, *tensors: 0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    return Launched


def _sweep(clip, n=64, **change):
    t = {"w": torch.zeros(n), "g": torch.zeros(n), "v": torch.zeros(n), "w16": torch.zeros(n, dtype=torch.bfloat16)} | change
    K.sgd_fused(t["w"], t["g"], t["v"], t["w16"], n, 0.1, 0.9, 0.0, 1.0, 1, clip=clip)


@pytest.mark.parametrize("change", [{}, {"v": None}, {"w16": None}])
def test_a_coefficient_that_is_not_on_the_gpu(no_launch, change):
    with pytest.raises(ValueError, match="clip has to be on a GPU"):
        _sweep(torch.zeros(2), **change)


# ---- small operands inside of others: what a launch would read while it writes there
ROWS, C = 8, 64


def _floats(n):
    """A float32 view of the last `n` floats of a 16-byte aligned buffer of `dtype`, which is larger than that."""
    return lambda t: t.view(torch.uint8).reshape(-1)[-4 * n:].view(torch.float32)


def _norm_operands():
    bf = lambda: torch.zeros((ROWS, C), dtype=torch.bfloat16)
    return {"x": bf(), "residual": bf(), "h": bf(), "y": bf(), "dy": bf(), "dx": bf(), "add": bf(), "rstd": torch.zeros(ROWS),
            "gamma": torch.ones(C), "dgamma": torch.zeros(C), "q": torch.zeros((ROWS, C), dtype=torch.float8_e4m3fn),
            "scales": torch.zeros(ROWS), "scratch": K.rms_norm_scratch(C, "cpu")}


def _fwd(o):
    K.rms_norm_fwd(o["x"], ROWS, C, C, 1e-5, o["gamma"], o["y"], rstd=o["rstd"], residual=o["residual"], h=o["h"])


def _fwd8(o):
    K.rms_norm_fwd_e4m3(o["x"], ROWS, C, C, 1e-5, o["gamma"], o["q"], o["scales"], residual=o["residual"], h=o["h"])


def _bwd(o):
    K.rms_norm_bwd(o["h"], o["dy"], ROWS, C, C, o["rstd"], o["gamma"], o["dgamma"], o["dx"], o["scratch"], add=o["add"])


READ = {_fwd: ["x", "residual", "gamma"], _fwd8: ["x", "residual", "gamma"], _bwd: ["h", "dy", "add", "rstd", "gamma"]}
WRITTEN = {_fwd: ["y", "h", "rstd"], _fwd8: ["q", "h", "scales"], _bwd: ["dx", "dgamma", "scratch"]}


@pytest.mark.parametrize("call,small,large", [
    (call, small, large) for call in (_fwd, _fwd8, _bwd) for small in ("rstd", "scales", "gamma", "dgamma") for large in READ[call] + WRITTEN[call]
    if small in READ[call] + WRITTEN[call] and small != large and {small, large} & set(WRITTEN[call])])
def test_small_operands_inside_of_others(as_on_a_gpu, call, small, large):
    o = _norm_operands()
    with pytest.raises(as_on_a_gpu):         # apart
        call(o)
    n = o[small].numel()
    if o[large].numel() * o[large].element_size() > 4 * n:
        inside = _floats(n)(o[large])
    else:                                    # the other way round: the larger one's operand begins in the smaller one
        room = torch.zeros(o[small].numel() + 4 + o[large].numel())
        inside, o[large] = room[:n], room[n - 4: n - 4 + o[large].numel()]
    with pytest.raises(ValueError, match="overlaps"):
        call(o | {small: inside})


def test_outputs_exactly_over_inputs_and_next_to_them(as_on_a_gpu):
    o = _norm_operands()
    for call, places in ((_fwd, [("y", "x"), ("y", "residual"), ("h", "x"), ("h", "residual")]), (_fwd8, [("h", "x"), ("h", "residual")]),
                         (_bwd, [("dx", "h"), ("dx", "dy"), ("dx", "add")])):
        for out, over in places:
            with pytest.raises(as_on_a_gpu):
                call(o | {out: o[over]})
    # inputs may overlap one another in any way
    flat = torch.zeros(2 * ROWS * C, dtype=torch.bfloat16)
    one, two = flat[: ROWS * C].view(ROWS, C), flat[8: 8 + ROWS * C].view(ROWS, C)
    for call, both in ((_fwd, ("x", "residual")), (_fwd8, ("x", "residual")), (_bwd, ("dy", "add")), (_bwd, ("h", "dy"))):
        with pytest.raises(as_on_a_gpu):
            call(o | dict(zip(both, (one, two))))
        with pytest.raises(as_on_a_gpu):
            call(o | dict(zip(both, (one, one))))
    # an output in the place of one of them meets the other
    with pytest.raises(ValueError, match="y overlaps residual"):
        _fwd(o | {"x": one, "residual": two, "y": one})
    with pytest.raises(ValueError, match="y overlaps h"):
        _fwd(o | {"x": one, "y": one, "h": one})
    # one after the other in one buffer
    flat = torch.zeros(5 * ROWS * C, dtype=torch.bfloat16)
    parts = iter(flat.view(5, ROWS, C))
    with pytest.raises(as_on_a_gpu):
        _fwd(o | {name: next(parts) for name in ("x", "y", "h", "residual")} | {"rstd": next(parts).view(-1)[: 2 * ROWS].view(torch.float32)})


def test_norm_and_coefficient_inside_of_gradients_or_scratch(as_on_a_gpu):
    flat, ws, out = torch.zeros(1000), K.grad_norm_scratch("cpu"), torch.zeros(2)
    grads = K.grad_list([flat[700:900], flat[10:500], flat[600:600], torch.zeros(7, dtype=torch.float16)])
    for at in (10, 11, 498, 700, 898, 9, 499, 899):
        with pytest.raises(ValueError, match="out overlaps a gradient"):
            K.grad_norm(grads, 1.0, flat[at: at + 2], ws)
        with pytest.raises(ValueError, match="out overlaps a gradient"):
            K.clip_grads(grads, flat[at: at + 2])
    for at in (0, 8, 500, 600, 698, 900, 998):
        for call in (lambda o: K.grad_norm(grads, 1.0, o, ws), lambda o: K.clip_grads(grads, o)):
            with pytest.raises(as_on_a_gpu):
                call(flat[at: at + 2])
    for at in (0, 500, 1478):
        with pytest.raises(ValueError, match="out overlaps scratch"):
            K.grad_norm(grads, 1.0, ws.view(torch.float32)[at: at + 2], ws)
    with pytest.raises(ValueError, match="scratch overlaps a gradient"):
        K.grad_norm([ws.view(torch.float32)[1479:]], 1.0, out, ws)
    for empty in ([], [flat[:0]]):
        with pytest.raises(as_on_a_gpu):
            K.grad_norm(empty, 1.0, out, ws)


@pytest.mark.parametrize("where", ["w", "g", "v", "w16"])
def test_a_coefficient_inside_of_what_the_sweep_writes(as_on_a_gpu, where):
    t = torch.zeros(64, dtype=torch.bfloat16 if where == "w16" else torch.float32)
    floats = t.view(torch.float32)
    with pytest.raises(ValueError, match="clip overlaps"):
        _sweep(floats[-2:], **{where: t})
    with pytest.raises(as_on_a_gpu):
        _sweep(torch.zeros(2), **{where: t})
    with pytest.raises(as_on_a_gpu):          # behind what the sweep takes of it
        _sweep(floats[-2:], n=64 - 4, **{where: t})


@pytest.mark.parametrize("scale", [2.0 ** 128 - 2.0 ** 103, 2.0 ** 128 * (1 - 2.0 ** -30)])
def test_scales_that_round_to_infinity(no_launch, scale):
    assert torch.tensor(scale, dtype=torch.float32).isinf()
    with pytest.raises(ValueError, match="scale"):
        K.grad_norm([], 1.0, torch.zeros(2), K.grad_norm_scratch("cpu"), scale=scale)
    with pytest.raises(ValueError, match="scale"):
        K.clip_grads([], torch.zeros(2), scale=scale)


@pytest.mark.parametrize("scale", [2.0 ** 128 - 2.0 ** 104, 2.0 ** -126])
def test_the_largest_and_smallest_scale(as_on_a_gpu, scale):
    with pytest.raises(as_on_a_gpu):
        K.grad_norm([], 1.0, torch.zeros(2), K.grad_norm_scratch("cpu"), scale=scale)
    with pytest.raises(as_on_a_gpu):
        K.clip_grads([], torch.zeros(2), scale=scale)
