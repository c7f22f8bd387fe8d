"""Arguments that the normalisation over channels and the gradient norm refuse, before anything is launched (no GPU)."""
import pytest
import torch

from rembrandt_b200.ops import native_ops as K


def _good(rows=4, C=64):
    bf = lambda: torch.zeros((rows, C), dtype=torch.bfloat16)
    return {"x": bf(), "residual": bf(), "h": bf(), "y": bf(), "dy": bf(), "dx": bf(), "add": bf(), "rstd": torch.zeros(rows), "gamma": torch.ones(C),
            "dgamma": torch.zeros(C), "q": torch.zeros((rows, C), dtype=torch.float8_e4m3fn), "scales": torch.zeros(rows),
            "ws": K.rms_norm_scratch(C, "cpu"), "rows": rows, "C": C, "valid": C, "eps": 1e-5}


def _fwd(a):
    K.rms_norm_fwd(a["x"], a["rows"], a["C"], a["valid"], a["eps"], a["gamma"], a["y"], rstd=a["rstd"], residual=a["residual"], h=a["h"])


def _fwd8(a):
    K.rms_norm_fwd_e4m3(a["x"], a["rows"], a["C"], a["valid"], a["eps"], a["gamma"], a["q"], a["scales"], residual=a["residual"], h=a["h"])


def _bwd(a):
    K.rms_norm_bwd(a["x"], a["dy"], a["rows"], a["C"], a["valid"], a["rstd"], a["gamma"], a["dgamma"], a["dx"], a["ws"], add=a["add"])


OPERANDS = {_fwd: ["x", "residual", "h", "y", "gamma", "rstd"], _fwd8: ["x", "residual", "h", "q", "gamma", "scales"],
            _bwd: ["x", "dy", "add", "dx", "rstd", "gamma", "dgamma", "ws"]}


@pytest.mark.parametrize("call", list(OPERANDS))
def test_operands(call):
    with pytest.raises(ValueError, match="GPU"):        # everything else is in order
        call(_good())
    for name in OPERANDS[call]:
        good = _good()[name]
        flat = torch.zeros(good.numel() + 32, dtype=torch.float32).to(good.dtype)
        wrong = [good.to(torch.float16), good.flatten()[:-1], None if name not in ("residual", "h", "add", "rstd") else "text"]
        if good.dim() == 2:
            wrong += [torch.zeros((64, 4), dtype=torch.float32).to(good.dtype).t(), flat[1: 1 + good.numel()]]
        for bad in wrong:
            if bad is None and call is _fwd and name == "rstd":
                continue
            with pytest.raises(ValueError):
                try:
                    call(_good() | {name: bad})
                except ValueError as e:
                    assert "GPU" not in str(e), (name, bad)
                    raise


@pytest.mark.parametrize("call", list(OPERANDS))
def test_shapes(call):
    for change in ({"C": 60}, {"C": 0}, {"C": 4}, {"C": 16392}, {"rows": -1}, {"valid": 0}, {"valid": 65}, {"rows": 5}, {"rows": 1 << 40}):
        with pytest.raises(ValueError):
            try:
                call(_good() | change)
            except ValueError as e:
                assert "GPU" not in str(e), change
                raise


@pytest.mark.parametrize("call", [_fwd, _fwd8])
@pytest.mark.parametrize("eps", [0.0, -1e-5, float("nan"), float("inf"), 1e-40, 1e39])
def test_epsilons(call, eps):
    with pytest.raises(ValueError, match="epsilon"):
        call(_good() | {"eps": eps})


def test_overlaps():
    a = _good()
    with pytest.raises(ValueError, match="y overlaps h"):
        _fwd(a | {"y": a["h"]})
    flat = torch.zeros(12 * 64, dtype=torch.bfloat16)
    part = lambda i: flat[i * 64: (i + 4) * 64].view(4, 64)
    with pytest.raises(ValueError, match="h overlaps x"):
        _fwd(a | {"x": part(0), "h": part(2)})
    with pytest.raises(ValueError, match="y overlaps residual"):
        _fwd(a | {"residual": part(3), "y": part(0)})
    with pytest.raises(ValueError, match="dx overlaps dy"):
        _bwd(a | {"dx": part(3), "dy": part(0)})
    with pytest.raises(ValueError, match="q overlaps x"):
        _fwd8(a | {"x": part(0), "q": flat[:128].view(torch.float8_e4m3fn).view(4, 64)})
    for same in ({"x": part(0), "h": part(0)}, {"residual": part(0), "h": part(0), "x": part(4), "y": part(4)}):
        with pytest.raises(ValueError, match="GPU"):
            _fwd(a | same)


def test_a_scratch_serves_fewer_channels():
    sizes = {C: K.rms_norm_scratch(C, "cpu").numel() for C in (8, 1024, 1032, 2048, 2056, 4096, 16384)}
    assert list(sizes.values()) == sorted(sizes.values()) and all(n >= 592 * C for C, n in sizes.items())
    a = _good(2, 2048)
    for C, enough in ((1024, False), (2048, True), (2056, True), (4096, True)):
        with pytest.raises(ValueError, match="GPU" if enough else "scratch"):
            _bwd(a | {"ws": K.rms_norm_scratch(C, "cpu")})


def test_gradients():
    for bad in (torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int32), None, 3.0):
        with pytest.raises(ValueError, match="gradient 0"):
            K.grad_list([bad])
    with pytest.raises(ValueError, match="gaps"):
        K.grad_list([torch.zeros(8, 8)[:, :4]])
    with pytest.raises(ValueError, match="gaps"):
        K.grad_list([torch.zeros(1).expand(8)])
    with pytest.raises(ValueError, match="GPU"):
        K.grad_list([torch.zeros(4)])
    with pytest.raises(ValueError, match="GPU"):
        K.grad_norm([], 1.0, torch.zeros(2), K.grad_norm_scratch("cpu"))
