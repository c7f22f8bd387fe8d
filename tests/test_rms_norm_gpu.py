"""Normalisation over channels against its formula in 64 bits: forward, backward, and forward into 8 bits.

Half a rounding step is 2^-8 of a bf16 value and 2^-4 of an e4m3 one (2^-10 of the row's scale below its normal numbers). The
fp32 sums before it run over at most C / 32 values one after the other, then over at most 1024 partial ones in pairs or
in groups of up to 32: `_sum_error`."""
import pytest
import torch

from rembrandt_b200.ops import native_ops as K

pytestmark = pytest.mark.gpu
EPS = 1e-5
U = 2.0 ** -24


def _sum_error(n):
    return (n / 32 + 64) * U


def _acts(gen, rows, C, c_valid, std=1.0):
    x = torch.randn((rows, C), generator=gen, device="cuda") * std
    x *= torch.exp(torch.randn((rows, 1), generator=gen, device="cuda"))
    x[:, c_valid:] = 0
    return x.bfloat16()


def _gamma(gen, C, c_valid):
    gamma = 1.0 + 0.3 * torch.randn(C, generator=gen, device="cuda")
    gamma[::7] *= -1.0
    gamma[c_valid:] = 5.0       # whatever stands behind the live channels plays no part
    return gamma


def _formula(h, c_valid, gamma, relu, eps=EPS):
    """(y, factor) in 64 bits."""
    live = torch.arange(h.shape[1], device=h.device) < c_valid
    h = torch.where(live, h.double(), 0.0)
    r = (h.square().sum(1, keepdim=True) / c_valid + eps).rsqrt()
    y = torch.where(live, h * r * gamma.double(), 0.0)
    return torch.relu(y) if relu else y, r[:, 0]


SHAPES = [(1, 8, 8), (1, 8, 1), (3, 32, 16), (361, 128, 128), (37, 96, 80), (1000, 64, 64), (5, 160, 129), (2, 1024, 1000), (7, 1056, 1050),
          (129, 4096, 4096), (2500, 1032, 1030), (1300, 2048, 2048), (33, 2080, 2055), (3, 16384, 16384), (2, 16352, 16350), (9, 768, 741), (2, 8200, 8193), (1, 4104, 4099), (64, 128, 100), (65, 128, 100), (4, 1024, 999), (256, 32, 20), (4099, 32, 32), (700, 512, 500), (20000, 192, 192)]


@pytest.mark.parametrize("rows,C,c_valid", SHAPES)
@pytest.mark.parametrize("residual,train,relu", [(False, False, True), (True, True, False), (True, True, True), (False, True, False)])
def test_forward(rows, C, c_valid, residual, train, relu):
    gen = torch.Generator(device="cuda").manual_seed(rows * C + c_valid)
    x, gamma = _acts(gen, rows, C, c_valid), _gamma(gen, C, c_valid)
    res = _acts(gen, rows, C, c_valid) if residual else None
    y, h = (torch.full((rows + 1, C), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    rstd = torch.full((rows + 1,), 7.0, device="cuda")
    K.rms_norm_fwd(x, rows, C, c_valid, EPS, gamma, y, rstd=rstd if train else None, residual=res, h=h if residual else None, relu=relu)
    total = (x.float() + res.float()).bfloat16() if residual else x
    if residual:
        assert torch.equal(h[:rows], total)
    want, r = _formula(total, c_valid, gamma, relu)
    if train:
        assert ((rstd[:rows] - r).abs() <= _sum_error(C) * r).all()
    assert ((y[:rows].double() - want).abs() <= (2.0 ** -8 + 2 * _sum_error(C)) * want.abs()).all()
    assert (y[:rows, c_valid:] == 0).all()
    # what lies behind the last row stays as it was
    assert y[rows].isnan().all() and h[rows].isnan().all() and rstd[rows] == 7.0


@pytest.mark.parametrize("rows,C,c_valid", SHAPES)
@pytest.mark.parametrize("residual,relu", [(False, True), (True, False)])
def test_forward_into_8_bits(rows, C, c_valid, residual, relu):
    gen = torch.Generator(device="cuda").manual_seed(rows * C + c_valid)
    x, gamma = _acts(gen, rows, C, c_valid), _gamma(gen, C, c_valid)
    if rows > 2:
        x[1] = 0
    res = _acts(gen, rows, C, c_valid) if residual else None
    h = torch.empty_like(x) if residual else None
    q = torch.zeros((rows + 1, C), device="cuda", dtype=torch.float8_e4m3fn)
    scales = torch.full((rows + 1,), 7.0, device="cuda")
    K.rms_norm_fwd_e4m3(x, rows, C, c_valid, EPS, gamma, q, scales, residual=res, h=h, relu=relu)
    total = (x.float() + res.float()).bfloat16() if residual else x
    if residual:
        assert torch.equal(h, total)
    want, _ = _formula(total, c_valid, gamma, relu)
    most = want.abs().amax(1)
    scale = torch.where(most == 0, 1.0, most / 448)
    assert ((scales[:rows] - scale).abs() <= 3 * _sum_error(C) * scale).all()
    got = q[:rows].double() * scales[:rows, None].double()
    off = (got - want).abs()
    assert (off <= (2.0 ** -4 + 8 * _sum_error(C)) * want.abs() + scale[:, None] * 2.0 ** -10 * 1.001).all()
    assert (q[:rows].float().abs().amax(1)[most > 0] == 448).all()
    assert (q[rows].float() == 0).all() and scales[rows] == 7.0


def _backward(h, dy, c_valid, r, gamma, relu, add):
    """By the chain rule in 64 bits, with the size of what was added up for it: (dx, dgamma, sizes of both)."""
    live = torch.arange(h.shape[1], device=h.device) < c_valid
    h, dy, r = torch.where(live, h.double(), 0.0), torch.where(live, dy.double(), 0.0), r.double()[:, None]
    gamma = torch.where(live, gamma.double(), 0.0)
    if relu:
        dy = torch.where(gamma * h > 0, dy, 0.0)
    xhat, gg = h * r, dy * gamma
    dx = r * (gg - xhat * (gg * xhat).sum(1, keepdim=True) / c_valid)
    size = r * (gg.abs() + xhat.abs() * (gg * xhat).abs().sum(1, keepdim=True) / c_valid)
    if add is not None:
        dx, size = dx + torch.where(live, add.double(), 0.0), size + add.double().abs()
    return dx, (dy * xhat).sum(0), size, (dy * xhat).abs().sum(0)


@pytest.mark.parametrize("rows,C,c_valid", SHAPES)
@pytest.mark.parametrize("add,relu", [(False, True), (True, False)])
def test_backward(rows, C, c_valid, add, relu):
    gen = torch.Generator(device="cuda").manual_seed(rows * C + c_valid)
    h, gamma, dy = _acts(gen, rows, C, c_valid), _gamma(gen, C, c_valid), _acts(gen, rows, C, c_valid, 1e-2)
    more = _acts(gen, rows, C, c_valid, 1e-2) if add else None
    rstd = _formula(h, c_valid, gamma, False)[1].float()
    before = torch.randn(C, generator=gen, device="cuda")
    dgamma, dx = before.clone(), torch.full((rows + 1, C), float("nan"), device="cuda", dtype=torch.bfloat16)
    ws = K.rms_norm_scratch(C, "cuda")
    K.rms_norm_bwd(h, dy, rows, C, c_valid, rstd, gamma, dgamma, dx, ws, add=more, relu=relu)
    want, dg, size, dg_size = _backward(h, dy, c_valid, rstd, gamma, relu, more)
    assert ((dx[:rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2 * _sum_error(C) * size).all()
    assert dx[rows].isnan().all()
    # a channel's sum: at most rows / 8 terms one after the other, then what is joined
    assert ((dgamma.double() - before - dg).abs() <= (rows / 8 + 700) * U * dg_size + 2 * U * before.abs()).all()
    assert torch.equal(dgamma[c_valid:], before[c_valid:]) and (dx[:rows, c_valid:] == 0).all()
    # the same sums again, in the same order, with the scratch as the first call has left it
    again, dx2 = before.clone(), torch.empty_like(dx)
    K.rms_norm_bwd(h, dy, rows, C, c_valid, rstd, gamma, again, dx2, ws, add=more, relu=relu)
    assert torch.equal(again, dgamma) and torch.equal(dx2[:rows], dx[:rows])


def test_gradients_are_the_differences_of_the_formula():
    """d(sum of dy * y) along a direction, by central differences of the formula in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    rows, C, c_valid = 6, 64, 50
    h, gamma, dy = _acts(gen, rows, C, c_valid), _gamma(gen, C, c_valid), _acts(gen, rows, C, c_valid)
    rstd = _formula(h, c_valid, gamma, False)[1].float()
    dgamma, dx = torch.zeros(C, device="cuda"), torch.empty_like(h)
    K.rms_norm_bwd(h, dy, rows, C, c_valid, rstd, gamma, dgamma, dx, K.rms_norm_scratch(C, "cuda"))
    live = (torch.arange(C, device="cuda") < c_valid).double()
    step = 1e-6
    for _ in range(8):
        way = torch.randn((rows, C), generator=gen, device="cuda").double() * live
        wayg = torch.randn(C, generator=gen, device="cuda").double() * live
        f = lambda t: (dy.double() * _formula(h.double() + t * way, c_valid, gamma.double() + t * wayg, False)[0]).sum()
        slope = (f(step) - f(-step)) / (2 * step)
        got = (dx.double() * way).sum() + (dgamma.double() * wayg).sum()
        # every value of dx is off by 2^-8 at most; differences of step 1e-6 by about 1e-8 of the values
        assert (got - slope).abs() <= 2.0 ** -8 * (dx.double() * way).abs().sum() + 1e-5 * (dy.double().abs().sum() + 1)


def test_rows_without_anything_and_rows_with_infinities():
    rows, C = 6, 64
    x = torch.ones((rows, C), device="cuda", dtype=torch.bfloat16)
    x[1] = 0
    x[2, 3] = float("inf")
    x[3, 5] = float("nan")
    x[4] = torch.finfo(torch.bfloat16).min
    gamma = torch.full((C,), 2.0, device="cuda")
    y, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
    K.rms_norm_fwd(x, rows, C, C, EPS, gamma, y, rstd=rstd)
    assert (y[1] == 0).all() and torch.equal(y[0], y[5]) and y[0].isfinite().all()
    assert y[2, 3].isnan() and (y[2, :3] == 0).all() and y[3].isnan().all()
    assert (y[4] == 0).all()        # squares of the type's lowest value pass fp32
    z = torch.empty_like(y)
    K.rms_norm_fwd(x, rows, C, C, EPS, gamma, z, relu=True)
    assert z[2, 3].isnan() and z[3].isnan().all() and torch.equal(z[:2], y[:2]) and (z[4] == 0).all()
    q, scales = torch.empty((rows, C), device="cuda", dtype=torch.float8_e4m3fn), torch.empty(rows, device="cuda")
    K.rms_norm_fwd_e4m3(x, rows, C, C, EPS, gamma, q, scales)
    assert scales[1] == 1 and (q[1].float() == 0).all() and (q[0].float() == 448).all()
    for i in (2, 3):
        assert scales[i].isnan() and q[i].float().isnan().all()
    dgamma, dx, dy = torch.zeros(C, device="cuda"), torch.empty_like(x), torch.ones_like(x)
    K.rms_norm_bwd(x[:2], dy, 2, C, C, rstd, gamma, dgamma, dx, K.rms_norm_scratch(C, "cuda"))
    assert dx[:2].isfinite().all() and dgamma.isfinite().all()
    want = 2.0 * rstd[1].double()           # a row of zeros: the slope is gamma / sqrt(eps)
    assert ((dx[1].double() - want).abs() <= (2.0 ** -8 + 4 * U) * want).all()


def test_what_stands_in_dead_channels_plays_no_part():
    gen = torch.Generator(device="cuda").manual_seed(5)
    rows, C, c_valid = 9, 96, 70
    clean = [_acts(gen, rows, C, c_valid) for _ in range(4)]
    dirty = [t.clone() for t in clean]
    for t, bad in zip(dirty, (float("nan"), float("inf"), float("nan"), -1.0)):
        t[:, c_valid:] = bad
    gamma = _gamma(gen, C, c_valid)
    gamma2 = gamma.clone()
    gamma2[c_valid:] = float("nan")
    out = []
    for (x, res, dy, add), g in ((clean, gamma), (dirty, gamma2)):
        y, h, dx, rstd, dg = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda"), torch.zeros(C, device="cuda")
        q, scales = torch.empty((rows, C), device="cuda", dtype=torch.float8_e4m3fn), torch.empty(rows, device="cuda")
        K.rms_norm_fwd_e4m3(x, rows, C, c_valid, EPS, g, q, scales, residual=res)
        K.rms_norm_fwd(x, rows, C, c_valid, EPS, g, y, rstd=rstd, residual=res, h=h, relu=True)
        K.rms_norm_bwd(h, dy, rows, C, c_valid, rstd, g, dg, dx, K.rms_norm_scratch(C, "cuda"), add=add, relu=True)
        out.append((y, h, rstd, q.float(), scales, dx, dg))
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,C", [(50, 64), (9, 4096), (300, 512)])
def test_outputs_over_inputs(rows, C):
    gen = torch.Generator(device="cuda").manual_seed(C)
    x, res, dy, add = (_acts(gen, rows, C, C) for _ in range(4))
    gamma = _gamma(gen, C, C)
    y, h, rstd, dg, dx = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda"), torch.zeros(C, device="cuda"), torch.empty_like(x)
    ws = K.rms_norm_scratch(C, "cuda")
    K.rms_norm_fwd(x, rows, C, C, EPS, gamma, y, rstd=rstd, residual=res, h=h)
    K.rms_norm_bwd(h, dy, rows, C, C, rstd, gamma, dg, dx, ws, add=add)
    for h_at, y_at in ((0, 1), (1, 0), (None, 0), (None, 1), (0, None), (1, None)):
        both = [x.clone(), res.clone()]
        hh = torch.empty_like(x) if h_at is None else both[h_at]
        yy = torch.empty_like(x) if y_at is None else both[y_at]
        K.rms_norm_fwd(both[0], rows, C, C, EPS, gamma, yy, rstd=rstd, residual=both[1], h=hh)
        assert torch.equal(yy, y) and torch.equal(hh, h)
    q, scales = torch.empty((rows, C), device="cuda", dtype=torch.float8_e4m3fn), torch.empty(rows, device="cuda")
    K.rms_norm_fwd_e4m3(x, rows, C, C, EPS, gamma, q, scales, residual=res)
    for h_at in (0, 1):
        both, q2, scales2 = [x.clone(), res.clone()], torch.empty_like(q), torch.empty_like(scales)
        K.rms_norm_fwd_e4m3(both[0], rows, C, C, EPS, gamma, q2, scales2, residual=both[1], h=both[h_at])
        assert torch.equal(both[h_at], h) and torch.equal(both[1 - h_at], (res, x)[h_at])
        assert torch.equal(q2.float(), q.float()) and torch.equal(scales2, scales)
    for over in range(3):
        ins = [h.clone(), dy.clone(), add.clone()]
        dg2 = torch.zeros(C, device="cuda")
        K.rms_norm_bwd(ins[0], ins[1], rows, C, C, rstd, gamma, dg2, ins[over], ws, add=ins[2])
        assert torch.equal(ins[over], dx) and torch.equal(dg2, dg)


def test_no_rows():
    x = torch.ones((1, 64), device="cuda", dtype=torch.bfloat16)
    gamma, dgamma = torch.ones(64, device="cuda"), torch.full((64,), 3.0, device="cuda")
    y, q = torch.full_like(x, 5.0), torch.ones((1, 64), device="cuda").to(torch.float8_e4m3fn)
    rstd = torch.full((1,), 5.0, device="cuda")
    K.rms_norm_fwd(x, 0, 64, 64, EPS, gamma, y, rstd=rstd)
    K.rms_norm_fwd_e4m3(x, 0, 64, 64, EPS, gamma, q, rstd)
    K.rms_norm_bwd(x, x, 0, 64, 64, rstd, gamma, dgamma, y, K.rms_norm_scratch(64, "cuda"))
    assert (y == 5).all() and rstd[0] == 5 and (dgamma == 3).all() and (q.float() == 1).all()
    none, no_rows = x[:0].clone(), rstd[:0].clone()
    K.rms_norm_fwd(none, 0, 64, 64, EPS, gamma, none.clone(), rstd=no_rows, residual=none.clone(), h=none.clone())
    K.rms_norm_fwd_e4m3(none, 0, 64, 64, EPS, gamma, none.to(torch.float8_e4m3fn), no_rows, residual=none.clone(), h=none.clone())
    K.rms_norm_bwd(none, none, 0, 64, 64, no_rows, gamma, dgamma, none.clone(), K.rms_norm_scratch(64, "cuda"), add=none)
    assert (dgamma == 3).all()


def test_two_graphs_with_their_own_scratch_run_at_the_same_time():
    gen = torch.Generator(device="cuda").manual_seed(12)
    rows, C = 30_000, 128
    h, dy, gamma = _acts(gen, rows, C, C), _acts(gen, rows, C, C), _gamma(gen, C, C)
    rstd = _formula(h, C, gamma, False)[1].float()
    graphs = []
    for scale in (1.0, 2.0):
        dg, dx, ws, d = torch.zeros(C, device="cuda"), torch.empty_like(h), K.rms_norm_scratch(C, "cuda"), dy * scale
        g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            dg.zero_()
            for _ in range(10):
                K.rms_norm_bwd(h, d, rows, C, C, rstd, gamma, dg, dx, ws)
        graphs.append((g, stream, dg, dx, d, ws))
    for _ in range(5):
        for g, stream, *_rest in graphs:
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    # deltas twice as large: every product and sum is twice as large, exactly
    assert torch.equal(graphs[1][2], 2 * graphs[0][2]) and torch.equal(graphs[1][3], 2 * graphs[0][3])
    assert graphs[0][2].abs().sum() > 0


def test_another_stream_and_a_captured_call():
    gen = torch.Generator(device="cuda").manual_seed(11)
    rows, C = 777, 256
    x, dy, gamma = _acts(gen, rows, C, C), _acts(gen, rows, C, C), _gamma(gen, C, C)
    want = None
    for how in ("here", "stream", "graph"):
        y, rstd, dx, dg, ws = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty_like(x), torch.zeros(C, device="cuda"), K.rms_norm_scratch(C, "cuda")

        def go():
            K.rms_norm_fwd(x, rows, C, C, EPS, gamma, y, rstd=rstd, relu=True)
            K.rms_norm_bwd(x, dy, rows, C, C, rstd, gamma, dg, dx, ws, relu=True)

        torch.cuda.synchronize()
        if how == "here":
            go()
        elif how == "stream":
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                go()
            s.synchronize()
        else:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                go()
            g.replay()
            torch.cuda.synchronize()
            first = dg.clone()
            g.replay()
            torch.cuda.synchronize()
            # half a step of each of two additions
            assert ((dg - 2 * first).abs() <= 4 * U * first.abs()).all()
            dg = first
        got = (y, rstd, dx, dg)
        if want is None:
            want = got
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_more_than_two_to_the_31_values():
    rows, C = 131080, 16384
    x = torch.zeros((rows, C), device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(1)
    gamma, rstd = _gamma(gen, C, C), torch.empty(rows, device="cuda")
    last = _acts(gen, 4, C, C)
    x[-4:] = last
    y = torch.empty_like(x)
    K.rms_norm_fwd(x, rows, C, C, EPS, gamma, y, rstd=rstd)
    want, _ = _formula(last, C, gamma, False)
    assert ((y[-4:].double() - want).abs() <= (2.0 ** -8 + 2 * _sum_error(C)) * want.abs()).all() and (y[:131072] == 0).all()
    dg = torch.zeros(C, device="cuda")
    K.rms_norm_bwd(x, x, rows, C, C, rstd, gamma, dg, y, K.rms_norm_scratch(C, "cuda"))
    dx, dgw, size, dg_size = _backward(last, last, C, rstd[-4:], gamma, False, None)
    assert ((y[-4:].double() - dx).abs() <= 2.0 ** -8 * dx.abs() + 2 * _sum_error(C) * size).all()
    assert ((dg - dgw).abs() <= (rows / 8 + 700) * U * dg_size).all()
