"""Networks normalised over channels, and clipped training, without a GPU: the operators' device path with stand-ins of the kernel
fronts against the reference path, parameters in and out, and the step engine's clipping in every synchronisation order."""
import math

import pytest
import torch

import kernel_emulation
from rembrandt_b200.cli import train_gogod
from rembrandt_b200.engine import StepEngine
from rembrandt_b200.models import config as C
from rembrandt_b200.models import zoo
from rembrandt_b200.models.config import (Act, AffineCfg, Conv2dCfg, Data3dCfg, ParamsInit, Pool2dCfg, PoolKind, RmsConv2dCfg,
                                          RmsNormCfg, RmsStackResConv2dCfg, SequentialOperatorConfig, SoftmaxKLLossCfg)
from rembrandt_b200.models.net import Net
from rembrandt_b200.ops import native_ops as K
from rembrandt_b200.optim.sgd import Momentum, SgdOptConfig, StepSizeSchedule, SyncOrder, clip_coefficient, reference_step
from rembrandt_b200.optim.stepper import SgdStepper
from rembrandt_b200.parallel.comm import LocalOverlapComm, NullComm

K_, X_ = ParamsInit.kaiming(), ParamsInit.xavier()


# ---- stand-ins of the kernel fronts
def _rows(t, rows, C_):
    return t.reshape(-1)[: rows * C_].view(rows, C_)


def _live(t, rows, C_, valid):
    out = _rows(t, rows, C_).float().clone()
    out[:, valid:] = 0
    return out


def _fwd(x, rows, C_, valid, eps, gamma, y, rstd=None, residual=None, h=None, relu=False):
    s = _live(x, rows, C_, valid)
    if residual is not None:
        s = (s + _live(residual, rows, C_, valid)).bfloat16().float()
    r = (s.square().sum(1, keepdim=True) / valid + eps).rsqrt()
    out = s * r * gamma[:C_]
    out[:, valid:] = 0
    _rows(y, rows, C_).copy_(out.clamp_min(0) if relu else out)
    if h is not None:
        _rows(h, rows, C_).copy_(s)
    if rstd is not None:
        rstd[:rows] = r[:, 0]


def _bwd(h, dy, rows, C_, valid, rstd, gamma, dgamma, dx, ws, add=None, relu=False):
    assert ws.numel() >= K.RMS_SCRATCH_ROWS * C_
    xhat, g = _live(h, rows, C_, valid) * rstd[:rows, None], _live(dy, rows, C_, valid)
    if relu:
        g = g * (xhat * gamma[:C_] > 0)
    dgamma[:valid] += (g * xhat).sum(0)[:valid]
    g = g * gamma[:C_]
    d = rstd[:rows, None] * (g - xhat * (g * xhat).sum(1, keepdim=True) / valid)
    d[:, valid:] = 0
    _rows(dx, rows, C_).copy_(d if add is None else d + _live(add, rows, C_, valid))


def _norm(tensors, max_norm, out, ws, scale=1.0):
    norm = scale * math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
    out[0], out[1] = norm, clip_coefficient(norm, max_norm)


def _sweep(w, g, v, w16, n, lr, mu, l2, grad_scale, mode, phase=7, clip=None):
    coef = 1.0 if clip is None else float(clip[1])
    if coef == 0.0:
        g[:n].zero_()
    kernel_emulation.sgd_fused(w, g, v, w16, n, lr, mu, l2, grad_scale * coef, mode, phase)


def _install(monkeypatch):
    kernel_emulation.install(monkeypatch)
    for name, fn in {"rms_norm_fwd": _fwd, "rms_norm_bwd": _bwd, "rms_norm_scratch": lambda C_, device: torch.zeros(K.RMS_SCRATCH_ROWS * C_), "grad_norm": _norm,
                     "grad_list": list, "grad_norm_scratch": lambda device: None, "sgd_fused": _sweep}.items():
        monkeypatch.setattr(K, name, fn)


def _head(cfg, classes=10):
    return cfg.affine(AffineCfg(classes, Act.IDENTITY, X_), "out").softmax_kl_loss(SoftmaxKLLossCfg(classes))


def blocks():
    cfg = SequentialOperatorConfig().data3d(Data3dCfg((12, 12, 3), normalize=True))
    cfg.rms_conv2d(RmsConv2dCfg(3, 1, 1, 16, Act.RECT, K_), "stem")
    cfg.rms_stack_res_conv2d(RmsStackResConv2dCfg(K_), "res1")
    cfg.rms_conv2d(RmsConv2dCfg(3, 2, 1, 40, Act.RECT, K_), "down")
    cfg.rms_stack_res_conv2d(RmsStackResConv2dCfg(K_), "res2")
    cfg.rms_conv2d(RmsConv2dCfg(3, 1, 1, 24, Act.TANH, K_), "smooth")
    cfg.pool2d(Pool2dCfg(6, 1, 0, PoolKind.AVERAGE), "gap")
    return _head(cfg)


def stem():
    """A 7 x 7 stride-2 pad-3 first layer on 3 channels: the input arrives space-to-depth'd."""
    cfg = SequentialOperatorConfig().data3d(Data3dCfg((22, 22, 3), normalize=True))
    cfg.rms_conv2d(RmsConv2dCfg(7, 2, 3, 16, Act.RECT, K_), "stem")
    cfg.pool2d(Pool2dCfg(3, 2, 1, PoolKind.MAX), "pool1")
    cfg.rms_stack_res_conv2d(RmsStackResConv2dCfg(K_), "res1")
    cfg.pool2d(Pool2dCfg(6, 1, 0, PoolKind.AVERAGE), "gap")
    return _head(cfg)


def alone():
    """The normalisation by itself: behind a convolution with and without ReLU, and behind an affine layer."""
    cfg = SequentialOperatorConfig().data3d(Data3dCfg((10, 10, 3), normalize=True))
    cfg.conv2d(Conv2dCfg(3, 1, 1, 24, Act.RECT, K_), "conv1")
    cfg.rms_norm(RmsNormCfg(), "norm1")
    cfg.conv2d(Conv2dCfg(3, 1, 1, 32, Act.IDENTITY, K_), "conv2")
    cfg.rms_norm(RmsNormCfg(Act.RECT, 1e-3), "norm2")
    cfg.affine(AffineCfg(50, Act.IDENTITY, X_), "fc1")
    cfg.rms_norm(RmsNormCfg(Act.LOGISTIC), "norm3")
    return _head(cfg)


def in_a_graph():
    """Behind the sum of two arms, one of which ends in a ReLU, and in an arm."""
    g = C.GraphOperatorConfig().input("data", Data3dCfg((8, 8, 3), normalize=True))
    g.op("conv1", Conv2dCfg(3, 1, 1, 32, Act.RECT, K_), "data")
    g.op("norm1", RmsNormCfg(Act.RECT), "conv1")
    g.op("conv2", Conv2dCfg(3, 1, 1, 32, Act.IDENTITY, K_), "norm1")
    g.op("sum", C.JoinCfg(2), ["conv2", "conv1"])
    g.op("norm2", RmsNormCfg(), "sum")
    g.op("fc", AffineCfg(10, Act.IDENTITY, X_), "norm2")
    return g.loss("loss", SoftmaxKLLossCfg(10), "fc")


def go():
    return zoo.go_policy_resnet(6, 16, 2, norm="rms")


def _both(monkeypatch, make, batch=4):
    _install(monkeypatch)
    monkeypatch.setattr(Net, "device_path_on_cpu", True)
    dev = Net(make(), batch, device="cpu", seed=(3, 4))
    monkeypatch.setattr(Net, "device_path_on_cpu", False)
    ref = Net(make(), batch, device="cpu", seed=(3, 4))
    assert torch.equal(dev.params, ref.params.detach())
    with torch.no_grad():                       # both see the bf16-rounded weights; scales that are not all one
        for net in (dev, ref):
            net.params.copy_(dev.params16.float())
            gen = torch.Generator().manual_seed(9)
            for op in net.ops:
                for s in op.segs:
                    if s.name.endswith(".scale"):
                        live = net.seg_view(s) != 0
                        net.seg_view(s)[live] = 1.0 + 0.25 * torch.randn(s.shape, generator=gen)[live]
    return dev, ref


@pytest.mark.parametrize("make,classes", [(blocks, 10), (stem, 10), (alone, 10), (in_a_graph, 10), (go, 361)])
@pytest.mark.parametrize("bits", [16, 32])
def test_device_path_matches_reference_path(monkeypatch, make, classes, bits):
    """With bf16 buffers by the figures of the same comparison of other networks: a noise of up to 0.15 of a gradient (0.3 behind the
    361-way softmax over one plane). With fp32 ones it shrinks with the half steps, 2^-24 / 2^-8, to 5e-6, grows with the root of
    the sums' lengths (below 5000: 70 times) to 3e-4, and a value within rounding of a ReLU's edge may take one of the 2 x 10^4 live
    deltas and more away, 7e-3 of their norm: 1e-2."""
    if bits == 32:
        monkeypatch.setattr(torch, "bfloat16", torch.float32)
        monkeypatch.setattr(torch.Tensor, "bfloat16", torch.Tensor.float)
    dev, ref = _both(monkeypatch, make)
    w, h, c = dev.input_op.cfg.in_dims
    torch.manual_seed(1)
    x, y = torch.randint(0, 256, (4, c, h, w), dtype=torch.uint8), torch.randint(0, classes, (4,))
    dev.load_batch(x, y.int())
    ref.load_batch(x, y)
    for n in (dev, ref):
        n.forward(True)
        n.backward()
    near = 2e-2 if bits == 16 else 1e-4
    dl, rl = dev.read_stats()[0], ref.read_stats()[0]
    assert abs(dl - rl) < near * max(1.0, abs(rl)), (dl, rl)
    biggest = max(float(ref.grads[s.offset: s.offset + s.numel].norm()) for s in dev.segs)
    for seg in dev.segs:
        a, b = (n.grads[seg.offset: seg.offset + seg.numel] for n in (dev, ref))
        if float(b.norm()) < 1e-4 * biggest:
            continue
        assert float((a - b).norm() / b.norm()) < (1e-2 if bits == 32 else 0.3 if make is go else 0.15), seg.name
    for op in dev.ops[1:-1]:
        live = op.out_hwc[2]
        if op.out is not None and op.out.shape[-1] > live:
            assert float(op.out[..., live:].abs().sum()) == 0.0, op.name
    # inference: nothing but the parameters counts, and no statistics are kept
    before = dev.params.clone()
    for n in (dev, ref):
        n.forward(False)
    dl, rl = dev.read_stats()[0], ref.read_stats()[0]
    assert abs(dl - rl) < near * max(1.0, abs(rl)) and torch.equal(dev.params, before)


def test_reference_path_gradients_are_differences():
    """d loss along a direction of all parameters, by central differences of the fp32 reference path in 64 bits."""
    net = Net(blocks(), 3, device="cpu", seed=(3, 4))
    for name in ("params", "grads"):
        setattr(net, name, getattr(net, name).detach().double())
    net.params.requires_grad_(True)
    net.params.grad = net.grads
    x, y = torch.randint(0, 256, (3, 3, 12, 12), dtype=torch.uint8, generator=torch.Generator().manual_seed(0)), torch.tensor([1, 5, 7])
    images = net.input_op.ref_forward(x, True, 0).double()
    net.input_op.ref_forward = lambda *a: images

    def loss(p):
        with torch.no_grad():
            net.params.copy_(p)
        net.load_batch(x, y)
        net.forward(True)
        return net._cpu_loss
    start = net.params.detach().clone()
    loss(start).backward()
    got = net.grads.clone()
    way = torch.randn(start.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    way *= (start != 0)
    step = 1e-7
    slope = (loss(start + step * way).item() - loss(start - step * way).item()) / (2 * step)
    # central differences of step 1e-7 in 64 bits: 1e-16 / 1e-7 = 1e-9 of the loss, and 1e-14 of its third derivative; a ReLU
    # that changes sides within the step adds a part of its slope
    assert abs(slope - float((got * way).sum())) < 1e-5 * float((got * way).abs().sum())


def test_parameters_go_out_and_in():
    a, b = (Net(blocks(), 2, device="cpu", seed=s) for s in ((3, 4), (5, 6)))
    assert not torch.equal(a.params, b.params)
    b.decode_params(a.encode_params())
    assert torch.equal(a.params, b.params)
    a.mom.normal_(generator=torch.Generator().manual_seed(0))
    for s in a.segs:        # padded channels have no momentum
        if s.name.endswith(".scale"):
            a.seg_view(s, "mom")[a.seg_view(s) == 0] = 0
    b.decode_state(a.encode_state())
    for s in a.segs:
        assert torch.equal(a.seg_view(s, "mom"), b.seg_view(s, "mom")), s.name
    assert a.params_len == sum(w * 9 for w in (3 * 16, 16 * 16, 16 * 16, 16 * 40, 40 * 40, 40 * 40, 40 * 24)) + 16 * 3 + 40 * 3 + 24 + 24 * 10 + 10


def test_wrong_configurations_are_refused():
    with pytest.raises(ValueError, match="normalisation"):
        zoo.go_policy_resnet(6, 16, 2, norm="layer")
    for eps in (0.0, -1.0, float("nan")):
        cfg = SequentialOperatorConfig().data3d(Data3dCfg((8, 8, 3), normalize=True)).rms_norm(RmsNormCfg(epsilon=eps))
        with pytest.raises(ValueError, match="epsilon"):
            Net(_head(cfg), 2, device="cpu")
        cfg = SequentialOperatorConfig().data3d(Data3dCfg((8, 8, 3), normalize=True)).rms_conv2d(RmsConv2dCfg(3, 1, 1, 8, epsilon=eps))
        with pytest.raises(ValueError, match="epsilon"):
            Net(_head(cfg), 2, device="cpu")
    cfg = SequentialOperatorConfig().data3d(Data3dCfg((2, 2, 3), normalize=True)).rms_conv2d(RmsConv2dCfg(1, 1, 0, 16_448))
    with pytest.raises(ValueError, match="channels"):
        Net(_head(cfg), 2, device="cpu")


# ---- clipping
def _batches(n, batch):
    g = torch.Generator().manual_seed(11)
    return [(torch.randint(0, 256, (batch, 1, 28, 28), dtype=torch.uint8, generator=g),
             torch.randint(0, 10, (batch,), dtype=torch.int32, generator=g)) for _ in range(n)]


@pytest.mark.parametrize("order", list(SyncOrder))
@pytest.mark.parametrize("mode", list(Momentum))
def test_clipped_steps_against_the_rule(order, mode):
    """Each step of the engine is one of the rule in 64 bits with the gradients times min(1, bound / norm)."""
    batch, bound = 8, 0.5
    opt = SgdOptConfig(minibatch_size=2 * batch, step_size=StepSizeSchedule.constant(0.1), momentum=mode, mu=0.9, l2_reg_coef=1e-2,
                       sync_order=order, clip_norm=bound)
    net = Net(zoo.mnist_fc1(), batch, device="cpu", seed=(3, 7), minibatch_size=2 * batch)
    eng = StepEngine(net, opt)
    assert eng.grad_norm() == 0.0
    d, clipped = net.decay_len, 0
    for i, (x, y) in enumerate(_batches(8, batch)):
        if i % 2 == 0:
            w, v, g0 = net.params.detach().double(), net.mom.double(), net.grads.double()
            probe = Net(zoo.mnist_fc1(), batch, device="cpu", seed=(3, 7), minibatch_size=2 * batch)
            with torch.no_grad():
                probe.params.copy_(net.params)
        probe.load_batch(x, y)
        probe.forward(True)
        probe.backward()
        eng.feed(x, y)
        eng.step()
        if i % 2 == 0:
            continue
        g = g0 + probe.grads.double()
        norm = float(g.norm())
        # fp32 gradients added in two orders: a few times 2^-24
        assert abs(eng.grad_norm() - norm) < 1e-5 * norm
        clipped += norm > bound
        coef = min(1.0, bound / norm)
        for lo, hi, l2 in ((0, d, 1e-2), (d, net.flat_len, 0.0)):
            reference_step(w[lo:hi], g[lo:hi], v[lo:hi], 0.1, 0.9 if mode != Momentum.ZERO else 0.0, l2, coef, mode)
        for got, want in ((net.params.detach(), w), (net.mom, v), (net.grads, g)):
            assert (got.double() - want).abs().max() < 1e-5 * max(1.0, float(want.abs().max()))
    assert clipped


def test_gradients_that_are_not_finite_leave_a_step_without_them():
    net = Net(zoo.mnist_fc1(), 4, device="cpu", seed=(3, 7))
    st = SgdStepper(net, Momentum.UPDATE, 0.9, 0.0, clip_norm=1.0)
    with torch.no_grad():
        net.mom.fill_(0.5)
        net.grads[3] = float("nan")
        before = net.params.detach().clone()
        st.step(0.1)
    assert math.isnan(st.grad_norm())
    assert torch.equal(net.mom, torch.full_like(net.mom, 0.45)) and torch.allclose(net.params.detach(), before + 0.45) and (net.grads == 0).all()


def test_clipping_on_the_device_branch_of_the_engine(monkeypatch):
    from test_engine_emulated import _device_engine
    opt = SgdOptConfig(minibatch_size=8, step_size=StepSizeSchedule.constant(0.05), momentum=Momentum.UPDATE, mu=0.9, l2_reg_coef=1e-3,
                       clip_norm=0.3)
    cpu_net = Net(zoo.mnist_fc1(), 8, device="cpu", seed=(2, 3))
    cpu_eng = StepEngine(cpu_net, opt)
    _install(monkeypatch)
    monkeypatch.setattr(kernel_emulation, "install", lambda mp: None)
    dev_eng, dev_net = _device_engine(monkeypatch, zoo.mnist_fc1, 8, opt)
    with torch.no_grad():
        cpu_net.params.copy_(dev_net.params16.float())
        dev_net.params.copy_(dev_net.params16.float())
    for x, y in _batches(4, 8):
        for eng in (dev_eng, cpu_eng):
            eng.feed(x, y)
            eng.step()
        # bf16 deltas (2^-8 of each, in no direction) against fp32 ones
        assert abs(dev_eng.grad_norm() - cpu_eng.grad_norm()) < 2.0 ** -6 * cpu_eng.grad_norm() and cpu_eng.grad_norm() > 0.3
    moved = cpu_net.params.detach() - dev_net.params
    assert float(moved.norm()) < 0.05 * 4 * 0.3 * 2.0 ** -4


def test_what_cannot_be_clipped_is_refused():
    net = Net(zoo.mnist_fc1(), 4, device="cpu", seed=(3, 7))
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="norm"):
            SgdStepper(net, Momentum.UPDATE, 0.9, 0.0, clip_norm=bad)
    st = SgdStepper(net, Momentum.UPDATE, 0.9, 0.0, clip_norm=1.0)
    for part in ({"lo": 0, "hi": 64}, {"lo": 64}, {"grid": (296, 128)}):
        with pytest.raises(ValueError, match="part"):
            st.step(0.1, **part)
    assert SgdStepper(net, Momentum.UPDATE, 0.9, 0.0).grad_norm() is None
    opt = SgdOptConfig(minibatch_size=4, clip_norm=1.0)
    with pytest.raises(ValueError, match="clip_norm"):
        StepEngine(net, opt, LocalOverlapComm())
    assert StepEngine(net, opt, NullComm()).stepper.clip_norm == 1.0


def _two_ranks(rank, world):
    import torch.distributed as dist
    from rembrandt_b200.parallel.comm import AllreduceComm
    torch.set_num_threads(1)
    net = Net(zoo.mnist_fc1(), 8, device="cpu", seed=(3, 7))
    opt = SgdOptConfig(minibatch_size=8, step_size=StepSizeSchedule.constant(0.5), momentum=Momentum.ZERO, mu=0.0, clip_norm=0.2)
    eng = StepEngine(net, opt, AllreduceComm())
    for i, (x, y) in enumerate(_batches(2 * 3, 8)):
        if i % world != rank:        # every rank its own batches
            continue
        before = net.params.detach().clone()
        eng.feed(x, y)
        eng.step()
        norm = eng.grad_norm()
        moved = float((net.params.detach() - before).norm())
        assert norm > 0.2 and abs(moved - 0.5 * 0.2) < 1e-5 * 0.1 + 2.0 ** -23 * float(before.norm())
        both = torch.tensor([norm, -norm], dtype=torch.float64)
        dist.all_reduce(both, op=dist.ReduceOp.MAX)
        assert both[0] == norm and both[1] == -norm      # the norm of the averaged gradients, on every rank
        first = net.params.detach().clone()
        dist.broadcast(first, 0)
        assert torch.equal(first, net.params.detach())


def test_ranks_clip_what_they_have_averaged():
    from cpu_ranks import run_ranks
    run_ranks(2, _two_ranks)


def test_clip_coefficient():
    assert clip_coefficient(2.0, 1.0) == 0.5 and clip_coefficient(1.0, 1.0) == 1.0 and clip_coefficient(0.0, 1.0) == 1.0
    assert clip_coefficient(float("inf"), 1.0) == 0.0 and clip_coefficient(float("nan"), 1.0) == 0.0


def test_the_go_tool_with_channel_normalisation_and_clipping(capsys):
    sgd = train_gogod.main(["--device", "cpu", "--batch", "8", "--iters", "3", "--display-iters", "1", "--synthetic-size", "64", "--channels", "8",
                            "--blocks", "2", "--planes", "6", "--norm", "rms", "--clip-norm", "0.25"])
    assert sgd.engine.iter == 3 and sgd.engine.stepper.clip_norm == 0.25
    assert any(type(op).__name__ == "RmsStackResConv2dOp" for op in sgd.engine.net.ops)
    assert "gradient norm" in capsys.readouterr().err
