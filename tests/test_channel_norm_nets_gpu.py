"""Networks normalised over channels, and clipped training, on the device: against the CPU reference path, and captured."""
import pytest
import torch

from rembrandt_b200.engine import StepEngine
from rembrandt_b200.models import zoo
from rembrandt_b200.models.net import Net
from rembrandt_b200.ops import native_ops as K
from rembrandt_b200.optim.sgd import Momentum, SgdOptConfig, StepSizeSchedule
from test_channel_norm_nets import alone, blocks, go, in_a_graph, stem

pytestmark = pytest.mark.gpu


def _inputs(net, batch, classes, seed=1):
    w, h, c = net.input_op.cfg.in_dims
    gen = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (batch, c, h, w), dtype=torch.uint8, generator=gen),
            torch.randint(0, classes, (batch,), generator=gen, dtype=torch.int32))


@pytest.mark.parametrize("make,classes", [(blocks, 10), (stem, 10), (alone, 10), (in_a_graph, 10), (go, 361)])
def test_device_path_matches_reference_path(make, classes):
    """The figures of the networks' other comparisons with bf16 activations and deltas: 0.15 of a gradient, 0.35 behind the 361-way
    softmax over one plane."""
    batch = 4
    g, c = Net(make(), batch, device="cuda", seed=(3, 4)), Net(make(), batch, device="cpu", seed=(3, 4))
    with torch.no_grad():
        c.params.copy_(g.params16.float().cpu())
        g.params.copy_(g.params16.float())
    x, y = _inputs(c, batch, classes)
    g.load_batch(x.cuda(), y.cuda())
    c.load_batch(x, y.long())
    for n in (g, c):
        n.forward(True)
        n.backward()
    gl, cl = g.read_stats()[0], c.read_stats()[0]
    assert abs(gl - cl) < 3e-2 * max(1.0, abs(cl)) and K.read_status() == 0
    gg = g.grads.cpu()
    biggest = max(float(c.grads[s.offset: s.offset + s.numel].norm()) for s in g.segs)
    for seg in g.segs:
        a, b = gg[seg.offset: seg.offset + seg.numel], c.grads[seg.offset: seg.offset + seg.numel]
        if float(b.norm()) >= 1e-3 * biggest:
            assert float((a - b).norm() / b.norm()) < (0.35 if make is go else 0.15), seg.name
    for n in (g, c):
        n.forward(False)
    gl, cl = g.read_stats()[0], c.read_stats()[0]
    assert abs(gl - cl) < 3e-2 * max(1.0, abs(cl))


def _engine(make, batch, clip, graph, momentum=Momentum.ZERO, lr=0.5, accum=1):
    opt = SgdOptConfig(minibatch_size=batch * accum, step_size=StepSizeSchedule.constant(lr), momentum=momentum, mu=0.9, l2_reg_coef=0.0,
                       clip_norm=clip)
    net = Net(make(), batch, device="cuda", seed=(5, 7), minibatch_size=batch * accum)
    return StepEngine(net, opt, use_graph=graph)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("accum", [1, 2])
def test_clipped_steps_of_a_network_with_channel_normalisation(graph, accum):
    """Without momentum or weight decay a step has the length rate * min(norm, bound), eager or captured, whatever the rate is set
    to in between; weights are rounded to half of 2^-23 of themselves."""
    batch, seen = 8, []
    for bound in (0.05, 1e6):
        eng = _engine(go, batch, bound, graph, accum=accum)
        norms = []
        for i in range(6):
            before = eng.net.params.clone()
            rate = 0.5 if i % 2 else 0.25
            eng.set_lr(rate)
            for k in range(accum):
                x, y = _inputs(eng.net, batch, 361, seed=10 * i + k)
                eng.feed(x.pin_memory(), y.pin_memory())
                eng.step()
            norm = eng.grad_norm()
            norms.append(norm)
            moved = float((eng.net.params.double() - before.double()).norm())
            want = rate * min(norm, bound)
            assert abs(moved - want) <= 1e-5 * want + 2.0 ** -23 * float(before.norm())
            assert float(eng.net.grads.abs().max()) == 0.0
            assert torch.equal(eng.net.params16, eng.net.params.bfloat16())
        if bound == 0.05:
            assert min(norms) > bound
        seen.append(norms[0])
        if graph:
            assert eng._graphs
    # the first batch's gradients are the same, clipped or not: sums of the convolutions in another order, 2^-24 of their terms each,
    # rounded to bf16 (2^-8 of a value, in either direction)
    assert abs(seen[0] - seen[1]) < 1e-3 * seen[0]
    # ... and those of the reference path: a noise of 0.35 at right angles to it adds 1 - sqrt(1 + 0.35^2) = 6 %
    ref = Net(go(), batch, device="cpu", seed=(5, 7), minibatch_size=batch * accum)
    with torch.no_grad():
        ref.params.copy_(ref.params.bfloat16().float())
    for k in range(accum):
        x, y = _inputs(ref, batch, 361, seed=k)
        ref.load_batch(x, y.long())
        ref.forward(True)
        ref.backward()
    assert abs(seen[0] / float(ref.grads.norm()) - 1.0) < 0.1


def test_clipping_with_momentum_captured_and_eager():
    """The same norms and parameters from both, but for the order of sums."""
    ends = []
    with K.gemm_options(deterministic=1):
        for graph in (False, True):
            eng = _engine(zoo.lenet, 8, 0.3, graph, Momentum.UPDATE_NESTEROV, lr=2e-3)
            norms = []
            for i in range(5):
                x, y = _inputs(eng.net, 8, 10, seed=i)
                eng.feed(x.pin_memory(), y.pin_memory())
                eng.step()
                norms.append(eng.grad_norm())
            start = Net(zoo.lenet(), 8, device="cpu", seed=(5, 7)).params.detach()
            ends.append((norms, eng.net.params.cpu() - start))
    (na, a), (nb, b) = ends
    for p, q in zip(na, nb):
        assert abs(p - q) < 1e-4 * p and p > 0.3
    assert float((a - b).norm()) < 1e-4 * float(a.norm())


def test_inference_does_not_depend_on_the_rest_of_a_batch():
    net = Net(go(), 4, device="cuda", seed=(5, 7), training=False)
    x, y = _inputs(net, 4, 361)
    outs = []
    for images in (x, x[[0, 0, 0, 0]]):
        net.load_batch(images.cuda(), y.cuda())
        net.forward(False)
        outs.append(net.loss_op.flat[0].clone())
    assert torch.equal(*outs)


def test_features_in_8_bits_are_those_of_the_network():
    """The last block's sum in 8 bits stands for what the block hands on: half a step of e4m3 (2^-4) and of bf16 (2^-8)."""
    net = Net(go(), 4, device="cuda", seed=(5, 7))
    x, y = _inputs(net, 4, 361)
    net.load_batch(x.cuda(), y.cuda())
    net.forward(True)
    u = net.ops[-3].u2
    rows, cp = u.rstd.numel(), u.kp
    q, scales = torch.empty((rows, cp), device="cuda", dtype=torch.float8_e4m3fn), torch.empty(rows, device="cuda")
    K.rms_norm_fwd_e4m3(u.conv_out, rows, cp, u.ko, u.eps, u.v(u.seg_g), q, scales, relu=True)
    got, want = q.float() * scales[:, None], net.ops[-3].out.reshape(rows, cp).float()
    assert want.abs().sum() > 0
    assert ((got - want).abs() <= (2.0 ** -4 + 2.0 ** -7) * want.abs() + scales[:, None] * 2.0 ** -10 * 1.01).all()
