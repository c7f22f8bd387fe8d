"""Clipped training as the tools and the stepper set it up (no GPU)."""
import pytest

from rembrandt_b200.cli import common, train_mnist
from rembrandt_b200.models import zoo
from rembrandt_b200.models.net import Net
from rembrandt_b200.optim.sgd import Momentum
from rembrandt_b200.optim.stepper import SgdStepper


@pytest.mark.parametrize("arguments,exchange", [
    (["--clip-norm", "1"], "allreduce"), ([], "fused_allreduce_sgd"), (["--clip-norm", "1", "--comm", "gossip_p2p"], "gossip_p2p"),
    (["--clip-norm", "1", "--comm", "fused_allreduce_sgd"], "fused_allreduce_sgd")])
def test_the_tools_exchange_on_several_gpus(monkeypatch, arguments, exchange):
    """The default exchange updates parameters from inside backward, which clipping refuses: with it the default is another."""
    class Chosen(Exception):
        pass

    def choose(name, **kw):
        raise Chosen(name)
    monkeypatch.setattr(common, "init_distributed", lambda *a: (0, 2))
    monkeypatch.setattr(common.comm_mod, "make_comm", choose)
    with pytest.raises(Chosen, match=f"^{exchange}$"):
        train_mnist.main(["--device", "cuda", *arguments])


@pytest.mark.parametrize("bound", [1e-60, 2.0 ** -150])
def test_bounds_that_are_no_float32_are_refused_when_the_stepper_is_made(bound):
    net = Net(zoo.mnist_fc1(), 2, device="cpu", seed=(3, 7))
    with pytest.raises(ValueError, match="norm"):
        SgdStepper(net, Momentum.UPDATE, 0.9, 0.0, clip_norm=bound)
    assert SgdStepper(net, Momentum.UPDATE, 0.9, 0.0, clip_norm=2.0 ** -149).clip_norm == 2.0 ** -149
