"""Clipped training as the tools and the stepper set it up (no GPU)."""
import pytest

from rembrandt_b200.cli import common, train_mnist


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
