"""The kernel benchmark's clipped step clips every time it is called."""
import pytest

from rembrandt_b200.cli import bench_ops

pytestmark = pytest.mark.gpu


def test_the_clipped_step_clips(monkeypatch):
    step = next(fn for name, fn, _ in bench_ops.cases(1) if name == "sgd_clipped_62M")
    sweep, seen = bench_ops.K.sgd_fused, []

    def look(*args, clip=None):
        seen.append(clip.tolist())
        sweep(*args, clip=clip)
    monkeypatch.setattr(bench_ops.K, "sgd_fused", look)
    for _ in range(3):
        step()
    # 62.4 million gradients of 1e-3: their norm is 7.9, the bound 1
    assert all(7.89 < norm < 7.9 and 1 / 7.9 < coefficient < 1 / 7.89 for norm, coefficient in seen) and len(seen) == 3
