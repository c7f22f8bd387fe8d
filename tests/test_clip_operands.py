"""Operands that a clipped update refuses before anything is launched (no GPU: a launch of the stand-in library fails the test)."""
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


def _sweep(clip, n=64, **change):
    t = {"w": torch.zeros(n), "g": torch.zeros(n), "v": torch.zeros(n), "w16": torch.zeros(n, dtype=torch.bfloat16)} | change
    K.sgd_fused(t["w"], t["g"], t["v"], t["w16"], n, 0.1, 0.9, 0.0, 1.0, 1, clip=clip)


@pytest.mark.parametrize("change", [{}, {"v": None}, {"w16": None}])
def test_a_coefficient_that_is_not_on_the_gpu(no_launch, change):
    with pytest.raises(ValueError, match="clip has to be on a GPU"):
        _sweep(torch.zeros(2), **change)
