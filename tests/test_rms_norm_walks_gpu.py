"""Normalisation over channels with more rows than the device holds at once, so that every block takes several groups of them and
some a last group that is not full, and with the widths between the others: by the bounds of the ordinary shapes."""
import pytest

from test_rms_norm_gpu import test_backward as backward
from test_rms_norm_gpu import test_forward as forward
from test_rms_norm_gpu import test_forward_into_8_bits as forward_into_8_bits

pytestmark = pytest.mark.gpu

WIDTHS = [(37, 384, 384), (35, 264, 259), (5, 288, 281), (21, 192, 177), (300, 96, 96), (41, 256, 256), (9, 640, 633)]
WALKS = [(100001, 32, 20), (60001, 64, 64), (100001, 96, 80), (30001, 128, 100), (40001, 192, 190), (20001, 256, 250), (20001, 320, 300),
         (20001, 384, 384), (20001, 512, 500), (20001, 768, 741), (12001, 1000, 999), (4001, 1040, 1033), (2001, 8200, 8193), (1201, 16384, 16000)]


@pytest.mark.parametrize("rows,C,c_valid", WIDTHS + WALKS)
@pytest.mark.parametrize("residual,relu", [(False, True), (True, False)])
def test_forward(rows, C, c_valid, residual, relu):
    forward(rows, C, c_valid, residual, True, relu)
    forward_into_8_bits(rows, C, c_valid, residual, relu)


@pytest.mark.parametrize("rows,C,c_valid", WIDTHS + WALKS)
@pytest.mark.parametrize("add,relu", [(False, False), (False, True), (True, False), (True, True)])
def test_backward(rows, C, c_valid, add, relu):
    backward(rows, C, c_valid, add, relu)
