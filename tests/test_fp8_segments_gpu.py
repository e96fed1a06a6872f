"""Offsets that fall or leave the rows, on the GPU."""
import pytest
import torch

from shift_b200.ops._ext import check_status
from test_fp8_segments_cpu import FALLING, check_contraction, check_nothing_to_contract, check_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("o", FALLING)
def test_rows(o):
    check_rows(o, "cuda")
    torch.cuda.synchronize()
    check_status()


@pytest.mark.parametrize("o", FALLING)
def test_contraction(o):
    check_contraction(o, "cuda")
    torch.cuda.synchronize()
    check_status()


@pytest.mark.parametrize("o", FALLING + [[20, 30, 30, 90]])
def test_nothing_to_contract(o):
    check_nothing_to_contract(o, "cuda")
