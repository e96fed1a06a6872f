"""Calls of the 8-bit products that are refused, on the CPU; the same calls on the GPU are in test_fp8_refusals_gpu.py."""
import pytest
import torch

from shift_b200.ops import fp8


def check_segments_are_needed(device):
    a, b = fp8.quantize(torch.ones(4, 4096, device=device)), fp8.quantize(torch.ones(6, 4096, device=device))
    for groups in (1, 2):
        out = torch.full((groups, 4, 6), 3.0, device=device)
        with pytest.raises(ValueError, match="offs"):
            fp8.grouped_wgrad(a, b, None, out)
        assert bool((out == 3).all())
    with pytest.raises(ValueError, match="offs"):
        fp8.grouped_matmul(a, b, None)


def test_segments_are_needed():
    check_segments_are_needed("cpu")
