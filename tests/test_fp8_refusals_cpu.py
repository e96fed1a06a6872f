"""Calls of the 8-bit products that are refused, on the CPU; the same calls on the GPU are in test_fp8_refusals_gpu.py."""
import pytest
import torch

from shift_b200.ops import fp8
from shift_b200.ops._ext import available, ext

needs_ext = pytest.mark.skipif(not available(), reason="the extension is not built")


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


def moved(x, by):
    """The same bytes, starting ``by`` bytes behind a boundary."""
    flat = torch.zeros(x.numel() + 16, dtype=torch.uint8, device=x.device)
    flat[by:by + x.numel()] = x.reshape(-1).view(torch.uint8)
    return flat[by:by + x.numel()].view(x.dtype).view(x.shape)


@needs_ext
@pytest.mark.parametrize("by", [1, 2, 3])
def test_scales_off_their_words_are_refused(by):
    """The extension's check of an operand, which comes before that of its device: no GPU is needed to see it."""
    a, b = (fp8.quantize(torch.ones(n, 600)) for n in (4, 6))
    a = a._replace(scale=moved(a.scale, by))
    assert bool((fp8.matmul(a, b) == 600).all())       # on the CPU any place will do
    with pytest.raises(ValueError, match="4 bytes"):
        ext().fp8_matmul(a.data, a.scale, 600, b.data, b.scale, 600, None, None, 0, False, False,
                         torch.zeros(1, dtype=torch.int32))


def check_out_rows_apart(device):
    a, b = fp8.quantize(torch.ones(4, 40, device=device)), fp8.quantize(torch.ones(8, 40, device=device))
    offs = torch.tensor([0, 2, 4], dtype=torch.int32, device=device)
    flat = torch.zeros(100, device=device)
    for out in (flat[:8].expand(4, 8), flat.as_strided((4, 8), (7, 1))):
        with pytest.raises(ValueError, match="overlap"):
            fp8.matmul(a, b, out=out)
        if out.stride(0):
            with pytest.raises(ValueError, match="overlap"):
                fp8.matmul(a, b, out=out, accumulate=True)
    for out in (flat[:4].expand(4, 4), flat.as_strided((4, 4), (3, 1))):
        with pytest.raises(ValueError, match="overlap"):
            fp8.grouped_matmul(a, b, offs, out=out)
    assert bool((flat == 0).all())
    assert bool((fp8.matmul(a, b, out=flat.as_strided((4, 8), (8, 1))) == 40).all())
    one = fp8.quantize(torch.ones(1, 40, device=device))
    assert bool((fp8.matmul(one, b, out=flat[:8].expand(1, 8)) == 40).all())       # a single row has no neighbour


def test_out_rows_apart():
    check_out_rows_apart("cpu")
