"""8-bit moments on the GPU and by the CPU's statement: the same codes, not only codes next to one another."""
import pytest
import torch

from shift_b200.optim import AdamWMany
from test_optim_cpu import H, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1.0, 0.37])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_and_scales_are_the_statements(dtype, scale):
    """Six steps, so that the codes of one enter the next; about a million roundings each."""
    sizes = [(1 << 18,), (777, 131)]
    dev, cpu = make(dtype, True, True, "cuda", sizes), make(dtype, True, True, "cpu", sizes)
    one, two = (AdamWMany(x[0], x[2], x[3], x[4]) for x in (dev, cpu))
    g = torch.Generator().manual_seed(8)
    for step in range(1, 7):
        grads = [torch.randn(p.shape, generator=g) * torch.exp(2 * torch.randn(p.shape, generator=g)) for p in cpu[0]]
        one.step([x.to(dtype).cuda() for x in grads], step=step, grad_scale=scale, **H)
        two.step([x.to(dtype) for x in grads], step=step, grad_scale=scale, **H)
        for a, b in zip(dev[2] + dev[3], cpu[2] + cpu[3]):
            assert torch.equal(a.code.float().cpu(), b.code.float())          # values: zeros of either sign are equal
            assert torch.equal(a.scale.view(torch.uint8).cpu(), b.scale.view(torch.uint8))
