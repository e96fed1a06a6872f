"""8-bit moments of quiet elements in the kernel."""
import pytest
import torch

from shift_b200.optim import AdamWMany, State8
from test_optim_quiet_cpu import longest_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("every", [1, 7])
@pytest.mark.parametrize("quiet", [1e-4, 1e-5, 1e-6, 1e-7])
def test_no_step_is_longer_than_the_ratio_of_the_moments_allows(quiet, every):
    assert longest_step(True, quiet, every, DEV) <= 17           # the bound is derived beside the CPU's test


@pytest.mark.parametrize("n", [300, 4096])
def test_roots_above_zero_keep_a_code_and_others_are_as_they_were(n):
    """Zero, tiny, ordinary and not finite gradients in one block, at sizes with and without a ragged end."""
    g = torch.randn(n, generator=torch.Generator().manual_seed(1))
    g[::5] = 0.0
    g[1::5] *= 1e-9
    g[2::50] = float("nan")
    g[3::70] = float("inf")
    w = torch.zeros(n, device=DEV)
    m, v = State8.zeros(w), State8.zeros(w)
    AdamWMany([w], [m], [v]).step([g.to(DEV)], lr=1e-3, step=1)
    code = v.code.view(torch.uint8).cpu()
    finite = torch.isfinite(g)
    assert torch.equal((code & 0x7F) > 0, g != 0)
    assert bool((code[finite & (g != 0) & (g.abs() < 1e-7)] == 1).all())
    assert torch.equal(torch.isnan(v.code.float().cpu()), ~finite)
