"""8-bit moments of elements whose gradients are far smaller than those of their block's loudest element."""
import pytest
import torch

from shift_b200.ops import reference as ref
from shift_b200.optim import AdamWMany, State8

LR = 1e-3


def longest_step(eight, quiet, every, device="cpu", steps=150):
    """The largest |change of a weight| / lr of a block with one gradient of deviation 1 and 127 of ``quiet``, which are
    there in one step of ``every``."""
    g = torch.Generator().manual_seed(3)
    w = torch.zeros(128, device=device)
    m, v = ((State8.zeros(w), State8.zeros(w)) if eight else (torch.zeros_like(w), torch.zeros_like(w)))
    opt = AdamWMany([w], [m], [v])
    worst = 0.0
    for t in range(1, steps + 1):
        grad = torch.randn(128, generator=g)
        grad[1:] *= quiet if t % every == 0 else 0.0
        before = w.clone()
        opt.step([grad.to(device)], lr=LR, wd=0.0, step=t)
        worst = max(worst, float((w - before).abs().max()) / LR)
    return worst


# Without rounding |m| <= 7.3 sqrt(v) (Cauchy-Schwarz: 0.1^2 / 0.001 times the sum of (0.81 / 0.999)^i), and c2 / c1 <= 1.
# A code of m is above its value by 1/8, one of sqrt(v) below by half at most once code 0 is out: 7.3 * 1.125 * 2 < 17.
@pytest.mark.parametrize("every", [1, 7])
@pytest.mark.parametrize("quiet", [1e-4, 1e-5, 1e-6, 1e-7])
def test_no_step_is_longer_than_the_ratio_of_the_moments_allows(quiet, every):
    assert longest_step(False, quiet, every) <= 7.3
    assert longest_step(True, quiet, every) <= 17


def test_a_root_above_zero_keeps_a_code():
    x = torch.zeros(256)
    x[0], x[1:4], x[200] = 1.0, torch.tensor([1e-7, 1e-30, 1e-45]), 1e-45
    for bits in (0, 0x8000, 0xFFFF):
        code, scale = ref.moment_encode(x, torch.full((256,), bits), root=True)
        assert torch.equal(code.view(torch.uint8) > 0, x > 0)
        assert code.view(torch.uint8)[1:4].tolist() == [1, 1, 1]
    assert ref.moment_encode(x, torch.zeros(256, dtype=torch.int64))[0].view(torch.uint8)[1] == 0     # exp_avg may vanish


def test_a_root_that_is_not_finite_stays_so():
    x = torch.ones(128)
    x[3], x[9], x[10] = float("nan"), float("inf"), 1e-9
    code, _ = ref.moment_encode(x, torch.zeros(128, dtype=torch.int64), root=True)
    assert torch.isnan(code.float()).nonzero().flatten().tolist() == [3, 9] and int(code.view(torch.uint8)[10]) == 1
