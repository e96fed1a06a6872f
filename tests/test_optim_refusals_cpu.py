"""What ``AdamWMany`` refuses: words and memory that a step would read and write at once."""
import pytest
import torch

from shift_b200.optim import AdamWMany


def words(device="cpu"):
    """(skip, step_dev, nonfinite) where the flag is a word that is read."""
    block = torch.zeros(8, dtype=torch.int32, device=device)
    return [(block[:1], None, block[:1]), (block, None, block[:1]), (None, block, block[3:4]), (None, block[1:5], block[1:])]


def make(device="cpu"):
    p, m, v = (torch.ones(300, device=device) for _ in range(3))
    return AdamWMany([p], [m], [v]), p, [torch.ones(300, device=device)]


@pytest.mark.parametrize("k", range(4))
def test_the_flag_is_not_a_word_that_is_read(k):
    opt, p, g = make()
    skip, step_dev, flag = words()[k]
    with pytest.raises(ValueError, match="nonfinite"):
        opt.step(g, skip=skip, step_dev=step_dev, nonfinite=flag)
    assert bool((p == 1).all())
    block = torch.zeros(8, dtype=torch.int32)
    block[1:4] = torch.tensor([1e-3, 0.1, 0.03]).view(torch.int32)
    opt.step(g, step_dev=block, skip=block[4:], nonfinite=block[5:])          # neighbours are no matter
    assert bool((p != 1).all())
