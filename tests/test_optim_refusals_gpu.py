"""What ``AdamWMany`` refuses on the GPU: the checks are the extension's."""
import pytest
import torch

from test_optim_refusals_cpu import check_inference_tensors, make, spoilt, words

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("k", range(4))
def test_the_flag_is_not_a_word_that_is_read(k):
    opt, p, g = make(DEV)
    skip, step_dev, flag = words(DEV)[k]
    with pytest.raises(ValueError, match="nonfinite"):
        opt.step(g, skip=skip, step_dev=step_dev, nonfinite=flag)
    assert bool((p == 1).all())
    block = torch.zeros(8, dtype=torch.int32, device=DEV)
    block[1:4] = torch.tensor([1e-3, 0.1, 0.03]).view(torch.int32)
    opt.step(g, step_dev=block, skip=block[4:], nonfinite=block[5:])          # neighbours are no matter
    assert bool((p != 1).all())


@pytest.mark.parametrize("eight", [False, True])
def test_tensors_that_were_given_other_memory(eight):
    for opt, p, g, which, k in spoilt(eight, DEV):
        before = p.clone()
        with pytest.raises(ValueError):
            opt.step(g)
        assert torch.equal(p, before), (which, k)


@pytest.mark.parametrize("eight", [False, True])
def test_tensors_that_were_moved_to_the_host(eight):
    from shift_b200.optim import AdamWMany, State8
    p = torch.ones(300, device=DEV)
    m, v = ((State8.zeros(p), State8.zeros(p)) if eight else (torch.zeros_like(p), torch.zeros_like(p)))
    opt = AdamWMany([p], [m], [v])
    p.data = p.data.cpu()
    for g in (torch.ones(300), torch.ones(300, device=DEV)):
        with pytest.raises(ValueError):
            opt.step([g])
    assert bool((p == 1).all())
    p.data = p.data.to(DEV)
    opt.step([torch.ones(300, device=DEV)])
    assert bool((p != 1).all())


def test_inference_tensors_are_refused_before_they_change():
    check_inference_tensors(DEV)
