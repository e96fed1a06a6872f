"""What ``AdamWMany`` refuses: words and memory that a step would read and write at once."""
import pytest
import torch

from shift_b200.optim import AdamWMany, State8


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


@pytest.mark.parametrize("eight", [False, True])
def test_tensors_that_share_a_part_of_their_memory(eight):
    def new(n):
        return State8.zeros(torch.empty(n)) if eight else torch.zeros(n)

    flat = torch.zeros(400)
    a, b = flat[:200], flat[199:]
    with pytest.raises(ValueError, match="share memory"):
        AdamWMany([a, b], [new(200), new(201)], [new(200), new(201)])
    with pytest.raises(ValueError, match="share memory"):
        AdamWMany([torch.zeros(200), torch.zeros(201)], [new(200), new(201)], [new(200), new(201)], masters=[a, b])
    if eight:
        code = torch.zeros(300, dtype=torch.uint8).view(torch.float8_e4m3fn)
        s = new(200)
        with pytest.raises(ValueError, match="share memory"):
            AdamWMany([torch.zeros(200)], [s._replace(code=code[:200])], [s._replace(code=code[100:], scale=s.scale.clone())])
    opt = AdamWMany([flat[:200], flat[200:]], [new(200), new(200)], [new(200), new(200)])         # neighbours may
    opt.step([torch.ones(200), torch.ones(200)])
    assert bool((flat < 0).all())


def spoilt(eight, device="cpu"):
    """Optimizers, made of sound tensors of which one was given other memory since."""
    other = [lambda x: x.float().half(), lambda x: x[:100].clone(),
             lambda x: torch.zeros(300, 2, device=device).to(x.dtype)[:, 0]]
    for which in ("exp_avg", "exp_avg_sq", "masters", "params"):
        for k, f in enumerate(other):
            if which == "params" and k == 0:
                continue                               # another floating type is a parameter's right
            p, w = torch.ones(300, device=device).bfloat16(), torch.ones(300, device=device)
            m, v = ((State8.zeros(p), State8.zeros(p)) if eight else (torch.zeros_like(w), torch.zeros_like(w)))
            opt = AdamWMany([p], [m], [v], [w])
            x = getattr(opt, which)[0]
            x = x.code if isinstance(x, State8) else x
            x.data = f(x)
            yield opt, p, [torch.ones(x.numel() if which == "params" else 300, device=device)], which, k
    if eight:
        p = torch.ones(300, device=device)
        for field in range(4):
            m, v = State8.zeros(p), State8.zeros(p)
            opt = AdamWMany([p], [m], [v])
            (m, v)[field // 2].scale.data = (m.scale[:1].clone() if field % 2 else m.scale.float())
            yield opt, p, [torch.ones(300, device=device)], "scale", field


@pytest.mark.parametrize("eight", [False, True])
def test_tensors_that_were_given_other_memory(eight):
    for opt, p, g, which, k in spoilt(eight):
        before = p.clone()
        with pytest.raises(ValueError):
            opt.step(g)
        assert torch.equal(p, before), (which, k)


def check_inference_tensors(device):
    with torch.inference_mode():
        opt, p, g = make(device)
        m = opt.exp_avg[0]
        opt.step(g)                                    # inside the mode they are as good as any
        before, moment = p.clone(), m.clone()
        assert bool((p != 1).all())
    with pytest.raises((ValueError, RuntimeError), match="nference"):
        opt.step(g)
    assert torch.equal(p, before) and torch.equal(m, moment)
    with pytest.raises(ValueError, match="inference"):
        AdamWMany([p], [m], [opt.exp_avg_sq[0]])


def test_inference_tensors_are_refused_before_they_change():
    check_inference_tensors("cpu")
