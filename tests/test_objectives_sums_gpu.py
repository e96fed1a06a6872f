"""How far log-probabilities are off where many of them are added up: on average, and as a rule."""
import pytest
import torch

import packed_oracle as orc
from shift_b200.ops import objectives as ob
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _logits(rows, vocab, label, std, order, dtype):
    g = torch.Generator(device=DEV).manual_seed(3)
    z = torch.randn(rows, vocab, device=DEV, generator=g) * std
    labels = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    z.scatter_add_(1, labels[:, None], torch.randn(rows, 1, device=DEV, generator=g) * 2 + label)
    if order is not None:
        z = z.sort(1, descending=order == "down").values
    return z.to(dtype), labels.int()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,label,std,order", [
    (4096, 32768, 6.0, 2.0, None),       # a model's
    (4096, 1021, 6.0, 2.0, None),
    (2048, 32768, 20.0, 2.0, None),      # likely labels: what is beside their term of 1 counts
    (2048, 32768, 0.0, 2.0, "up"),       # the running maximum rises all along the row
    (2048, 32768, 0.0, 2.0, "down"),
    (2048, 32768, 0.0, 0.1, None),       # all alike
    (2048, 32768, 0.0, 5.0, None),       # few that count
])
def test_errors_do_not_add_up(rows, vocab, label, std, order, dtype):
    """A pair of one row each has that row's log-probability, minus a reference to 24 bits of it, as its margin.

    A term is an exponential, a thread's sum is scaled by another where its maximum rises and by one more when threads are
    joined.  On average the hardware's are 2.2e-8 to 5.1e-8 too small and 3.6e-8 is put back: 1.5e-8 is left of each, 4.5e-8 of
    three.  By itself a term is off by up to 8e-8 as a rule; where a hundredth or less of the sum hangs on each, 1e-8 of it."""
    z, labels = _logits(rows, vocab, label, std, order, dtype)
    logp = torch.cat([orc.label_logp(a, b)[0] for a, b in zip(z.split(256), labels.split(256))])
    ref = logp.float()
    offs = torch.arange(rows + 1, device=DEV).repeat_interleave(2)[1:].int().contiguous()
    _, margin = ob.preference_loss_fwd_bwd(z, labels, ref, offs, beta=1.0)
    check_status()
    off = margin.double() - (logp - ref.double())
    assert abs(float(off.mean())) <= 4.5e-8, off.mean()
    assert float(off.square().mean().sqrt()) <= 5.5e-8, off.square().mean().sqrt()


@pytest.mark.parametrize("gap", [30.0, 60.0, 200.0])
def test_a_certain_label_is_no_more_than_certain(gap):
    """logp stays at or below 0, and is what the others leave of it."""
    z = torch.zeros(64, 32768, device=DEV)
    labels = torch.arange(64, dtype=torch.int32, device=DEV) * 511
    z.scatter_(1, labels.long()[:, None], gap)
    want, *_ = orc.label_logp(z, labels)
    logp, _ = ob.token_logp_fwd(z, labels)
    assert (logp <= 0).all()
    orc.close(logp, want, 2.0 ** -24 * (1 + want.abs()), "logp")
