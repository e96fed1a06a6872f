"""Policy loss of rows whose log-probability is NaN: nothing makes them look clean."""
import math

import pytest
import torch

from shift_b200.ops import objectives as ob


def check(device):
    z = torch.randn(6, 37, generator=torch.Generator().manual_seed(1))
    z[0, 5] = z[1, 0] = z[2, 36] = math.nan
    labels = torch.tensor([3, 4, -100, 6, 7, 8], dtype=torch.int32, device=device)
    old = torch.tensor([-3.0, -3.0, -3.0, -math.inf, math.nan, -200.0], device=device)
    adv = torch.tensor([0.0, 1.0, 0.0, 0.0, 0.0, 0.0], device=device)
    for kl in (0.0, 0.1):
        x = z.to(device, copy=True)
        ref = torch.full((6,), -3.0, device=device) if kl else None
        loss, logp = ob.policy_loss_fwd_bwd(x, labels, old, adv, ref_logp=ref, kl_coef=kl, clip_low=0.5, clip_high=0.5)
        assert torch.isnan(loss[[0, 1, 4]]).all() and torch.isnan(logp[[0, 1]]).all()
        assert torch.isnan(x[[0, 1, 4]]).all()
        assert not loss[2].any() and not x[2].any()        # without a label whatever it holds
        # an infinite ratio, or a huge one, and no advantage: nothing but the KL term
        assert torch.isfinite(loss[[3, 5]]).all() and torch.isfinite(x[[3, 5]]).all()
        assert kl != 0 or (not loss[[3, 5]].any() and not x[[3, 5]].any())


def test_rows_of_nan():
    check("cpu")


@pytest.mark.gpu
def test_rows_of_nan_gpu():
    check("cuda")
