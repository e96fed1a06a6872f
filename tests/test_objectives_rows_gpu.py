"""Losses of label log-probabilities on the GPU: vocabularies whose slice fills shared memory to the limit without opt-in, each
as the first call of a process; rows behind 2^31 elements."""
import os
import subprocess
import sys

import pytest
import torch

import packed_oracle as orc
from shift_b200.ops import objectives as ob
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"
SUM = 2.0 ** -18.5                      # a row's log-sum-exp, absolute: ten exponentials of 2^-22 and fp32 roundings


def _policy_against_64_bits(dtype, vocab, rows=200):
    g = torch.Generator().manual_seed(vocab)
    z = torch.randn(rows, vocab, generator=g).to(dtype).to(DEV)
    labels = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32).to(DEV)
    want_logp, *_ = orc.label_logp(z, labels)
    old = (want_logp + torch.randn(rows, generator=g).to(DEV) * 0.3).float()
    ratio = torch.exp(want_logp - old.double())
    want = orc.logits_grad(z, labels, -ratio)
    loss, logp = ob.policy_loss_fwd_bwd(z, labels, old, torch.ones(rows, device=DEV), clip_low=10.0, clip_high=1e9)
    check_status()
    orc.close(logp, want_logp, SUM + 2.0 ** -23 * want_logp.abs(), "logp")
    orc.close(loss, -ratio, 2 * SUM * ratio + 2.0 ** -23 * ratio, "loss")
    # one rounding to the type; the ratio and the softmax are off by 2 SUM each, relative, and at the label two of them cancel
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 4 * SUM * want.abs() + orc.tiny(dtype) + orc.tiny(torch.float32)
    tol.scatter_add_(1, labels.long()[:, None], 4 * SUM * ratio[:, None])
    orc.close(z, want, tol, "dlogits")


# Slices of 49072 to 49152 bytes, of one CTA a row and of two
FIRST = [("bfloat16", 24528), ("bfloat16", 24575), ("float16", 49151), ("bfloat16", 49056), ("float32", 12280), ("float32", 24528)]


@pytest.mark.parametrize("dtype,vocab", FIRST)
def test_policy_loss_as_the_first_call(dtype, vocab):
    """An earlier, larger call of the same type must not be what makes this one launch."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = f"import torch, test_objectives_rows_gpu as t; t._policy_against_64_bits(torch.{dtype}, {vocab})"
    env = {**os.environ, "PYTHONPATH": os.pathsep.join([here, os.path.dirname(here)])}
    got = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]


def test_gradients_of_rows_behind_two_to_the_31():
    """What is written there, not only what is read: the last rows of 2.2e9 logits, and a row on each side of 2^31 elements."""
    rows, vocab = 17000, 131072
    at = torch.tensor([0, (1 << 31) // vocab - 1, (1 << 31) // vocab, rows - 2, rows - 1], device=DEV)
    g = torch.Generator().manual_seed(6)
    some = torch.randn(len(at), vocab, generator=g).to(torch.bfloat16).to(DEV)
    labels = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    labels[at] = torch.tensor([5, 9, 131071, 0, 77], dtype=torch.int32, device=DEV)
    z = torch.ones(rows, vocab, dtype=torch.bfloat16, device=DEV)
    d = torch.zeros(rows, device=DEV)
    d[at] = torch.tensor([1.5, -2.0, 0.5, 3.0, -1.0], device=DEV)
    want_logp, *_ = orc.label_logp(some, labels[at])

    def compare(got, d_at, slack):
        want = orc.logits_grad(some, labels[at], d_at)
        tol = (torch.finfo(torch.bfloat16).eps / 2 + slack) * want.abs() + orc.tiny(torch.bfloat16) + orc.tiny(torch.float32)
        tol.scatter_add_(1, labels[at].long()[:, None], slack * d_at.double().abs()[:, None])
        orc.close(got[at], want, tol, "dlogits")
        assert int(torch.count_nonzero(got.view(torch.int16).view(rows, -1).any(1))) == len(at)      # the others are zeros

    z[at] = some
    logp, lse = ob.token_logp_fwd(z, labels)
    orc.close(logp[at], want_logp, SUM + 2.0 ** -23 * want_logp.abs(), "logp")
    ob.token_logp_bwd(z, labels, lse, d)
    compare(z, d[at], 2 * SUM)
    z.fill_(1)
    z[at] = some
    old = torch.zeros(rows, device=DEV)
    old[at] = (want_logp + 0.1).float()
    adv = torch.zeros(rows, device=DEV)
    adv[at] = d[at]
    _, logp = ob.policy_loss_fwd_bwd(z, labels, old, adv, clip_low=10.0, clip_high=1e9)
    orc.close(logp[at], want_logp, SUM + 2.0 ** -23 * want_logp.abs(), "logp")
    compare(z, -torch.exp(want_logp - old[at].double()) * d[at].double(), 4 * SUM)
    check_status()


@pytest.mark.parametrize("shift", [0.0, 1000.0, -3000.0])
def test_preference_gradients_far_from_zero(shift):
    """fp32 logits that are all far from zero: a log-sum-exp near 1000 has steps of 6e-5, its softmax must not."""
    rows, vocab = 40, 3001
    g = torch.Generator().manual_seed(8)
    z = (torch.randn(rows, vocab, generator=g) * 2 + shift).to(DEV)
    labels = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32).to(DEV)
    logp, *_ = orc.label_logp(z, labels)
    ref = (logp + torch.randn(rows, generator=g).to(DEV) * 0.1).float()
    gap = logp - ref.double()
    h = 0.01 * (gap[:25].sum() - gap[25:].sum())
    d = torch.full((rows,), 0.01 * float(torch.sigmoid(-h)), dtype=torch.float64, device=DEV)
    d[:25] *= -1
    want = orc.logits_grad(z, labels, d)
    offs = torch.tensor([0, 25, 40], dtype=torch.int32, device=DEV)
    ob.preference_loss_fwd_bwd(z, labels, ref, offs, beta=0.01)
    # d: the margin is off by 0.01 SUM a row, and so is its sigmoid at most; softmax: SUM for the sum, 2^-20 for the difference
    # z - lse (up to some tens) and its exponential; at the label two parts cancel
    slack = 0.01 * rows * SUM + SUM + 2.0 ** -20
    tol = (slack + 2.0 ** -24) * want.abs() + orc.tiny(torch.float32)
    tol.scatter_add_(1, labels.long()[:, None], slack * d.abs()[:, None])
    orc.close(z, want, tol, "dlogits")
