"""Losses of label log-probabilities on the GPU: vocabularies whose slice fills shared memory to the limit without opt-in, each
as the first call of a process."""
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
