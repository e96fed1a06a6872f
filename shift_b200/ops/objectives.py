"""Losses of label log-probabilities, from the logits.

With lse = log sum exp of a row's logits, logp = logits[label] - lse and
d = dL/dlogp, the gradient at the logits is d (onehot - softmax).

* ``token_logp_fwd`` / ``token_logp_bwd``  the log-probability of every row's
  label (a reference or behaviour policy's side), and its gradient for a loss
  of the caller's own
* ``policy_loss_fwd_bwd``      clipped ratio to the behaviour policy, with a KL
  term to a reference policy
* ``preference_loss_fwd_bwd``  pairs of packed sequences, chosen against
  rejected

They stand beside ``ops.functional.xent_fwd_bwd`` and are used like it: the
logits are overwritten by ``scale`` times the loss's gradient, per-row losses
come back unscaled.  Logits are bf16, fp16 or fp32 of any vocabulary and row
stride, labels int32; a row whose label is not in [0, vocabulary) has none:
its loss and log-probability are 0, and so is its gradient, whatever its logits
hold.  CPU tensors take the fp32 statements of ``ops.reference``.
"""
from __future__ import annotations

import torch

from . import reference as ref
from ._ext import ext, status_word


# The CUDA entry points check their arguments themselves (csrc/objectives_host.cpp); this is for CPU tensors.
def _check(logits, labels, who, **rows):
    if logits.dim() != 2 or logits.shape[1] < 1 or logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"{who}: logits [rows, vocabulary] in bf16, fp16 or fp32, got {tuple(logits.shape)} of "
                         f"{logits.dtype}")
    T = logits.shape[0]
    if labels.dtype != torch.int32 or tuple(labels.shape) != (T,) or labels.device != logits.device:
        raise ValueError(f"{who}: labels are int32 [{T}] beside the logits")
    for name, x in rows.items():
        if x is not None and (x.dtype != torch.float32 or tuple(x.shape) != (T,) or x.device != logits.device):
            raise ValueError(f"{who}: {name} is fp32 [{T}] beside the logits")


def token_logp_fwd(logits: torch.Tensor, labels: torch.Tensor):
    """(logp [T], lse [T]), fp32: the label's log-probability (0 without one) and every row's log-sum-exp."""
    if logits.is_cuda:
        return tuple(ext().token_logp_fwd(logits, labels))
    _check(logits, labels, "token_logp_fwd")
    lse = torch.logsumexp(logits.double(), 1)
    return ref.label_logp(logits, labels, lse).float(), lse.float()


def token_logp_bwd(logits: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor, dlogp: torch.Tensor) -> torch.Tensor:
    """Overwrites the logits of ``token_logp_fwd`` by dlogp (onehot - softmax), and returns them.  ``lse`` is fp32: where
    logits lie near 1000 it has steps of 6e-5, and half of one is in every softmax value."""
    if logits.is_cuda:
        ext().token_logp_bwd(logits, labels, lse, dlogp)
        return logits
    _check(logits, labels, "token_logp_bwd", lse=lse, dlogp=dlogp)
    return ref.label_logp_grad_(logits, labels, lse, dlogp)


def policy_loss_fwd_bwd(logits: torch.Tensor, labels: torch.Tensor, old_logp: torch.Tensor, adv: torch.Tensor,
                        ref_logp: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                        kl_coef: float = 0.0, scale: float = 1.0, weight: torch.Tensor | None = None):
    """(loss [T], logp [T]), fp32, of every labelled row, with r = exp(logp - old_logp):

    loss = -min(r adv, clip(r, 1 - clip_low, 1 + clip_high) adv) + kl_coef (exp(g) - g - 1),  g = ref_logp - logp

    The logits are overwritten by scale * weight * dloss/dlogits (``weight`` [T], default 1).  Where the clip binds, the
    first term has no gradient; on its border it still has.  A row of zero advantage has none, however
    large its ratio; a ratio of NaN makes loss and gradient NaN with any advantage."""
    if logits.is_cuda:
        return tuple(ext().policy_loss(logits, labels, old_logp, adv, ref_logp, weight, clip_low, clip_high, kl_coef,
                                       scale, status_word(logits.device)))
    who = "policy_loss_fwd_bwd"
    _check(logits, labels, who, old_logp=old_logp, adv=adv, ref_logp=ref_logp, weight=weight)
    if not (0 <= clip_low and 0 <= clip_high):
        raise ValueError(f"{who}: clipped to 1 - {clip_low}, 1 + {clip_high}")
    if kl_coef != 0 and ref_logp is None:
        raise ValueError(f"{who}: a KL term needs ref_logp")
    lse = torch.logsumexp(logits.double(), 1)
    logp = ref.label_logp(logits, labels, lse)
    loss, d = ref.policy_terms(logp, old_logp, adv, ref_logp, clip_low, clip_high, kl_coef)
    live = ref.has_label(labels, logits.shape[1])
    loss, d = (torch.where(live, t, torch.zeros_like(t)) for t in (loss, d))
    d = d * scale if weight is None else d * scale * weight
    ref.label_logp_grad_(logits, labels, lse, d)
    return loss.float(), logp.float()


def preference_loss_fwd_bwd(logits: torch.Tensor, labels: torch.Tensor, ref_logp: torch.Tensor, offs: torch.Tensor,
                            beta: float = 0.1, scale: float = 1.0):
    """(loss [P], margin [P]), fp32, of P pairs of packed sequences: 2 p is chosen, 2 p + 1 rejected.

    margin = beta (sum over the chosen of (logp - ref_logp) - the same over the rejected), over labelled rows;
    loss = -log sigmoid(margin).  ``offs``: int32 [2 P + 1] on the device, as for ``ops.packed.sequences``.  The logits are
    overwritten by scale * dloss/dlogits (zeros in rows of no pair)."""
    if logits.is_cuda:
        return tuple(ext().preference_loss(logits, labels, ref_logp, offs, beta, scale))
    who = "preference_loss_fwd_bwd"
    _check(logits, labels, who, ref_logp=ref_logp)
    if (offs.dtype != torch.int32 or offs.dim() != 1 or offs.numel() < 3 or offs.numel() % 2 == 0
            or offs.device != logits.device):
        raise ValueError(f"{who}: offs are int32 [2 pairs + 1] beside the logits")
    lse = torch.logsumexp(logits.double(), 1)
    gap = torch.where(ref.has_label(labels, logits.shape[1]), ref.label_logp(logits, labels, lse) - ref_logp.double(),
                      torch.zeros_like(lse))
    d, loss, margin = torch.zeros_like(lse), [], []
    segs = ref.segments(offs, logits.shape[0])
    for (a, b), (_, c) in zip(segs[0::2], segs[1::2]):
        h = beta * (gap[a:b].sum() - gap[b:c].sum())
        margin.append(h)
        loss.append(torch.nn.functional.softplus(-h))
        d[a:b] = -beta * scale * torch.sigmoid(-h)
        d[b:c] = beta * scale * torch.sigmoid(-h)
    ref.label_logp_grad_(logits, labels, lse, d)
    return torch.stack(loss).float(), torch.stack(margin).float()
