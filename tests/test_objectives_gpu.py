"""Losses of label log-probabilities on the GPU against 64 bits."""
import math

import pytest
import torch

import packed_oracle as orc
from shift_b200.ops import objectives as ob

pytestmark = pytest.mark.gpu
DEV = "cuda"
# A term of a row's sum is an exponential (2^-22, and the rounding of its argument), scaled by another one each time its
# thread's running maximum rises and once when the threads' sums are joined: at most ten of them with fp32 roundings of 2^-24
# between, less than 2^-18.5 of the sum, so of lse and logp in absolute terms.
SUM = 2.0 ** -18.5
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [(1, 1), (3, 7), (5, 64), (2, 1021), (17, 4096), (1, 32768), (200, 2056), (3, 100003), (2, 262144), (149, 9)]


def _inputs(rows, vocab, dtype, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(rows, vocab + pad, generator=g).mul_(2)
    labels = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    wide[torch.arange(rows), labels.long()] += 5
    labels[2::5] = -100
    labels[4::11] = vocab                                  # no label either
    z = wide.to(dtype).to(DEV)[:, :vocab]
    return z, labels.to(DEV), g


def _rows(g, rows, std=1.0):
    return (torch.randn(rows, generator=g) * std).to(DEV)


def _grad_close(got, want, d, dtype, off=None):
    """One rounding to the type; the softmax is off by the exponent's 2^-22 of its argument (up to some tens), the sum's
    and lse's 2^-22: 2^-17 of |d| softmax, and of d where the label's two parts cancel.  `off`: how far each row's d itself
    may be off, where it is a sum whose terms cancel; the row's values are off by as much of their share of d."""
    if off is not None:
        share = want.abs() / d.abs()[:, None].clamp(min=1e-300)
        off = off[:, None] * share
    tol = (0 if off is None else off) + torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -17 * (want.abs() + orc.tiny(torch.float32)) + orc.tiny(dtype)
    label = want.abs().argmax(1)
    tol = tol.scatter_add(1, label[:, None], 2.0 ** -17 * d.double().abs()[:, None])
    orc.close(got, want, tol, "dlogits")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_token_logp(rows, vocab, dtype):
    for pad in (0, 3, 8):
        z, labels, g = _inputs(rows, vocab, dtype, pad=pad)
        logp, lse, live, _ = orc.label_logp(z, labels)
        got = ob.token_logp_fwd(z, labels)
        orc.close(got[0], logp, SUM + 2.0 ** -23 * logp.abs(), "logp")
        orc.close(got[1], lse, SUM + 2.0 ** -23 * lse.abs(), "lse")
        assert not got[0][~live].any()
        d = _rows(g, rows)
        want = orc.logits_grad(z, labels, d)
        assert ob.token_logp_bwd(z, labels, got[1], d) is z
        _grad_close(z, want, d, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_policy_loss(rows, vocab, dtype):
    for pad, ref, kl, weighted in ((0, True, 0.05, False), (3, False, 0.0, True), (8, True, 0.1, True)):
        z, labels, g = _inputs(rows, vocab, dtype, seed=1, pad=pad)
        logp, _, live, _ = orc.label_logp(z, labels)
        old, adv = (logp + _rows(g, rows, 0.3)).float(), _rows(g, rows)
        adv[1::7] = 0
        r = (logp + _rows(g, rows, 0.3)).float() if ref else None
        w = _rows(g, rows).abs() if weighted else None
        ratio = torch.exp(logp - old.double())
        gain, cut = ratio * adv.double(), ratio.clamp(0.8, 1.3) * adv.double()
        loss, d = -torch.minimum(gain, cut), -torch.where(gain <= cut, gain, torch.zeros_like(gain))
        if ref:
            gap = r.double() - logp
            loss, d = loss + kl * (gap.exp() - gap - 1), d + kl * (1 - gap.exp())
        d = d * 0.25 if w is None else d * 0.25 * w.double()
        want = orc.logits_grad(z, labels, d)
        got = ob.policy_loss_fwd_bwd(z, labels, old, adv, ref_logp=r, clip_low=0.2, clip_high=0.3, kl_coef=kl, scale=0.25,
                                     weight=w)
        orc.close(got[1], logp, SUM + 2.0 ** -23 * logp.abs(), "logp")
        # the ratio is off by as much, relative
        tol = 2 * SUM * (1 + (ratio * adv.double()).abs()) + 2.0 ** -24 * loss.abs()
        orc.close(got[0], torch.where(live, loss, torch.zeros_like(loss)), tol, "loss")
        # a row whose ratio lies within that of the clip's border may fall on either side of it
        edge = torch.where(adv >= 0, 1.3, 0.8).double()
        sure = (ratio - edge).abs() > 1e-5
        # d = (term of the ratio) + (term of the KL), each off by 2 SUM of the exponentials in it
        parts = (ratio * adv.double()).abs() + (kl * (1 + gap.exp()) if ref else 0)
        off = 2 * SUM * parts * 0.25 * (1 if w is None else w.double())
        _grad_close(z[sure], want[sure], (d * live)[sure], dtype, off[sure])


def _pairs(offs, rows):
    b = orc.cut(offs, rows)
    return [(slice(b[i], b[i + 1]), slice(b[i + 1], b[i + 2])) for i in range(0, len(b) - 1, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offs,rows,vocab", [([0, 1, 2], 2, 5), ([0, 3, 9], 9, 1000), ([4, 60, 90, 90, 200], 230, 1021),
                                             ([0, 0, 0], 4, 64), ([0, 300, 800, 900, 1500], 1500, 520), ([5, 2, 9], 7, 33)])
def test_preference_loss(offs, rows, vocab, dtype):
    z, labels, g = _inputs(rows, vocab, dtype, seed=2)
    logp, _, live, _ = orc.label_logp(z, labels)
    ref = (logp + _rows(g, rows, 0.4)).float()
    gap = torch.where(live, logp - ref.double(), torch.zeros_like(logp))
    beta, scale = 0.2, 0.5
    d, loss, margin, room = torch.zeros_like(logp), [], [], []
    for won, lost in _pairs(offs, rows):
        h = beta * (gap[won].sum() - gap[lost].sum())
        margin.append(h)
        loss.append(torch.nn.functional.softplus(-h))
        room.append(beta * sum(float((SUM + 2.0 ** -23 * logp[s].abs()).sum()) for s in (won, lost)) + 1e-7)
        d[won], d[lost] = -beta * scale * torch.sigmoid(-h), beta * scale * torch.sigmoid(-h)
    want = orc.logits_grad(z, labels, d)
    got = ob.preference_loss_fwd_bwd(z, labels, ref, torch.tensor(offs, dtype=torch.int32, device=DEV), beta=beta, scale=scale)
    for a, b, name in ((got[0], loss, "loss"), (got[1], margin, "margin")):
        b = torch.stack(b)
        orc.close(a, b, torch.tensor(room, device=DEV).double() + 2.0 ** -23 * b.abs(), name)
    _grad_close(z, want, d * (1 + 64 * max(room)), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(dtype):
    z, labels, g = _inputs(40, 3001, dtype, seed=3)
    z[0], z[1, 5], z[3, 7], z[5, :] = math.nan, math.nan, math.inf, -math.inf
    z[6, 1:] = -math.inf                                   # one value left
    z[8, :3000] = torch.finfo(dtype).min
    z[10, ::2] = -math.inf
    labels[:11] = torch.tensor([1, 2, -100, 4, -1, 3, 0, 1, 3000, 2, 1], dtype=torch.int32)
    z[2], z[4] = math.nan, math.inf                        # rows without a label
    logp, lse, live, _ = orc.label_logp(z, labels)
    got = ob.token_logp_fwd(z, labels)
    orc.close(got[0], logp, 2.0 ** -20 * (1 + logp.abs().nan_to_num(posinf=0)), "logp")
    orc.close(got[1], lse, 2.0 ** -20 * (1 + lse.abs().nan_to_num(posinf=0)), "lse")
    d = torch.ones(40, device=DEV)
    want = orc.logits_grad(z, labels, d)
    old, keep = logp.float().nan_to_num(0, 0, 0), z.clone()
    ob.token_logp_bwd(z, labels, got[1], d)
    assert not z[2].any() and not z[4].any()
    rest = torch.tensor([i for i in range(40) if i not in (0, 1, 3, 5)], device=DEV)
    _grad_close(z[rest], want[rest], d[rest], dtype)
    assert torch.isnan(z[[0, 1, 5]]).all() and torch.isnan(z[3, 7])
    adv = torch.ones(40, device=DEV)
    loss, _ = ob.policy_loss_fwd_bwd(keep, labels, old, adv, clip_low=0.5, clip_high=0.5)
    assert torch.isnan(loss[[0, 1, 5]]).all() and not loss[[2, 4]].any() and not keep[2].any() and not keep[4].any()
    assert torch.isfinite(keep[rest]).all()


def test_clip_decides_whole_rows():
    z = torch.zeros(6, 8, device=DEV)
    labels = torch.zeros(6, dtype=torch.int32, device=DEV)
    logp = torch.full((6,), -math.log(8.0), device=DEV)
    step = torch.tensor([0.3, 0.3, -0.3, -0.3, 0.1, 50.0], device=DEV)     # log ratios
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 2.0, 0.0], device=DEV)
    loss, _ = ob.policy_loss_fwd_bwd(z, labels, logp - step, adv, clip_low=0.2, clip_high=0.2)
    want = torch.tensor([-1.2, math.exp(0.3), -math.exp(-0.3), 0.8, -2 * math.exp(0.1), 0.0], device=DEV)
    assert torch.allclose(loss, want, rtol=1e-5, atol=1e-6)
    assert [bool(r.any()) for r in z] == [False, True, True, False, True, False]


def test_empty():
    z = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16)
    none = torch.empty(0, device=DEV)
    labels = torch.empty(0, dtype=torch.int32, device=DEV)
    assert [t.numel() for t in ob.token_logp_fwd(z, labels)] == [0, 0]
    ob.token_logp_bwd(z, labels, none, none)
    assert ob.policy_loss_fwd_bwd(z, labels, none, none)[0].numel() == 0
    loss, margin = ob.preference_loss_fwd_bwd(z, labels, none, torch.zeros(5, dtype=torch.int32, device=DEV))
    assert torch.allclose(loss, torch.full((2,), math.log(2.0), device=DEV)) and not margin.any()
