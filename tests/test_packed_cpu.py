"""Packed sequences, rotary positions and label log-probability losses on the CPU: the statements against 64 bits and
against differences, refusals, and the model that calls them."""
import math

import pytest
import torch

import packed_oracle as orc
from shift_b200.engine import Engine
from shift_b200.models.qwen_moe import MoEConfig
from shift_b200.ops import objectives as ob
from shift_b200.ops import packed


def _seqs(offs, rows):
    return packed.sequences(torch.tensor(offs, dtype=torch.int32), rows)


def test_sequences():
    s = _seqs([2, 5, 5, 3, 9], 8)
    assert s.start.tolist() == [1, 2, 2, 2, 2, 5, 5, 5] and s.pos.tolist() == [-1, -1, 0, 1, 2, 0, 1, 2]
    assert s.stop.tolist() == [0, 1, 5, 5, 5, 8, 8, 8] and s.ends.tolist() == [2, 8]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("scaling", [None, packed.RotaryScaling("linear", 4.0), packed.RotaryScaling("base", 8.0),
                                     packed.RotaryScaling("ramp", 16.0, 512), ("ramp", 8.0, 256, 16.0, 2.0, 1.5)])
def test_rotary(layout, scaling):
    plan = packed.Rotary(32, 1.0e4, rot_dim=24, layout=layout, scaling=scaling, device="cpu")
    x = torch.randn(9, 3 * 32 + 5)
    pos = torch.tensor([0, -1, 7, 2 ** 31 - 1, 5, 1000003, 3, 2, -2 ** 31], dtype=torch.int32)
    for inverse in (False, True):
        want = orc.rotary(x, pos, plan.freq, 3, 32, 24, layout, plan.magnitude, inverse)
        got = packed.rotary(x.clone(), pos, plan, 3, inverse=inverse)
        assert torch.allclose(got.double(), want, rtol=1e-6, atol=1e-6)
    # turns of the kernel's plan: the frequencies to 64 bits
    turns = torch.tensor([t % 2 ** 64 for t in plan.turns.tolist()], dtype=torch.float64) / 2.0 ** 64
    assert torch.allclose(turns * 2 * math.pi, plan.freq % (2 * math.pi), rtol=1e-12)


def test_scaled_frequencies():
    plain = packed.Rotary(64, 1.0e4, device="cpu").freq
    assert torch.allclose(packed.Rotary(64, 1.0e4, scaling=packed.RotaryScaling("linear", 8.0), device="cpu").freq, plain / 8)
    base = packed.Rotary(64, 1.0e4, scaling=packed.RotaryScaling("base", 8.0), device="cpu").freq
    assert base[0] == 1 and math.isclose(float(base[-1]), float(plain[-1]) / 8, rel_tol=1e-9)
    ramp = packed.Rotary(64, 1.0e4, scaling=packed.RotaryScaling("ramp", 8.0, 4096), device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(ramp.freq[turns > 33], plain[turns > 33]) and torch.allclose(ramp.freq[-1], plain[-1] / 8)
    assert (ramp.freq <= plain + 1e-12).all() and (ramp.freq >= plain / 8 - 1e-12).all()
    assert math.isclose(ramp.magnitude, 0.1 * math.log(8) + 1)


@pytest.mark.parametrize("offs,rows,Hq,Hkv", [([0, 1], 1, 1, 1), ([2, 7, 7, 20], 23, 4, 2), ([0, 0], 5, 2, 2)])
def test_attention(offs, rows, Hq, Hkv):
    D, seqs = 64, _seqs(offs, rows)
    qkv, do = torch.randn(rows, (Hq + 2 * Hkv) * D), torch.randn(rows, Hq * D)
    want = orc.attention(qkv, offs, Hq, Hkv, D, 0.2, do)
    o, lse = packed.attention_fwd(qkv, seqs, Hq, Hkv, D, 0.2)
    g = packed.attention_bwd(qkv, o, lse, do, seqs, Hq, Hkv, D, 0.2)
    assert torch.allclose(o.double(), want["o"], atol=1e-5) and torch.allclose(g.double(), want["dqkv"], atol=1e-4)
    assert torch.allclose(lse.double(), want["lse"], atol=1e-5)
    out, into = torch.full_like(o, 3.0), torch.full_like(qkv, 4.0)
    packed.attention_fwd(qkv, seqs, Hq, Hkv, D, 0.2, out=out)
    packed.attention_bwd(qkv, o, lse, do, seqs, Hq, Hkv, D, 0.2, out=into)
    live = seqs.pos >= 0
    assert torch.equal(out[live], o[live]) and (out[~live] == 3).all() and (into[~live] == 4).all()


def test_attention_gradient_against_differences():
    torch.manual_seed(1)
    D, rows, seqs = 64, 6, _seqs([0, 2, 6], 6)
    qkv, do = torch.randn(rows, 4 * D), torch.randn(rows, 2 * D)
    o, lse = packed.attention_fwd(qkv, seqs, 2, 1, D, 0.125)
    g = packed.attention_bwd(qkv, o, lse, do, seqs, 2, 1, D, 0.125)
    step = torch.randn_like(qkv)
    side = [float((orc.attention(qkv.double() + e * step.double(), [0, 2, 6], 2, 1, D, 0.125)["o"] * do).sum())
            for e in (1e-4, -1e-4)]
    assert math.isclose((side[0] - side[1]) / 2e-4, float((g * step).sum()), rel_tol=1e-4)


def _logits(rows=6, vocab=11, seed=0):
    g = torch.Generator().manual_seed(seed)
    labels = torch.tensor([0, 3, -100, 10, 11, 5], dtype=torch.int32)[:rows]
    return torch.randn(rows, vocab, generator=g), labels, g


def _by_differences(loss, z, grad):
    """grad against differences of loss(z) in 64 bits along a random direction."""
    step = torch.randn(z.shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
    a, b = (float(loss(z.double() + e * step)) for e in (1e-5, -1e-5))
    assert math.isclose((a - b) / 2e-5, float((grad.double() * step).sum()), rel_tol=1e-4, abs_tol=1e-7)


def test_token_logp():
    z, labels, g = _logits()
    d = torch.randn(6, generator=g)
    logp, lse = ob.token_logp_fwd(z, labels)
    want, want_lse, live, _ = orc.label_logp(z, labels)
    assert torch.allclose(logp.double(), want, atol=1e-6) and torch.allclose(lse.double(), want_lse, atol=1e-6)
    assert live.tolist() == [True, True, False, True, False, True]
    grad = ob.token_logp_bwd(z.clone(), labels, lse, d)
    _by_differences(lambda x: (orc.label_logp(x, labels)[0] * d).sum(), z, grad)


def test_policy_loss():
    z, labels, g = _logits(seed=3)
    base, *_ = orc.label_logp(z, labels)
    old = (base + torch.tensor([0.1, -0.5, 0.0, 0.5, 0.0, -0.1])).float()
    ref, adv, w = (base + 0.2).float(), torch.tensor([1.0, 2.0, 1.0, -1.0, 1.0, 0.0]), torch.rand(6, generator=g)

    def loss(x):
        logp, _, live, _ = orc.label_logp(x, labels)
        r = torch.exp(logp - old.double())
        per = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv) + 0.1 * (torch.exp(ref - logp) - (ref - logp) - 1)
        return (per * live * w).sum() * 0.5

    grad = z.clone()
    per, logp = ob.policy_loss_fwd_bwd(grad, labels, old, adv, ref_logp=ref, kl_coef=0.1, scale=0.5, weight=w)
    assert math.isclose(float((per * w).sum() * 0.5), float(loss(z.double())), rel_tol=1e-5)
    _by_differences(loss, z, grad)
    assert not grad[2].any() and not grad[4].any()


def test_preference_loss():
    z, labels, _ = _logits(seed=4)
    base, *_ = orc.label_logp(z, labels)
    ref = (base + torch.tensor([0.3, -0.2, 9.0, 0.1, 9.0, -0.4])).float()
    offs = torch.tensor([0, 2, 3, 4, 6], dtype=torch.int32)

    def loss(x):
        logp, _, live, _ = orc.label_logp(x, labels)
        gap = (logp - ref.double()) * live
        s = [gap[a:b].sum() for a, b in zip([0, 2, 3, 4], [2, 3, 4, 6])]
        return -0.25 * (torch.nn.functional.logsigmoid(0.3 * (s[0] - s[1])) + torch.nn.functional.logsigmoid(0.3 * (s[2] - s[3])))

    grad = z.clone()
    per, margin = ob.preference_loss_fwd_bwd(grad, labels, ref, offs, beta=0.3, scale=0.25)
    assert per.shape == margin.shape == (2,) and math.isclose(float(per.sum() * 0.25), float(loss(z.double())), rel_tol=1e-5)
    _by_differences(loss, z, grad)


# ----------------------------------------------------------------------------- refusals
def test_refusals():
    seqs, z, labels, _ = _seqs([0, 4], 4), *_logits()
    none = torch.zeros(6)
    cases = [
        lambda: packed.sequences(torch.tensor([0, 4]), 4),
        lambda: packed.sequences(torch.tensor([0], dtype=torch.int32), 4),
        lambda: packed.sequences(torch.tensor([0, 4], dtype=torch.int32), -1),
        lambda: packed.Rotary(64, rot_dim=7, device="cpu"),
        lambda: packed.Rotary(64, rot_dim=66, device="cpu"),
        lambda: packed.Rotary(64, layout="other", device="cpu"),
        lambda: packed.Rotary(64, theta=0.0, device="cpu"),
        lambda: packed.Rotary(64, scaling=packed.RotaryScaling("other", 2.0), device="cpu"),
        lambda: packed.Rotary(64, scaling=packed.RotaryScaling("linear", 0.0), device="cpu"),
        lambda: packed.Rotary(64, scaling=packed.RotaryScaling("ramp", 2.0), device="cpu"),
        lambda: packed.Rotary(2, scaling=packed.RotaryScaling("base", 2.0), device="cpu"),
        lambda: packed.rotary(torch.zeros(4, 64), seqs.pos, packed.Rotary(64, device="cpu"), 2),
        lambda: packed.rotary(torch.zeros(4, 64), seqs.pos.long(), packed.Rotary(64, device="cpu"), 1),
        lambda: packed.rotary(torch.zeros(4, 64).double(), seqs.pos, packed.Rotary(64, device="cpu"), 1),
        lambda: packed.attention_fwd(torch.zeros(4, 3 * 64), seqs, 1, 1, 32, 1.0),
        lambda: packed.attention_fwd(torch.zeros(4, 5 * 64), seqs, 3, 2, 64, 1.0),
        lambda: packed.attention_fwd(torch.zeros(5, 3 * 64), seqs, 1, 1, 64, 1.0),
        lambda: packed.attention_fwd(torch.zeros(4, 3 * 64), seqs, 1, 1, 64, 1.0, out=torch.zeros(4, 32)),
        lambda: ob.token_logp_fwd(z.double(), labels),
        lambda: ob.token_logp_fwd(z, labels.long()),
        lambda: ob.token_logp_bwd(z, labels, none[:5], none),
        lambda: ob.policy_loss_fwd_bwd(z, labels, none, none, kl_coef=0.1),
        lambda: ob.policy_loss_fwd_bwd(z, labels, none, none, clip_low=-0.1),
        lambda: ob.preference_loss_fwd_bwd(z, labels, none, torch.tensor([0, 3], dtype=torch.int32)),
        lambda: ob.preference_loss_fwd_bwd(z, labels, none, torch.tensor([0, 3, 4])),
    ]
    for k, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {k} was not refused")


# ----------------------------------------------------------------------------- the model
CFG = dict(vocab=64, hidden=64, layers=2, heads=2, kv_heads=1, head_dim=32, experts=4, top_k=2, expert_ffn=32, max_seq=64)


def _grads(eng, batches, B, S):
    loss = eng.forward_backward(batches, B, S)
    return float(loss), eng.store.grad.clone()


def test_equal_sequences_packed_are_the_batch(monkeypatch):
    """Sequences of one length give what the batch of that shape gives."""
    cfg = MoEConfig(**{**CFG, "head_dim": 64})
    eng = Engine(cfg, "cpu", bucket_numel=1 << 16)
    tok = torch.randint(0, 64, (2, 8), dtype=torch.int32)
    lab = torch.randint(0, 64, (2, 8), dtype=torch.int32)
    loss, grad = _grads(eng, [(tok, lab)], 2, 8)
    both = _grads(eng, [(tok, lab, {"seqs": _seqs([0, 8, 16], 16)})], 2, 8)
    assert math.isclose(loss, both[0], rel_tol=1e-6) and torch.allclose(grad, both[1], rtol=1e-4, atol=1e-7)


def test_packed_model_sees_each_sequence_alone():
    """Without the router's shared load, a packed batch's gradient is the sum of its sequences' own."""
    cfg = MoEConfig(**{**CFG, "head_dim": 64, "aux_coef": 0.0, "rope_layout": "interleaved", "rope_dim": 32,
                       "rope_scaling": packed.RotaryScaling("ramp", 4.0, 16)})
    eng = Engine(cfg, "cpu", bucket_numel=1 << 16)
    tok = torch.randint(0, 64, (1, 14), dtype=torch.int32)
    lab = torch.randint(0, 64, (1, 14), dtype=torch.int32)
    lab[0, 11:] = -100                                     # rows of no sequence
    loss, grad = _grads(eng, [(tok, lab, {"seqs": _seqs([0, 4, 5, 11], 14)})], 1, 14)
    total, parts = 0.0, torch.zeros_like(grad)
    for a, b in ((0, 4), (4, 5), (5, 11)):
        one, g = _grads(eng, [(tok[:, a:b].contiguous(), lab[:, a:b].contiguous())], 1, b - a)
        total, parts = total + one * (b - a) / 14, parts + g * ((b - a) / 14)
    assert math.isclose(loss, total, rel_tol=1e-5) and torch.allclose(grad, parts, rtol=1e-4, atol=1e-7)


def test_model_takes_an_objective():
    cfg = MoEConfig(**{**CFG, "head_dim": 64, "aux_coef": 0.0})
    eng = Engine(cfg, "cpu", bucket_numel=1 << 16)
    tok = torch.randint(0, 64, (1, 12), dtype=torch.int32)
    lab = torch.randint(0, 64, (1, 12), dtype=torch.int32)
    seqs = _seqs([0, 5, 12], 12)
    # a policy loss at ratio 1 and unit advantages has the gradient of cross entropy
    want = _grads(eng, [(tok, lab, {"seqs": seqs})], 1, 12)[1]
    held = {}

    def objective(logits, labels):
        held["logp"], _ = ob.token_logp_fwd(logits, labels)
        return ob.policy_loss_fwd_bwd(logits, labels, held["logp"], torch.ones(12), scale=1 / 12)[0]

    loss, grad = _grads(eng, [(tok, lab, {"seqs": seqs, "objective": objective})], 1, 12)
    assert math.isclose(loss, -1.0, rel_tol=1e-5) and torch.allclose(grad, want, rtol=1e-3, atol=1e-7)
    pair = lambda logits, labels: ob.preference_loss_fwd_bwd(logits, labels, held["logp"], seqs.offs, beta=0.5)[0]  # noqa: E731
    loss, grad = _grads(eng, [(tok, lab, {"seqs": seqs, "objective": pair})], 1, 12)
    assert math.isclose(loss * 12, math.log(2.0), rel_tol=1e-5) and torch.isfinite(grad).all() and grad.any()
    with pytest.raises(ValueError, match="16 rows"):
        eng.forward_backward([(tok, lab, {"seqs": _seqs([0, 16], 16)})], 1, 12)


@pytest.mark.parametrize("kind", ["linear", "base", "ramp"])
@pytest.mark.parametrize("magnitude", [0.0, 1.0, 2.5])
def test_a_given_magnitude_is_taken(kind, magnitude):
    scaling = packed.RotaryScaling(kind, 8.0, 4096, magnitude=magnitude)
    plan = packed.Rotary(64, 1.0e4, scaling=scaling, device="cpu")
    assert plan.magnitude == magnitude
    x = torch.randn(3, 64)
    turned = packed.rotary(x.clone(), torch.tensor([0, 1, 5], dtype=torch.int32), plan, 1)
    assert torch.allclose(turned.norm(dim=1), magnitude * x.norm(dim=1), atol=1e-5)
