"""Packed-sequence operators as they are used: refusals, streams, graphs, large offsets, the model that calls them."""
import math

import pytest
import torch

import packed_oracle as orc
from shift_b200.engine import Engine
from shift_b200.models.qwen_moe import MoEConfig
from shift_b200.ops import objectives as ob
from shift_b200.ops import packed
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _offs(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _randn(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


# ----------------------------------------------------------------------------- refusals
def test_refusals():
    seqs = packed.sequences(_offs(0, 40), 40)
    qkv, o = _randn(40, 4 * 64), _randn(40, 2 * 64)
    lse = torch.zeros(2, 40, device=DEV)
    z, labels, row = _randn(6, 32), torch.zeros(6, dtype=torch.int32, device=DEV), torch.zeros(6, device=DEV)
    plan = packed.Rotary(64)
    bad = [
        lambda: packed.sequences(_offs(0, 4).long(), 4),
        lambda: packed.sequences(_offs(0), 4),
        lambda: packed.sequences(_offs(0, 1, 2, 3)[::2], 4),
        lambda: packed.sequences(_offs(0, 4), -1),
        lambda: packed.rotary(qkv, seqs.pos, plan, 5),
        lambda: packed.rotary(qkv, seqs.pos[:39], plan, 1),
        lambda: packed.rotary(qkv, seqs.pos.long(), plan, 1),
        lambda: packed.rotary(qkv, seqs.pos.cpu(), plan, 1),
        lambda: packed.rotary(qkv.double(), seqs.pos, plan, 1),
        lambda: packed.rotary(qkv, seqs.pos, plan, 1, out=o.float()),
        lambda: packed.rotary(qkv[:, :128], seqs.pos, plan, 1, out=qkv[:, 64:192]),
        lambda: packed.rotary(qkv[:1].expand(40, 256), seqs.pos, plan, 1),
        lambda: packed.rotary(qkv, seqs.pos, packed.Rotary(64, device="cpu"), 1),
        lambda: packed.attention_fwd(qkv, seqs, 2, 1, 32, 1.0),
        lambda: packed.attention_fwd(qkv, seqs, 3, 2, 64, 1.0),
        lambda: packed.attention_fwd(qkv, seqs, 2, 2, 64, 1.0),
        lambda: packed.attention_fwd(qkv[:39], seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(qkv.float(), seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(qkv, seqs, 2, 1, 64, 0.0),
        lambda: packed.attention_fwd(qkv, seqs, 2, 1, 64, math.nan),
        lambda: packed.attention_fwd(qkv, seqs, 2, 1, 64, -1.0),
        lambda: packed.attention_fwd(_randn(40, 260)[:, 2:258], seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(_randn(40, 258)[:, :256], seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(qkv[:1].expand(40, 256), seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(qkv, packed.Sequences(seqs.offs, seqs.plan[:100], 40), 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(qkv, packed.sequences(torch.tensor([0, 40], dtype=torch.int32), 40), 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(qkv, seqs, 2, 1, 64, 1.0, out=o.half()),
        lambda: packed.attention_fwd(qkv, seqs, 2, 1, 64, 1.0, out=o[:, :64]),
        lambda: packed.attention_bwd(qkv, o, lse[:1], o, seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_bwd(qkv, o, lse.half(), o, seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_bwd(qkv, o, lse, o[:, :64], seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_bwd(qkv, o, lse, o.half(), seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_bwd(qkv, o, lse, o, seqs, 2, 1, 64, 1.0, out=o),
        lambda: packed.attention_bwd(qkv, o, lse, o, seqs, 2, 1, 64, 1.0, out=qkv),
        lambda: packed.attention_fwd(qkv, seqs, 2, 1, 64, 1.0, out=qkv[:, 64:192]),
        lambda: ob.token_logp_fwd(z.double(), labels),
        lambda: ob.token_logp_fwd(z, labels.long()),
        lambda: ob.token_logp_fwd(z, labels[:5]),
        lambda: ob.token_logp_fwd(z, labels.cpu()),
        lambda: ob.token_logp_fwd(z.t(), labels),
        lambda: ob.token_logp_fwd(z[:1].expand(6, 32), labels),
        lambda: ob.token_logp_bwd(z, labels, row, row[:5]),
        lambda: ob.token_logp_bwd(z, labels, row.double(), row),
        lambda: ob.policy_loss_fwd_bwd(z, labels, row, row, kl_coef=0.1),
        lambda: ob.policy_loss_fwd_bwd(z, labels, row, row, clip_low=-0.1),
        lambda: ob.policy_loss_fwd_bwd(z, labels, row, row, weight=row.cpu()),
        lambda: ob.preference_loss_fwd_bwd(z, labels, row, _offs(0, 6)),
        lambda: ob.preference_loss_fwd_bwd(z, labels, row, _offs(0, 3, 6).long()),
    ]
    for k, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"case {k} was not refused")
    torch.cuda.synchronize()
    check_status()


def test_columns_of_one_buffer_side_by_side():
    """Views of a buffer's rows that lie next to each other are not refused as overlapping."""
    seqs = packed.sequences(_offs(0, 40, 90), 90)
    wide = _randn(90, 256 + 128 + 256)
    qkv, o, g = wide[:, :256], wide[:, 256:384], wide[:, 384:]
    do = _randn(90, 128, seed=1)
    want, lse = packed.attention_fwd(qkv.contiguous(), seqs, 2, 1, 64, 0.125)
    packed.attention_fwd(qkv, seqs, 2, 1, 64, 0.125, out=o)
    packed.attention_bwd(qkv, o, lse, do, seqs, 2, 1, 64, 0.125, out=g)
    assert torch.equal(o, want)
    assert torch.equal(g, packed.attention_bwd(qkv.contiguous(), want, lse, do, seqs, 2, 1, 64, 0.125))
    plan = packed.Rotary(64)
    packed.rotary(qkv, seqs.pos, plan, 3, out=g)
    assert torch.equal(g[:, :192], packed.rotary(qkv.clone(), seqs.pos, plan, 3)[:, :192])


# ----------------------------------------------------------------------------- streams and graphs
HEADS = (4, 2, 64, 0.125)


def _pass(offs, qkv, do, z, labels, old, adv):
    """One of each, in a user's order; `qkv` and `z` are consumed."""
    seqs = packed.sequences(offs, qkv.shape[0])
    plan = _pass.plan
    packed.rotary(qkv, seqs.pos, plan, 6)
    o, lse = packed.attention_fwd(qkv, seqs, *HEADS)
    g = packed.attention_bwd(qkv, o, lse, do, seqs, *HEADS)
    packed.rotary(g, seqs.pos, plan, 6, inverse=True)
    keep = z.clone()
    pol = ob.policy_loss_fwd_bwd(z, labels, old, adv, ref_logp=old, kl_coef=0.1)
    pre = ob.preference_loss_fwd_bwd(keep, labels, old, offs)
    return [o, lse, g, *pol, z, *pre, keep]


def _inputs(seed, rows=700, vocab=3001):
    g = torch.Generator().manual_seed(seed)
    labels = torch.randint(-20, vocab, (rows,), generator=g, dtype=torch.int32).to(DEV)
    return (_randn(rows, 8 * 64, seed=seed), _randn(rows, 4 * 64, seed=seed + 1), _randn(rows, vocab, seed=seed + 2), labels,
            torch.randn(rows, generator=g).to(DEV) - 8, torch.randn(rows, generator=g).to(DEV))


@pytest.fixture(autouse=True)
def _plan():
    _pass.plan = packed.Rotary(64, 1.0e4)


def _same(got, want):
    for k, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(torch.nan_to_num(a, neginf=-1e9), torch.nan_to_num(b, neginf=-1e9)), k


def test_two_streams_at_once():
    cases = [(_offs(0, 100, 433, 500, 640), _inputs(1)), (_offs(10, 11, 300, 690, 700), _inputs(5))]
    want = [_pass(o, *(t.clone() for t in x)) for o, x in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for k, (s, (o, x)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[k].append(_pass(o, *(t.clone() for t in x)))
    torch.cuda.synchronize()
    check_status()
    for k in (0, 1):
        for g in got[k]:
            _same(g, want[k])


def test_captured_and_replayed_with_other_offsets():
    static, fresh = [t.clone() for t in _inputs(2)], _inputs(2)
    offs = _offs(0, 100, 433, 500, 640)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _pass(offs, *static)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                     # two graphs of the same, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _pass(offs, *static)
        graphs.append((graph, out))
    for values in ((0, 100, 433, 500, 640), (3, 3, 650, 651, 700), (0, 1, 2, 3, 4), (0, 0, 0, 0, 0)):
        want = _pass(_offs(*values), *(t.clone() for t in fresh))
        for graph, out in graphs:
            offs.copy_(_offs(*values))
            for a, b in zip(static, fresh):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            _same(out, want)
    check_status()


def test_rows_behind_two_to_the_31():
    """Offsets in elements that pass 32 bits: the last rows of a long buffer, and of many logits."""
    rows, Hq, Hkv, D = 1500000, 4, 4, 128
    qkv = torch.zeros(rows, 12 * D, dtype=torch.bfloat16, device=DEV)
    tail, do = _randn(300, 12 * D, seed=3), torch.zeros(rows, Hq * D, dtype=torch.bfloat16, device=DEV)
    qkv[-300:], do[-300:] = tail, _randn(300, Hq * D, seed=4)
    seqs = packed.sequences(_offs(*range(0, rows - 300, 4000), rows - 300, rows - 100, rows), rows)
    o, lse = packed.attention_fwd(qkv, seqs, Hq, Hkv, D, 0.1)
    g = packed.attention_bwd(qkv, o, lse, do, seqs, Hq, Hkv, D, 0.1)
    check_status()
    want = orc.attention(tail, [0, 200, 300], Hq, Hkv, D, 0.1, do[-300:])
    orc.close(o[-300:], want["o"], want["o_tol"], "o")
    orc.close(g[-300:], want["dqkv"], want["dqkv_tol"], "dqkv")
    assert not o[:-300].any() and not g[:-300].any()
    assert abs(float(lse[0, 3999]) - math.log(4000.0)) < 1e-4
    packed.rotary(qkv, seqs.pos, packed.Rotary(D), 8)
    plan = packed.Rotary(D)
    turned = orc.rotary(tail, seqs.pos[-300:], plan.freq.to(DEV), 8, D, D, "half", 1.0, False)
    orc.close(qkv[-300:], turned, 2.0 ** -8 * turned.abs() + 2.0 ** -16, "rotary")
    del qkv, do, o, g
    rows, vocab = 17000, 131072
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=DEV)
    labels = torch.full((rows,), 5, dtype=torch.int32, device=DEV)
    z[-1] = _randn(vocab, seed=6)
    last = z[-1:].clone()
    want, *_ = orc.label_logp(last, labels[-1:])
    old, adv = torch.full((rows,), -11.7835, device=DEV), torch.ones(rows, device=DEV)
    loss, logp = ob.policy_loss_fwd_bwd(z, labels, old, adv, clip_low=10.0, clip_high=1e9)
    assert abs(float(logp[-1]) - float(want)) < 1e-5 and abs(float(logp[0]) + math.log(vocab)) < 1e-5
    assert abs(float(z[0, 5]) + math.exp(-math.log(vocab) + 11.7835)) < 1e-2 and float(z[-1].float().abs().max()) > 0


# ----------------------------------------------------------------------------- the model
def _cos(a, b):
    a, b = a.float().reshape(-1), b.float().reshape(-1)
    return float(torch.dot(a, b) / (a.norm() * b.norm() + 1e-12))


def test_model_on_packed_sequences():
    """Gradients on the GPU against the CPU's fp32 statement of the same packed step, with each objective."""
    cfg = MoEConfig(vocab=1024, hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, experts=8, top_k=2, expert_ffn=256,
                    max_seq=512, rope_dim=48, rope_layout="interleaved", rope_scaling=packed.RotaryScaling("ramp", 4.0, 64))
    gpu = Engine(cfg, "cuda", bucket_numel=1 << 20)
    cpu = Engine(cfg, "cpu", bucket_numel=1 << 20)
    for name, w in gpu.store.model_state_dict().items():
        cpu.store.w(name).copy_(w.float().cpu())
    T, offs = 300, [0, 70, 71, 200, 290]
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, 1024, (1, T), generator=g, dtype=torch.int32)
    lab = torch.randint(0, 1024, (1, T), generator=g, dtype=torch.int32)
    lab[0, ::9], lab[0, 290:] = -100, -100
    old, adv = torch.full((T,), -7.0), torch.randn(T, generator=g)
    objectives = [
        None,
        lambda d: lambda z, y: ob.policy_loss_fwd_bwd(z, y, old.to(d), adv.to(d), ref_logp=old.to(d), kl_coef=0.1,
                                                      scale=1 / T)[0],
        lambda d: lambda z, y: ob.preference_loss_fwd_bwd(z, y, old.to(d), torch.tensor(offs, dtype=torch.int32, device=d),
                                                          beta=0.05)[0],
    ]
    for make in objectives:
        losses = []
        for eng, d in ((gpu, "cuda"), (cpu, "cpu")):
            more = {"seqs": packed.sequences(torch.tensor(offs, dtype=torch.int32, device=d), T)}
            if make is not None:
                more["objective"] = make(d)
            losses.append(float(eng.forward_backward([(tok.to(d), lab.to(d), more)], 1, T)))
        check_status()
        assert abs(losses[0] - losses[1]) < 2e-2 * max(1.0, abs(losses[1])), losses
        for name in ("layers.0.attn.qkv", "layers.1.attn.o", "layers.0.mlp.w1", "layers.0.ln1.weight", "lm_head.weight",
                     "embed.weight"):
            c = _cos(gpu.store.g(name).float().cpu(), cpu.store.g(name))
            assert c > 0.98, (name, c)


def test_model_packed_equals_its_batch():
    """Sequences of one length through the packed operators and through the batched ones."""
    cfg = MoEConfig.tiny()
    eng = Engine(cfg, "cuda", bucket_numel=1 << 20)
    g = torch.Generator().manual_seed(3)
    tok, lab = (torch.randint(0, 1024, (4, 128), generator=g, dtype=torch.int32).cuda() for _ in range(2))
    a = float(eng.forward_backward([(tok, lab)], 4, 128))
    ga = eng.store.grad.float().clone()
    b = float(eng.forward_backward([(tok, lab, {"seqs": packed.sequences(_offs(0, 128, 256, 384, 512), 512)})], 4, 128))
    check_status()
    assert abs(a - b) < 1e-3 and _cos(ga, eng.store.grad) > 0.999
