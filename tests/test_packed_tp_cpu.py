"""Packed sequences with the model split: over two tensor-parallel ranks (threads with an in-process exchange) and over two
pipeline stages.  Loss and gradients are the whole model's."""
import threading

import torch

from shift_b200.engine import Engine
from shift_b200.models.qwen_moe import MoEConfig, Partition
from shift_b200.ops import packed
from test_tp_cpu import ThreadTP

ROPE = dict(rope_dim=48, rope_layout="interleaved", rope_scaling=packed.RotaryScaling("ramp", 4.0, 32))
OFFS, ROWS = [3, 40, 41, 70, 71, 120], 128                 # one sequence lies on both sides of the ranks' border


def _cfg():
    return MoEConfig(vocab=512, hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, experts=8, top_k=2, expert_ffn=256,
                     max_seq=256, **ROPE)


def _batch(cfg):
    g = torch.Generator().manual_seed(2)
    tok, lab = (torch.randint(0, cfg.vocab, (1, ROWS), generator=g, dtype=torch.int32) for _ in range(2))
    return tok, lab, packed.sequences(torch.tensor(OFFS, dtype=torch.int32), ROWS)


def _close(got, want, name):
    assert (got - want).abs().max() <= 2e-4 * max(1.0, float(want.abs().max())) + 1e-7, name


def test_two_tensor_parallel_ranks():
    torch.manual_seed(0)
    cfg, tp = _cfg(), 2
    tok, lab, seqs = _batch(cfg)
    full = Engine(cfg, "cpu", bucket_numel=1 << 20)
    want = float(full.forward_backward([(tok, lab, {"seqs": seqs})], 1, ROWS))
    D, hq, hkv, e_per = cfg.head_dim, cfg.heads // tp, cfg.kv_heads // tp, cfg.experts // tp

    def shard(name, w, t):
        if name.endswith("attn.qkv"):
            heads = w.view(cfg.heads + 2 * cfg.kv_heads, D, -1).split([cfg.heads, cfg.kv_heads, cfg.kv_heads])
            return torch.cat([h.chunk(tp)[t] for h in heads]).reshape(-1, w.shape[1])
        if name.endswith("attn.o"):
            return w.view(w.shape[0], tp, hq * D)[:, t]
        return w[t * e_per:(t + 1) * e_per] if name.endswith(("mlp.w1", "mlp.w2")) else w

    comm, engines, losses, errors = ThreadTP(tp), [None] * tp, [None] * tp, []

    def run(t):
        try:
            part = Partition(expert_lo=t * e_per, expert_hi=(t + 1) * e_per, tp_size=tp)
            eng = Engine(cfg, "cpu", part=part, bucket_numel=1 << 20, tp=comm.view(t))
            for name, w in full.store.model_state_dict().items():
                eng.store.w(name).copy_(shard(name, w, t))
            losses[t], engines[t] = float(eng.forward_backward([(tok, lab, {"seqs": seqs})], 1, ROWS)), eng
        except BaseException as e:  # pragma: no cover - surfaced below
            errors.append(e)
            comm.bar.abort()

    ranks = [threading.Thread(target=run, args=(t,)) for t in range(tp)]
    for r in ranks:
        r.start()
    for r in ranks:
        r.join(120)
    assert not errors, errors
    assert abs(sum(losses) - want) < 1e-4
    for name in full.store.model_state_dict():
        g = full.store.g(name)
        if name.endswith(("attn.qkv", "attn.o", "mlp.w1", "mlp.w2")):
            for t in range(tp):
                _close(engines[t].store.g(name), shard(name, g, t), name)
        else:
            _close(engines[0].store.g(name) + engines[1].store.g(name), g, name)


def test_two_pipeline_stages():
    """Every stage is given the sequences."""
    cfg = _cfg()
    tok, lab, seqs = _batch(cfg)
    full = Engine(cfg, "cpu", bucket_numel=1 << 20)
    want = float(full.forward_backward([(tok, lab, {"seqs": seqs})], 1, ROWS))
    stages = [Engine(cfg, "cpu", part=Partition(layer_hi=1, has_head=False), bucket_numel=1 << 20),
              Engine(cfg, "cpu", part=Partition(layer_lo=1, has_embed=False), bucket_numel=1 << 20)]
    weights = full.store.model_state_dict()
    for eng in stages:
        for name in eng.store.offsets:
            eng.store.w(name).copy_(weights[name])
        eng.store.zero_grad()
    hidden, _ = stages[0].model.forward(tok, None, None, 1, ROWS, loss_scale=1 / ROWS, seqs=seqs)
    _, loss = stages[1].model.forward(None, hidden, lab, 1, ROWS, loss_scale=1 / ROWS, seqs=seqs)
    stages[0].model.backward(stages[1].model.backward())
    assert abs(float(loss) / ROWS - want) < 1e-5
    for eng in stages:
        for name in eng.store.offsets:
            _close(eng.store.g(name), full.store.g(name), name)
