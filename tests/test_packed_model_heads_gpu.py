"""The model with heads of 128 on packed sequences, against the CPU's fp32 statement of the same step."""
import pytest
import torch

from shift_b200.engine import Engine
from shift_b200.models.qwen_moe import MoEConfig
from shift_b200.ops import packed
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rope", [dict(), dict(rope_dim=96, rope_layout="interleaved",
                                               rope_scaling=packed.RotaryScaling("ramp", 8.0, 64))])
def test_heads_of_128(rope):
    cfg = MoEConfig(vocab=1024, hidden=256, layers=2, heads=4, kv_heads=2, head_dim=128, experts=8, top_k=2, expert_ffn=256,
                    max_seq=512, **rope)
    T, offs = 300, [5, 70, 71, 200, 290]
    gpu, cpu = Engine(cfg, "cuda", bucket_numel=1 << 20), Engine(cfg, "cpu", bucket_numel=1 << 20)
    for name, w in gpu.store.model_state_dict().items():
        cpu.store.w(name).copy_(w.float().cpu())
    g = torch.Generator().manual_seed(1)
    tok, lab = (torch.randint(0, 1024, (1, T), generator=g, dtype=torch.int32) for _ in range(2))
    losses = []
    for eng, d in ((gpu, "cuda"), (cpu, "cpu")):
        more = {"seqs": packed.sequences(torch.tensor(offs, dtype=torch.int32, device=d), T)}
        losses.append(float(eng.forward_backward([(tok.to(d), lab.to(d), more)], 1, T)))
    check_status()
    assert abs(losses[0] - losses[1]) < 2e-2 * max(1.0, abs(losses[1])), losses
    for name in ("layers.0.attn.qkv", "layers.1.attn.o", "layers.0.mlp.w1", "lm_head.weight", "embed.weight"):
        a, b = gpu.store.g(name).float().cpu().reshape(-1), cpu.store.g(name).reshape(-1)
        assert float(torch.dot(a, b) / (a.norm() * b.norm() + 1e-12)) > 0.98, name
