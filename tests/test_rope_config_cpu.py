"""Other statements of the model take the configuration's rotary positions too."""
import pytest
import torch

from shift_b200.engine import Engine
from shift_b200.models.eager_moe import EagerMoE
from shift_b200.models.qwen_moe import MoEConfig
from shift_b200.models.reference_model import reference_loss
from shift_b200.ops import packed

ROPES = [dict(), dict(rope_dim=32), dict(rope_layout="interleaved"),
         dict(rope_dim=48, rope_layout="interleaved", rope_scaling=packed.RotaryScaling("ramp", 4.0, 16)),
         dict(rope_scaling=packed.RotaryScaling("linear", 3.0)), dict(rope_scaling=("base", 4.0))]


def _cfg(rope):
    return MoEConfig(vocab=64, hidden=64, layers=2, heads=2, kv_heads=1, head_dim=64, experts=4, top_k=2, expert_ffn=32,
                     max_seq=64, **rope)


@pytest.mark.parametrize("rope", ROPES)
def test_oracle_of_the_model(rope):
    cfg = _cfg(rope)
    eng = Engine(cfg, "cpu", bucket_numel=1 << 16)
    g = torch.Generator().manual_seed(5)
    tok, lab = (torch.randint(0, 64, (2, 24), generator=g, dtype=torch.int32) for _ in range(2))
    for name, w in eng.store.model_state_dict().items():   # scores that tell one position from another
        if name.endswith("attn.qkv"):
            w.mul_(20)
            eng.store.w(name).copy_(w)
    got = float(eng.forward_backward([(tok, lab)], 2, 24))
    params = {k: v.clone().float().requires_grad_() for k, v in eng.store.model_state_dict().items()}
    loss = reference_loss(cfg, params, tok, lab, 2, 24, with_aux=False)
    loss_aux = reference_loss(cfg, params, tok, lab, 2, 24)
    assert abs(got - float(loss.detach())) < 1e-5
    loss_aux.backward()
    for name in ("layers.0.attn.qkv", "layers.1.attn.o", "embed.weight"):
        assert torch.allclose(eng.store.g(name).float(), params[name].grad, rtol=1e-3, atol=1e-6), name


@pytest.mark.parametrize("rope", ROPES[1:])
def test_stock_model_refuses_what_it_has_not(rope):
    with pytest.raises(ValueError, match="rotary"):
        EagerMoE(_cfg(rope))
    EagerMoE(_cfg({}))
