"""Rows that no sequence covers take no part in the model's loss, whatever their labels say."""
import pytest
import torch

from shift_b200.engine import Engine
from shift_b200.models.qwen_moe import MoEConfig
from shift_b200.ops import objectives as ob
from shift_b200.ops import packed


def check(device):
    cfg = MoEConfig(vocab=1024, hidden=256, layers=1, heads=4, kv_heads=2, head_dim=64, experts=8, top_k=2, expert_ffn=256,
                    max_seq=64, aux_coef=0.0)
    eng = Engine(cfg, device, bucket_numel=1 << 20)
    g = torch.Generator().manual_seed(3)
    tok, lab = (torch.randint(0, 1024, (1, 24), generator=g, dtype=torch.int32).to(device) for _ in range(2))
    seqs = packed.sequences(torch.tensor([3, 9, 10, 20], dtype=torch.int32, device=device), 24)
    none = lab.clone()
    none[0, :3] = none[0, 20:] = -100
    seen = []

    def objective(logits, labels):
        seen.append(labels.clone())
        logp = torch.full((24,), -4.0, device=device)
        return ob.policy_loss_fwd_bwd(logits, labels, logp, torch.ones(24, device=device), scale=1 / 24)[0]

    for more in ({"seqs": seqs}, {"seqs": seqs, "objective": objective}):
        got = []
        for labels in (lab, none):
            got.append((float(eng.forward_backward([(tok, labels, more)], 1, 24)), eng.store.grad.clone()))
        assert got[0][0] == got[1][0] and torch.equal(got[0][1], got[1][1])
    assert all(torch.equal(s < 0, none[0] < 0) and torch.equal(s[3:20], lab[0, 3:20]) for s in seen) and len(seen) == 2
    assert (lab >= 0).all()                                # the caller's labels are left as they were


def test_rows_of_no_sequence():
    check("cpu")


@pytest.mark.gpu
def test_rows_of_no_sequence_gpu():
    check("cuda")
