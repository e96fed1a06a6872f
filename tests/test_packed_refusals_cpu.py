"""What the packed-sequence operators refuse on the GPU they refuse on the CPU."""
import math

import pytest
import torch

from shift_b200.ops import packed

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_attention(device):
    dtype = torch.bfloat16
    seqs = packed.sequences(torch.tensor([0, 5, 9], dtype=torch.int32, device=device), 9)
    qkv, o = torch.zeros(9, 4 * 64, dtype=dtype, device=device), torch.zeros(9, 2 * 64, dtype=dtype, device=device)
    lse = torch.zeros(2, 9, device=device)
    bad = [lambda s=s: packed.attention_fwd(qkv, seqs, 2, 1, 64, s) for s in (0.0, -1.0, math.nan, math.inf)]
    bad += [lambda s=s: packed.attention_bwd(qkv, o, lse, o, seqs, 2, 1, 64, s) for s in (0.0, -1.0, math.nan, math.inf)]
    bad += [
        lambda: packed.attention_fwd(qkv.double(), seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(qkv.int(), seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_bwd(qkv, o, lse[:1], o, seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_bwd(qkv, o, lse.half(), o, seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_bwd(qkv, o, lse, o.half(), seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_bwd(qkv, o.half(), lse, o, seqs, 2, 1, 64, 1.0),
        lambda: packed.attention_fwd(qkv, seqs, 2, 1, 64, 1.0, out=qkv[:, 64:192]),
        lambda: packed.attention_bwd(qkv, o, lse, o, seqs, 2, 1, 64, 1.0, out=qkv),
    ]
    for k, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"case {k} was not refused")
    packed.attention_bwd(qkv, *packed.attention_fwd(qkv, seqs, 2, 1, 64, 1.0), o, seqs, 2, 1, 64, 1.0)


@pytest.mark.parametrize("device", DEVICES)
def test_rotary(device):
    x, pos, plan = torch.randn(9, 192, device=device), torch.zeros(9, dtype=torch.int32, device=device), packed.Rotary(64, device=device)
    bad = [
        lambda: packed.rotary(x[:, :128], pos, plan, 1, out=x[:, 64:192]),
        lambda: packed.rotary(x[:1].expand(9, 192), pos, plan, 1),
        lambda: packed.rotary(x, pos, plan, 1, out=x[:, :128].clone()[:8]),
        lambda: packed.rotary(x, pos, plan, -1),
    ]
    for k, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"case {k} was not refused")
    packed.rotary(x[:, :64], pos, plan, 1, out=x[:, 128:])          # columns of one buffer, side by side
