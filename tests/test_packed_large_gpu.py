"""Packed attention of heads of 64 and 128 with more tiles than the SMs take at once, against 64 bits: items behind a CTA's first
one, pairs of heads and tiles of 256 queries, both sides of the rule by which two groups share a tile's keys."""
import pytest
import torch

import packed_oracle as orc
from shift_b200.ops import packed
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _check(offs, rows, Hq, Hkv, D, dtype):
    qkv, do = _randn(rows, (Hq + 2 * Hkv) * D, seed=rows + Hq, dtype=dtype), _randn(rows, Hq * D, seed=rows, dtype=dtype)
    seqs = packed.sequences(torch.tensor(offs, dtype=torch.int32, device=DEV), rows)
    o, lse = packed.attention_fwd(qkv, seqs, Hq, Hkv, D, D ** -0.5)
    got = packed.attention_bwd(qkv, o, lse, do, seqs, Hq, Hkv, D, D ** -0.5)
    check_status()
    want = orc.attention(qkv, offs, Hq, Hkv, D, D ** -0.5, do)
    orc.close(o, want["o"], want["o_tol"], "o")
    orc.close(lse, want["lse"], 1e-5 * (1 + want["lse"].abs().nan_to_num(posinf=0)), "lse")
    for name, cols in (("dv", slice((Hq + Hkv) * D, None)), ("dk", slice(Hq * D, (Hq + Hkv) * D)), ("dq", slice(0, Hq * D))):
        orc.close(got[:, cols], want["dqkv"][:, cols], want["dqkv_tol"][:, cols], name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (8, 8), (9, 3), (16, 1)])
@pytest.mark.parametrize("offs,rows", [([0, 5000], 5000), ([3, 900, 901, 2048, 2048, 4990], 5003),
                                       (list(range(0, 5101, 100)), 5120)])
def test_many_tiles(offs, rows, Hq, Hkv, D, dtype):
    _check(offs, rows, Hq, Hkv, D, dtype)


@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (3, 3)])
def test_both_sides_of_the_shared_tiles(Hq, Hkv):
    most = 2 * torch.cuda.get_device_properties(0).multi_processor_count // Hq * 128       # rows, at which tiles are still shared
    for rows in (most, most + 1):
        _check([0, rows // 3, rows - 40], rows, Hq, Hkv, 64, torch.bfloat16)
