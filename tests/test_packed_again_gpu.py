"""Packed attention where rows that are not finite meet others through masked zeros: what is computed again, row by row, comes
after a CTA's last tile and may take as long as it takes."""
import math

import pytest
import torch

import packed_oracle as orc
from shift_b200.ops import packed
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _step(qkv, do, offs, heads):
    seqs = packed.sequences(torch.tensor(offs, dtype=torch.int32, device=DEV), qkv.shape[0])
    o, lse = packed.attention_fwd(qkv, seqs, *heads)
    g = packed.attention_bwd(qkv, o, lse, do, seqs, *heads)
    check_status()
    return o, lse, g


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,rows", [(2, 2, 64, 900), (8, 1, 64, 900), (9, 3, 64, 5003), (8, 2, 64, 5003), (8, 8, 128, 2500),
                                           (8, 1, 128, 700), (3, 3, 128, 5003)])
def test_many_rows_of_many_tiles(Hq, Hkv, D, rows, dtype):
    """A short sequence with infinite values in every second tile: its neighbours in those tiles have their own results, in every
    form of the kernels (tiles shared by two groups, pairs of heads, 256 queries, groups dealt out over CTAs)."""
    heads, offs, loud = (Hq, Hkv, D, D ** -0.5), [0], torch.zeros(rows, dtype=torch.bool)
    for t in range(100, rows - 40, 256):
        offs += [t, t + 5]
        loud[t:t + 5] = True
    offs += [rows]
    qkv, do = _randn(rows, (Hq + 2 * Hkv) * D, seed=rows, dtype=dtype), _randn(rows, Hq * D, seed=rows + 1, dtype=dtype)
    qkv[loud.to(DEV)] = 0
    do[loud.to(DEV)] = 0
    want = orc.attention(qkv, offs, *heads, do)
    qkv[loud.to(DEV), 1::3] = math.inf
    do[loud.to(DEV), 2::3] = -math.inf
    o, lse, g = _step(qkv, do, offs, heads)
    quiet = (~loud).to(DEV)
    orc.close(o[quiet], want["o"][quiet], want["o_tol"][quiet], "o")
    orc.close(lse[:, quiet], want["lse"][:, quiet], 1e-5 * (1 + want["lse"][:, quiet].abs()), "lse")
    orc.close(g[quiet], want["dqkv"][quiet], want["dqkv_tol"][quiet], "dqkv")


@pytest.mark.parametrize("D", [64, 128])
def test_a_long_document_with_one_bad_row(D):
    """An infinite `do` at its beginning, infinite keys and values at its end: 117 rows of dV and 127 of O and dQ hang on some ten
    thousand rows each.  No wait runs out, every row is written, and those that saw nothing bad have what they had."""
    rows, Hq, Hkv = 24000, 8, 1
    heads = (Hq, Hkv, D, D ** -0.5)
    qkv, do = _randn(rows, (Hq + 2 * Hkv) * D, seed=1), _randn(rows, Hq * D, seed=2)
    first = _step(qkv, do, [0, rows], heads)
    sizes = _step(torch.cat([qkv[:, :Hq * D + D], qkv[:, Hq * D + D:].abs()], 1), do.abs(), [0, rows], heads)
    x, y = qkv.clone(), do.clone()
    y[10, 3::D] = math.inf
    x[-1, Hq * D:] = math.inf
    o, lse, g = _step(x, y, [0, rows], heads)
    kept = slice(0, rows - 1)
    half = 2.0 ** -8
    # both sides round their probabilities (or neither) and their results; sums of absolute values bound what that may be
    assert torch.equal(lse[:, kept], first[1][:, kept])
    assert ((o - first[0])[kept].abs() <= 2 * half * (sizes[0][kept].float() * 1.01 + first[0][kept].abs())).all()
    assert torch.isnan(o[-1]).all()
    tile, q = slice(rows // 128 * 128 if rows % 128 else rows - 128, rows - 1), slice(0, Hq * D)
    got, want = g[tile, q].double(), first[2][tile, q].double()      # roundings of dS and the result, of random sign
    assert (got - want).norm() <= 3 * half * want.norm() and torch.equal(g[11:tile.start, q], first[2][11:tile.start, q])
    dv = g[11:, (Hq + Hkv) * D:]
    want, room = first[2][11:, (Hq + Hkv) * D:], sizes[2][11:, (Hq + Hkv) * D:]
    # the last row has no probabilities any more, so it gives the values before it NaN; its own query sees every key
    assert torch.isnan(dv).all() and torch.isfinite(want).all() and torch.isfinite(room).all()
    # without the last row: the values behind row 10 have what they had
    x[-1] = qkv[-1]
    o, lse, g = _step(x, y, [0, rows], heads)
    dv = g[11:, (Hq + Hkv) * D:]
    assert ((dv - want).abs() <= 2 * half * (room.float() * 1.01 + want.abs())).all()
    assert torch.equal(g[128:], first[2][128:]) and torch.equal(o, first[0])
    assert not torch.isfinite(g[:11, (Hq + Hkv) * D + 3]).any()
