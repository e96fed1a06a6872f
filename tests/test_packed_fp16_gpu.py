"""fp16 gradients of packed attention: what scales them for one row is not seen by others, and probabilities of long rows count."""
import math

import pytest
import torch

import packed_oracle as orc
from shift_b200.ops import packed
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(*shape, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.float16).to(DEV)


def _step(qkv, do, offs, heads):
    seqs = packed.sequences(torch.tensor(offs, dtype=torch.int32, device=DEV), qkv.shape[0])
    o, lse = packed.attention_fwd(qkv, seqs, *heads)
    g = packed.attention_bwd(qkv, o, lse, do, seqs, *heads)
    check_status()
    return g


def _parts(heads):
    Hq, Hkv, D, _ = heads
    return slice(0, Hq * D), slice(Hq * D, (Hq + Hkv) * D), slice((Hq + Hkv) * D, None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (3, 3), (8, 1)])
@pytest.mark.parametrize("loud", [2.0 ** 10, 6e4])
def test_a_sequence_of_large_gradients_leaves_others_theirs(loud, Hq, Hkv, D):
    """Sequences of very different `do` in shared tiles: each has the bits that it has beside one without any."""
    heads, offs, rows = (Hq, Hkv, D, D ** -0.5), [2, 700, 760, 1500], 1503
    qkv, do = _randn(rows, (Hq + 2 * Hkv) * D, seed=1), _randn(rows, Hq * D, seed=2, std=2.0 ** -10)
    quiet = do.clone()
    quiet[700:760] = 0
    do[700:760] = (_randn(60, Hq * D, seed=3).float().clamp(-1, 1) * loud).half()
    got, want = _step(qkv, do, offs, heads), _step(qkv, quiet, offs, heads)
    for rows_ in (slice(0, 700), slice(760, rows)):
        assert torch.equal(got[rows_], want[rows_])
    exact = orc.attention(qkv, offs, *heads, quiet)["dqkv"]
    for cols in _parts(heads):                             # and they are there: three roundings of 2^-11, the result's step
        for rows_ in (slice(2, 700), slice(760, 1500)):
            w = exact[rows_, cols]
            assert (want[rows_, cols].double() - w).norm() <= 3 * 2.0 ** -11 * w.norm() + 2.0 ** -25 * w.numel() ** 0.5


@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_a_key_is_not_seen_by(D):
    """Large gradients of a sequence's first rows: keys behind them are seen by none of those rows."""
    heads, rows, first = (4, 2, D, D ** -0.5), 1300, 333
    qkv, do = _randn(rows, 8 * D, seed=4), _randn(rows, 4 * D, seed=5, std=2.0 ** -10)
    want = _step(qkv, do, [0, rows], heads)
    do[:first] *= 2.0 ** 12
    got = _step(qkv, do, [0, rows], heads)
    assert torch.equal(got[first:], want[first:])


@pytest.mark.parametrize("D", [64, 128])
def test_heads_of_other_keys(D):
    """Large gradients of one group's heads: the other group's gradients have the bits that they had."""
    heads, rows = (4, 2, D, D ** -0.5), 600
    qkv, do = _randn(rows, 8 * D, seed=6), _randn(rows, 4 * D, seed=7, std=2.0 ** -10)
    want = _step(qkv, do, [0, rows], heads).view(rows, 8, D)
    do[:, :2 * D] *= 2.0 ** 12
    got = _step(qkv, do, [0, rows], heads).view(rows, 8, D)
    for h in (2, 3, 5, 7):
        assert torch.equal(got[:, h], want[:, h])


@pytest.mark.parametrize("D", [64, 128])
def test_an_infinite_gradient_elsewhere(D):
    """One infinite `do`: rows of other sequences, and later rows of its own, keep their gradients."""
    heads, offs, rows = (4, 2, D, D ** -0.5), [0, 300, 900], 900
    qkv, do = _randn(rows, 8 * D, seed=8), _randn(rows, 4 * D, seed=9, std=2.0 ** -10)
    exact = orc.attention(qkv, offs, *heads, do)
    do[350, 3] = math.inf
    got = _step(qkv, do, offs, heads)
    for rows_ in (slice(0, 300), slice(351, 900)):
        for cols in _parts(heads):
            w = exact["dqkv"][rows_, cols]
            assert (got[rows_, cols].double() - w).norm() <= 3 * 2.0 ** -11 * w.norm() + 2.0 ** -25 * w.numel() ** 0.5
    assert not torch.isfinite(got[350, :D]).any() and not torch.isfinite(got[300:351, 4 * D:5 * D]).any()


@pytest.mark.parametrize("D", [64, 128])
def test_probabilities_below_what_fp16_holds(D):
    """70000 keys of equal scores: a probability is 1.4e-5, in fp16 a number of eight bits.  dV is their sum over the last rows'
    do alone, so nothing averages the error out; each is rounded to 11 bits, and so is the result."""
    rows, heads = 70001, (1, 1, D, 1.0)
    qkv, do = torch.zeros(rows, 3 * D, dtype=torch.float16, device=DEV), torch.zeros(rows, D, dtype=torch.float16, device=DEV)
    do[-1] = _randn(D, seed=10) * 64 + 256
    got = _step(qkv, do, [0, rows], heads)[:, 2 * D:].double()
    want = do[-1].double() / rows
    assert ((got - want).abs() <= 2.0 ** -11 * 2.02 * want.abs() + 2.0 ** -20 * want.abs() + orc.tiny(torch.float16)).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** -12, 1.0])
def test_values_as_large_as_documented(size, D):
    """Rows of v whose magnitudes add up to 15900 and a `do` that goes along with one half of them and against the other: the
    largest dS that there can be, 2 * 15900 * |do|, scaled to 2 at most, is below 65504."""
    rows, heads = 300, (2, 1, D, D ** -0.5)
    g = torch.Generator().manual_seed(11)
    way = torch.randint(0, 2, (D,), generator=g) * 2 - 1
    side = torch.randint(0, 2, (rows, 1), generator=g) * 2 - 1
    qkv = _randn(rows, 4 * D, seed=12, std=0.3)
    qkv[:, 3 * D:] = (side * way * (15900 / D)).half()
    do = (way.repeat(2) * 1.99 * size * torch.ones(rows, 1)).half().to(DEV)
    got = _step(qkv, do, [0, rows], heads)
    want = orc.attention(qkv, [0, rows], *heads, do)["dqkv"]
    big = want.abs() > 6e4                                 # what fp16 does not hold as a result
    for cols in _parts(heads):
        w, off = want[:, cols], (got[:, cols].double() - want[:, cols])[~big[:, cols]]
        assert torch.isfinite(off).all() and off.norm() <= 3 * 2.0 ** -11 * w.norm() + 2.0 ** -25 * w.numel() ** 0.5
