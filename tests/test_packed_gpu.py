"""Packed sequences on the GPU: the row plan, rotary positions and attention against 64 bits."""
import math
import random

import pytest
import torch

import packed_oracle as orc
from shift_b200.ops import packed
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


def _seqs(offs, rows):
    return packed.sequences(torch.tensor(offs, dtype=torch.int32, device=DEV), rows)


def _randn(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def _orders(seqs):
    """The plan's tile orders: of 128 queries, of 256 queries, of 128 keys."""
    n, n2 = -(-seqs.rows // 128), -(-seqs.rows // 256)
    return seqs.plan[3 * seqs.rows + 2:].split([n, n2, n])


# ----------------------------------------------------------------------------- the plan
@pytest.mark.parametrize("offs,rows", [
    ([0, 1], 1), ([0, 0], 0), ([0, 300], 300), ([3, 3, 3, 200, 255, 256, 257, 600], 700), ([0, 5, 2, 9], 9),
    ([-4, 7, 1000], 600), ([10, 4], 20), ([500, 600], 512), (list(range(0, 1025)), 1024), ([0] * 700 + [64, 512, 513], 515),
])
def test_sequences(offs, rows):
    got = _seqs(offs, rows)
    want = packed.sequences(torch.tensor(offs, dtype=torch.int32), rows)
    for name in ("start", "pos", "stop", "ends"):
        assert torch.equal(getattr(got, name).cpu(), getattr(want, name)), name
    for order, tile in zip(_orders(got), (128, 256, 128)):
        assert sorted(order.tolist()) == list(range(-(-rows // tile)))


def test_orders_put_the_costliest_tiles_first():
    offs, rows = [0, 100, 2100, 2400, 6000], 6100
    got = _seqs(offs, rows)
    start, stop = got.start.tolist(), got.stop.tolist()
    fwd = [(min(128 * t + 128, rows) + 127) // 128 - start[128 * t] // 128 for t in _orders(got)[0].tolist()]
    bwd = [(stop[min(128 * t + 128, rows) - 1] - 128 * t + 127) // 128 for t in _orders(got)[2].tolist()]
    assert fwd == sorted(fwd, reverse=True) and bwd == sorted(bwd, reverse=True)


# ----------------------------------------------------------------------------- rotary
SCALINGS = [None, packed.RotaryScaling("linear", 4.0), packed.RotaryScaling("base", 8.0),
            packed.RotaryScaling("ramp", 16.0, 4096)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot,heads,extra", [(64, 64, 5, 8), (128, 96, 3, 0), (64, 16, 1, 0), (6, 6, 2, 3), (118, 58, 7, 1),
                                                 (10, 4, 4, 2), (256, 256, 2, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotary(dtype, dim, rot, heads, extra, layout):
    rows = 37
    x = _randn(rows, heads * dim + extra, seed=dim + rot, dtype=dtype)
    pos = torch.tensor([0, -1, 1, 2 ** 31 - 1, -2 ** 31, 1000003] + [random.Random(i).randrange(1 << 20) for i in range(rows - 6)],
                       dtype=torch.int32, device=DEV)
    for n, scaling in enumerate(SCALINGS):
        if rot < 4 and scaling:
            continue
        plan = packed.Rotary(dim, 1.0e6, rot_dim=rot, layout=layout, scaling=scaling)
        for inverse in (False, True):
            want = orc.rotary(x, pos, plan.freq.to(DEV), heads, dim, rot, layout, plan.magnitude, inverse)
            got = x.clone()
            assert packed.rotary(got, pos, plan, heads, inverse=inverse) is got
            # angles: 64-bit frequencies of 1e-16 at positions up to 2^31, fp32 sines; the result rounded once
            size = x.abs().double().amax(1, keepdim=True) * plan.magnitude * 2
            orc.close(got, want, torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -20 * size + orc.tiny(dtype), (scaling, inverse))
            out = torch.full_like(x, 9.0)
            packed.rotary(x, pos, plan, heads, inverse=inverse, out=out)
            assert torch.equal(out[:, :heads * dim], got[:, :heads * dim]) and (out[:, heads * dim:] == 9).all()


def test_rotary_views_of_any_alignment():
    buf = _randn(50, 700, seed=3)
    pos = torch.arange(50, dtype=torch.int32, device=DEV)
    for layout in ("half", "interleaved"):
        plan = packed.Rotary(64, 1.0e4, layout=layout)
        for lo in (0, 1, 2, 4, 8, 11):
            for step in (1, 3):
                x = buf[::step, lo:lo + 5 * 64]
                want = packed.rotary(x.contiguous(), pos[:x.shape[0]].contiguous(), plan, 5)
                other = buf.clone()
                packed.rotary(other[::step, lo:lo + 320], pos[:x.shape[0]].contiguous(), plan, 5)
                assert torch.equal(other[::step, lo:lo + 320], want)
                other[::step, lo:lo + 320] = x
                assert torch.equal(other, buf)


def test_rotary_and_its_inverse_are_transposed():
    plan = packed.Rotary(64, 1.0e4, rot_dim=48, scaling=packed.RotaryScaling("ramp", 4.0, 256))
    x, y = _randn(90, 128, seed=1, dtype=torch.float32), _randn(90, 128, seed=2, dtype=torch.float32)
    pos = torch.arange(90, dtype=torch.int32, device=DEV) * 37
    a = (packed.rotary(x.clone(), pos, plan, 2).double() * y.double()).sum()
    b = (packed.rotary(y.clone(), pos, plan, 2, inverse=True).double() * x.double()).sum()
    assert abs(float(a - b)) < 1e-4


# ----------------------------------------------------------------------------- attention
SHAPES = [   # offsets, rows, query heads, key heads
    ([0, 1], 1, 1, 1),
    ([0, 1, 2, 4, 7], 7, 2, 2),
    ([0, 128], 128, 2, 1),
    ([0, 129], 129, 4, 1),
    ([0, 300], 300, 3, 3),
    ([0, 700], 700, 4, 2),
    ([0, 100, 101, 356, 357, 600], 640, 4, 4),
    ([5, 133, 133, 390, 500], 517, 6, 2),
    ([0, 64, 128, 192, 256, 320, 384], 384, 8, 1),
    ([200, 200, 300], 513, 3, 1),
    ([0, 0], 260, 2, 2),
    ([0, 1100], 1100, 2, 2),
    (list(range(0, 257, 2)), 257, 5, 5),
]


def _attend(offs, rows, Hq, Hkv, D, dtype, seed=0, std=1.0):
    qkv = _randn(rows, (Hq + 2 * Hkv) * D, seed=seed, dtype=dtype, std=std)
    seqs = _seqs(offs, rows)
    o, lse = packed.attention_fwd(qkv, seqs, Hq, Hkv, D, D ** -0.5)
    check_status()
    return qkv, seqs, o, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("offs,rows,Hq,Hkv", SHAPES)
def test_attention_fwd(offs, rows, Hq, Hkv, D, dtype):
    qkv, _, o, lse = _attend(offs, rows, Hq, Hkv, D, dtype)
    want = orc.attention(qkv, offs, Hq, Hkv, D, D ** -0.5)
    orc.close(o, want["o"], want["o_tol"], "o")
    orc.close(lse, want["lse"], 1e-5 * (1 + want["lse"].abs().nan_to_num(posinf=0)), "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("offs,rows,Hq,Hkv", SHAPES)
def test_attention_bwd(offs, rows, Hq, Hkv, D, dtype):
    qkv, seqs, o, lse = _attend(offs, rows, Hq, Hkv, D, dtype, seed=1)
    do = _randn(rows, Hq * D, seed=2, dtype=dtype)
    got = packed.attention_bwd(qkv, o, lse, do, seqs, Hq, Hkv, D, D ** -0.5)
    check_status()
    want = orc.attention(qkv, offs, Hq, Hkv, D, D ** -0.5, do)
    for name, cols in (("dv", slice((Hq + Hkv) * D, None)), ("dk", slice(Hq * D, (Hq + Hkv) * D)), ("dq", slice(0, Hq * D))):
        orc.close(got[:, cols], want["dqkv"][:, cols], want["dqkv_tol"][:, cols], name)


def _case(offs, rows, Hq=4, Hkv=2, D=64, dtype=torch.bfloat16, seed=5):
    return (_randn(rows, (Hq + 2 * Hkv) * D, seed=seed, dtype=dtype), _randn(rows, Hq * D, seed=seed + 1, dtype=dtype),
            _seqs(offs, rows), (Hq, Hkv, D, D ** -0.5))


def _step(qkv, do, seqs, heads):
    o, lse = packed.attention_fwd(qkv, seqs, *heads)
    return o, lse, packed.attention_bwd(qkv, o, lse, do, seqs, *heads)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_rows_of_no_sequence_are_not_looked_at(value, D):
    offs, rows = [70, 200, 330, 500], 700
    qkv, do, seqs, heads = _case(offs, rows, D=D)
    want = _step(qkv, do, seqs, heads)
    loud, ldo = qkv.clone(), do.clone()
    for t in (loud, ldo):
        t[:70] = value
        t[500:] = value
    got = _step(loud, ldo, seqs, heads)
    check_status()
    for name, g, w in zip(("o", "lse", "dqkv"), got, want):
        assert torch.equal(g, w), name
    assert not got[0][:70].any() and not got[2][500:].any() and (got[1][:, 500:] == -math.inf).all()


@pytest.mark.parametrize("D", [64, 128])
def test_sequences_do_not_hear_each_other(D):
    """NaN in one sequence, in the tiles of others, changes none of their results by more than the order of a sum."""
    offs, rows = [0, 100, 250, 390], 390
    for heads in ((4, 2), (3, 3)):
        qkv, do, seqs, heads = _case(offs, rows, *heads, D=D)
        loud, ldo = qkv.clone(), do.clone()
        loud[120, ::7] = math.nan
        ldo[130, 5] = math.inf
        got = _step(loud, ldo, seqs, heads)
        check_status()
        want = orc.attention(qkv, offs, *heads, do)
        for rows_ in (slice(0, 100), slice(250, 390)):
            orc.close(got[0][rows_], want["o"][rows_], want["o_tol"][rows_], "o")
            orc.close(got[1][:, rows_], want["lse"][:, rows_], 1e-4, "lse")
            orc.close(got[2][rows_], want["dqkv"][rows_], want["dqkv_tol"][rows_], "dqkv")
        orc.close(got[0][100:120], want["o"][100:120], want["o_tol"][100:120], "rows before the NaN")
        assert torch.isnan(got[0][120:250]).any(1).all()


@pytest.mark.parametrize("D", [64, 128])
def test_masked_values_count_as_nothing_however_large(D):
    """Other sequences' finite values of 3e38, in shared tiles, leave results as they are to the bit."""
    offs, rows = [0, 100, 250, 390, 600], 600
    for heads in ((4, 2), (3, 3)):
        qkv, do, seqs, heads = _case(offs, rows, *heads, D=D)
        kv = (heads[0] + heads[1]) * D
        qkv[100:250] = 0
        do[100:250] = 0
        want = _step(qkv, do, seqs, heads)
        qkv[100:250, kv:], do[100:250, ::3] = 3e38, 3e38
        got = _step(qkv, do, seqs, heads)
        check_status()
        for rows_ in (slice(0, 100), slice(250, 600)):
            assert torch.equal(got[0][rows_], want[0][rows_]) and torch.equal(got[1][:, rows_], want[1][:, rows_])
            assert torch.equal(got[2][rows_], want[2][rows_])


def test_attention_leaves_rows_of_no_sequence_in_a_given_out():
    offs, rows = [10, 140, 300], 400
    qkv, do, seqs, heads = _case(offs, rows)
    want = _step(qkv, do, seqs, heads)
    o, g = torch.full((rows, 256 + 8), 3.0, device=DEV, dtype=qkv.dtype), torch.full_like(qkv, 4.0)
    view = o[:, 8:]
    assert packed.attention_fwd(qkv, seqs, *heads, out=view)[0] is view
    packed.attention_bwd(qkv, view, want[1], do, seqs, *heads, out=g)
    assert torch.equal(view[10:300], want[0][10:300]) and (o[:, :8] == 3).all() and (o[:10] == 3).all() and (o[300:] == 3).all()
    assert torch.equal(g[10:300], want[2][10:300]) and (g[:10] == 4).all() and (g[300:] == 4).all()


def test_attention_of_strided_rows():
    offs, rows = [0, 333], 333
    qkv, do, seqs, heads = _case(offs, rows)
    want = _step(qkv, do, seqs, heads)
    wide, wdo = torch.full((2 * rows, 528), math.nan, device=DEV, dtype=qkv.dtype), torch.empty(rows, 264, device=DEV, dtype=qkv.dtype)
    wide[::2, 8:520], wdo[:, :256] = qkv, do
    got = _step(wide[::2, 8:520], wdo[:, :256], seqs, heads)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_attention_is_deterministic_and_splits_heads():
    for heads, rows in (((8, 1), 300), ((16, 4), 1500)):
        qkv, do, seqs, heads = _case([0, rows // 3, rows], rows, *heads)
        first = _step(qkv, do, seqs, heads)
        for _ in range(3):
            for a, b in zip(first, _step(qkv, do, seqs, heads)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_large_scores(dtype):
    """Scores of some hundreds: maxima that rise late, probabilities that vanish."""
    offs, rows, Hq, Hkv, D = [0, 40, 800], 800, 2, 1, 64
    qkv = _randn(rows, (Hq + 2 * Hkv) * D, seed=9, dtype=dtype)
    qkv[:, :(Hq + Hkv) * D] *= 6
    qkv[300:310, Hq * D:(Hq + 1) * D] *= 3
    seqs = _seqs(offs, rows)
    o, lse = packed.attention_fwd(qkv, seqs, Hq, Hkv, D, D ** -0.5)
    want = orc.attention(qkv, offs, Hq, Hkv, D, D ** -0.5)
    orc.close(o, want["o"], want["o_tol"], "o")
    orc.close(lse, want["lse"], 1e-5 * (1 + want["lse"].abs()), "lse")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** 9])
def test_fp16_gradients_of_any_size(size, D):
    """dS of a long row is near 2^-20 of do's size, below what fp16 holds well, or above what it holds at all."""
    rows, heads = 1500, (2, 1, D, D ** -0.5)
    qkv, do = _randn(rows, 4 * D, seed=11, dtype=torch.float16), _randn(rows, 2 * D, seed=12, dtype=torch.float16) * size
    got = _step(qkv, do, _seqs([0, rows], rows), heads)[2].double()
    check_status()
    want = orc.attention(qkv, [0, rows], *heads, do)["dqkv"]
    for cols in (slice(0, 2 * D), slice(2 * D, 3 * D), slice(3 * D, None)):
        w = want[:, cols]
        # roundings of P, dS and the result, 2^-11 each of a value of random sign, and the result's own smallest step
        bound = 3 * 2.0 ** -11 * w.norm() + 2.0 ** -25 * w.numel() ** 0.5
        assert (got[:, cols] - w).norm() <= bound


def test_a_step_of_nan_takes_no_longer():
    """Where everything is NaN, nothing is computed again row by row (that would take some hundred times as long)."""
    rows, heads = 8192, (4, 2, 64, 0.125)
    qkv, do, seqs = _randn(rows, 8 * 64, seed=1), _randn(rows, 4 * 64, seed=2), _seqs([0, rows], rows)
    bad = torch.full_like(qkv, math.nan)
    times = []
    for x, g in ((qkv, do), (bad, do), (qkv, torch.full_like(do, math.nan))):
        _step(x, g, seqs, heads)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        got = _step(x, g, seqs, heads)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    check_status()
    assert torch.isnan(got[2][:, :6 * 64]).all() and max(times[1:]) < 20 * times[0], times


@pytest.mark.parametrize("where", [0, 1, 5, 14, 63, 130, 255])
@pytest.mark.parametrize("D", [64, 128])
def test_a_score_of_nan_stays(where, D):
    """One key that is NaN makes every later row of its sequence NaN, statistics and gradients among it, and no earlier one.
    Its value is finite, so that it is the score that has to tell."""
    rows, first, heads = 256, 3, (2, 1, D, D ** -0.5)
    qkv, do = _randn(rows, 4 * D, seed=where + 1), _randn(rows, 2 * D, seed=where + 2)
    seqs = _seqs([first, rows], rows)
    at = max(where, first)
    qkv[at, 2 * D + 1] = math.nan
    o, lse, d = _step(qkv, do, seqs, heads)
    check_status()
    late = torch.arange(rows, device=DEV) >= at
    inside = torch.arange(rows, device=DEV) >= first
    assert torch.isnan(o[late]).all() and torch.isfinite(o[~late]).all()
    assert torch.isnan(lse[:, late]).all() and torch.isfinite(lse[:, inside & ~late]).all()
    assert torch.isnan(d[late, :2 * D]).all() and torch.isfinite(d[~late, :2 * D]).all()
    # every key of the sequence is met by its last row, which is NaN
    assert torch.isnan(d[inside, 2 * D:]).all() and torch.isfinite(d[~inside]).all()


@pytest.mark.parametrize("rows,Hq,Hkv", [(300, 2, 1), (5000, 8, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_infinite_scores(D, rows, Hq, Hkv):
    at, seqs, heads = 137, _seqs([0, rows], rows), (Hq, Hkv, D, D ** -0.5)
    late = torch.arange(rows, device=DEV) >= at
    x, do = _randn(rows, (Hq + 2 * Hkv) * D, seed=8), _randn(rows, Hq * D, seed=9)
    x[:, :(Hq + Hkv) * D:D] = x[:, :(Hq + Hkv) * D:D].abs() + 1                  # the first column of every head
    # one row of one head whose scores are all minus infinity: 0 / 0, and an empty sum's logarithm
    y = x.clone()
    y[at, 0] = -math.inf
    o, lse, d = _step(y, do, seqs, heads)
    check_status()
    assert torch.isnan(o[at, :D]).all() and torch.isfinite(o[~(torch.arange(rows, device=DEV) == at)]).all()
    assert torch.isfinite(o[at, D:]).all() and lse[0, at] == -math.inf and (~torch.isfinite(lse)).sum() == 1
    assert torch.isnan(d[:at + 1, Hq * D:Hq * D + D]).all() and torch.isfinite(d[at + 1:]).all()
    # a key whose score is minus infinity counts for nothing
    y = x.clone()
    y[at, Hq * D] = -math.inf
    o, lse, d = _step(y, do, seqs, heads)
    check_status()
    assert torch.isfinite(o).all() and torch.isfinite(lse).all() and torch.isfinite(d[:, Hq * D:]).all()
    # a score of plus infinity makes its row NaN
    y[at, Hq * D] = math.inf
    o, lse, d = _step(y, do, seqs, heads)
    check_status()
    group = Hq // Hkv * D
    assert torch.isnan(o[late, :group]).all() and torch.isfinite(o[~late]).all() and torch.isfinite(o[:, group:]).all()
    assert not torch.isfinite(lse[:Hq // Hkv, late]).any() and torch.isfinite(lse[:, ~late]).all()
