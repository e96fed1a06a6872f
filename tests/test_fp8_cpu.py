"""8-bit matrices on the CPU: the fp32 statements against 64 bits, and what the entry points refuse."""
import math

import pytest
import torch

import fp8_oracle as orc
from shift_b200.ops import fp8


def _matrix(rows, cols, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
    x[::5] = 0
    return x.to(dtype)


def _same_codes(q, code, exps):
    got = q.data[:, :q.cols].double()
    assert torch.equal(torch.nan_to_num(got, nan=1e9, posinf=2e9, neginf=-2e9),
                       torch.nan_to_num(code, nan=1e9, posinf=2e9, neginf=-2e9))
    n = exps.shape[1]
    byte = q.scale.view(torch.uint8).permute(1, 0, 2).reshape(q.rows, -1).int()
    assert torch.equal(byte[:, :n], exps.cpu() + 127) and int(byte[:, n:].abs().sum()) == 0


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 130), (129, 513), (64, 128)])
def test_quantize_against_64_bits(rows, cols, tiles, fmt):
    x = _matrix(rows, cols, rows + cols)
    q, qt = fp8.quantize(x, fmt, tiles=tiles, both=True)
    _same_codes(q, *orc.quantize(x, fmt, tiles))
    _same_codes(qt, *orc.quantize(x.t(), fmt, tiles))
    assert q.data.shape[1] % 16 == 0 and qt.data.shape[1] % 16 == 0


def test_quantize_keeps_non_finite_values_and_extremes():
    x = torch.zeros(4, 256)
    x[0, :6] = torch.tensor([math.inf, -math.inf, math.nan, 448.0, 1.0, -3.4e38])
    x[1, 0] = 2.0 ** -149                              # the smallest subnormal alone in its block
    x[2, 128] = 449.0                                  # just above a power of two times 448: a larger scale
    x[3, :] = math.nan
    for fmt in ("e4m3", "e5m2"):
        q = fp8.quantize(x, fmt)
        _same_codes(q, *orc.quantize(x, fmt, False))
        back = fp8.dequantize(q)
        assert not bool(torch.isfinite(back[0, :3]).any()) and bool(torch.isfinite(back[0, 3:5]).all())
        # 3.4e38 is 0.999 * 2^128: the nearest code stands for 2^128 itself, which fp32 does not hold
        assert float(orc.values(q)[0, 5]) == -2.0 ** 128 and float(back[0, 5]) == -math.inf
        assert bool(torch.isnan(back[3]).all()) and float(back[2, 0]) == 0.0


def test_batches_quantize_like_their_matrices():
    x = torch.stack([_matrix(130, 200, s) for s in range(3)])
    q, qt = fp8.quantize(x, tiles=True, both=True)
    for g in range(3):
        a, at = fp8.quantize(x[g], tiles=True, both=True)
        assert torch.equal(q.data.view(torch.uint8)[130 * g:130 * (g + 1)], a.data.view(torch.uint8))
        assert torch.equal(qt.scale.view(torch.uint8)[:, 200 * g:200 * (g + 1)], at.scale.view(torch.uint8))


@pytest.mark.parametrize("M,N,K", [(5, 7, 300), (1, 16, 1), (130, 64, 513)])
def test_matmul(M, N, K):
    a = fp8.quantize(_matrix(M, K, 1), "e5m2")
    b = fp8.quantize(_matrix(N, K, 2, torch.float32), "e4m3", tiles=True)
    y = fp8.matmul(a, b)
    orc.check_product(y, orc.values(a), orc.values(b))
    acc = torch.randn(M, N)
    y = fp8.matmul(a, b, out=acc.clone(), accumulate=True)
    orc.check_product(y, orc.values(a), orc.values(b), base=acc)


def test_grouped_forms_and_uncovered_rows():
    offs = torch.tensor([0, 0, 100, 130], dtype=torch.int32)
    x, w = _matrix(140, 96, 3), torch.stack([_matrix(32, 96, s) for s in range(3)])
    a, b = fp8.quantize(x), fp8.quantize(w, tiles=True)
    out = torch.full((140, 32), 7.0)
    fp8.grouped_matmul(a, b, offs, out=out)
    va, vb = orc.values(a), orc.values(b).view(3, 32, 96)
    orc.check_product(out[:100], va[:100], vb[1])
    orc.check_product(out[100:130], va[100:130], vb[2])
    assert bool((out[130:] == 7).all())
    offs = torch.tensor([0, 128, 128, 310], dtype=torch.int32)
    at, bt = fp8.quantize(_matrix(24, 310, 4)), fp8.quantize(_matrix(40, 310, 5))
    dw = torch.ones(3, 24, 40)
    fp8.grouped_wgrad(at, bt, offs, dw)
    orc.check_product(dw[2], orc.values(at)[:, 128:], orc.values(bt)[:, 128:])
    assert bool((dw[1] == 0).all())
    fp8.grouped_wgrad(at, bt, offs, dw, accumulate=True)
    orc.check_product(dw[0], 2 * orc.values(at)[:, :128], orc.values(bt)[:, :128], rounds=2)


def test_a_linear_layer_has_the_gradients_of_its_quantised_operands():
    x, w, dy = _matrix(70, 96, 6), _matrix(48, 96, 7), _matrix(70, 48, 8)
    (xq, xqt), (wq, wqt) = fp8.quantize(x, both=True), fp8.quantize(w, tiles=True, both=True)
    gq, gqt = fp8.quantize(dy, "e5m2", both=True)
    orc.check_product(fp8.matmul(gq, wqt), orc.values(gq), orc.values(wq).t())       # tiles: one set of values
    orc.check_product(fp8.matmul(gqt, xqt, out_dtype=torch.float32), orc.values(gqt), orc.values(xqt))
    # quantised along either side a value moves by at most half a step of the type
    for q, back, ref, half in ((xq, fp8.dequantize(xqt).t(), x, 2 ** -4), (gq, fp8.dequantize(gqt).t(), dy, 2 ** -3)):
        amax = ref.double().abs().max()
        assert bool(((back.double() - ref.double()).abs() <= half * ref.double().abs() + amax * 2.0 ** -17).all())
        assert bool(((fp8.dequantize(q).double() - ref.double()).abs() <= half * ref.double().abs()
                     + amax * 2.0 ** -17).all())


def test_empty_sides():
    q, qt = fp8.quantize(torch.zeros(0, 40), both=True)
    assert q.rows == 0 and qt.rows == 40 and qt.cols == 0
    b = fp8.quantize(torch.ones(3, 40))
    assert tuple(fp8.matmul(q, b).shape) == (0, 3)
    z = fp8.matmul(qt, fp8.quantize(torch.ones(5, 0)), out_dtype=torch.float32)
    assert tuple(z.shape) == (40, 5) and bool((z == 0).all())


def _bad(q, **kw):
    return q._replace(**kw)


def test_refusals():
    x = torch.ones(4, 40)
    a, b = fp8.quantize(x), fp8.quantize(torch.ones(6, 40))
    for bad in (lambda: fp8.quantize(x, "e3m4"), lambda: fp8.quantize(x.double()), lambda: fp8.quantize(x[0]),
                lambda: fp8.matmul(a, fp8.quantize(torch.ones(6, 41))),
                lambda: fp8.matmul(a, b, accumulate=True),
                lambda: fp8.matmul(a, b, out=torch.empty(4, 5)),
                lambda: fp8.matmul(a, b, out=torch.empty(4, 6, dtype=torch.float16)),
                lambda: fp8.matmul(a, b, out=torch.empty(6, 4).t()),
                lambda: fp8.matmul(_bad(a, cols=400), b), lambda: fp8.matmul(_bad(a, cols=-1), b),
                lambda: fp8.matmul(_bad(a, scale=a.scale[:, :2]), b),
                lambda: fp8.matmul(_bad(a, data=a.data.view(torch.uint8)), b),
                lambda: fp8.grouped_matmul(a, b, torch.zeros(5, dtype=torch.int32)),
                lambda: fp8.grouped_matmul(a, b, torch.zeros(3)),
                lambda: fp8.grouped_matmul(a, b, torch.zeros(1, dtype=torch.int32)),
                lambda: fp8.grouped_wgrad(a, b, torch.tensor([0, 40], dtype=torch.int32), torch.empty(2, 4, 6)),
                lambda: fp8.grouped_wgrad(a, b, torch.tensor([3, 40], dtype=torch.int32), torch.empty(1, 4, 6)),
                lambda: fp8.grouped_wgrad(a, b, torch.tensor([0, 39], dtype=torch.int32), torch.empty(1, 4, 6))):
        with pytest.raises(ValueError):
            bad()
