"""8-bit matrices on the GPU: the kernels against 64 bits, at the sizes and layouts where they can go wrong."""
import math

import pytest
import torch

import fp8_oracle as orc
from shift_b200.ops import fp8
from shift_b200.ops import reference as ref
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _matrix(rows, cols, seed, dtype=torch.bfloat16, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
    if rows > 4:
        x[::5] = 0
    return x.to(dtype).to(DEV)


def _same(q, data, scale):
    got = q.data[:, :q.cols].float().cpu()
    want = data.view(q.data.dtype)[:, :q.cols].float()
    assert torch.equal(torch.nan_to_num(got, nan=1e9, posinf=2e9, neginf=-2e9),
                       torch.nan_to_num(want, nan=1e9, posinf=2e9, neginf=-2e9))
    assert torch.equal(q.scale.view(torch.uint8).cpu(), scale)


def _check_quantize(x, fmt, tiles, both):
    got = fp8.quantize(x, fmt, tiles=tiles, both=both)
    want = ref.fp8_quantize(x.cpu(), fmt, tiles, both)
    for i, q in enumerate(got if both else (got,)):
        _same(q, *want[2 * i:2 * i + 2])
    return got


# ----------------------------------------------------------------------------- quantiser
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tiles,both", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 1000), (128, 512), (129, 513), (300, 1024), (1000, 24), (7, 40)])
def test_quantize(rows, cols, tiles, both, dtype):
    for fmt in ("e4m3", "e5m2"):
        _check_quantize(_matrix(rows, cols, rows * cols, dtype), fmt, tiles, both)


def test_quantize_strided_misaligned_and_batched():
    x = _matrix(200, 700, 3)
    _check_quantize(x[:, 1:600], "e4m3", False, True)          # base and rows off 16 bytes
    _check_quantize(x[::3, 8:520], "e5m2", False, True)        # a row stride
    _check_quantize(x[5:6, :9], "e4m3", True, True)
    w = torch.stack([_matrix(130, 200, s) for s in range(5)])
    _check_quantize(w, "e4m3", True, True)
    _check_quantize(w[1::2, :, 40:], "e4m3", True, True)
    _check_quantize(w[:, 3:90], "e4m3", False, True)
    with pytest.raises(RuntimeError, match="contiguous"):
        fp8.quantize(x.t())


def test_quantize_non_finite_and_extremes():
    x = torch.zeros(260, 256)
    x[0, :6] = torch.tensor([math.inf, -math.inf, math.nan, 448.0, 1.0, -3.3e38])
    x[1, 0] = 2.0 ** -133
    x[2, 128] = 450.0
    x[3] = math.nan
    x[200, 7] = -math.inf
    x[259, 255] = 1e-30
    for dtype in (torch.float32, torch.bfloat16):
        for fmt in ("e4m3", "e5m2"):
            for tiles in (False, True):
                _check_quantize(x.to(dtype).to(DEV), fmt, tiles, True)


def test_quantize_empty():
    for shape in ((0, 64), (64, 0), (0, 3, 5)):
        q, qt = fp8.quantize(torch.empty(shape, device=DEV), both=True)
        assert q.cols == shape[-1] and qt.cols == shape[-2]


# ----------------------------------------------------------------------------- products
def _pair(M, N, K, fa="e4m3", fb="e4m3", spread=2.0):
    return fp8.quantize(_matrix(M, K, M + K, spread=spread), fa), fp8.quantize(_matrix(N, K, N + 7 * K, spread=spread), fb)


def _done():
    torch.cuda.synchronize()
    check_status()


SIZES = [(1, 16, 16), (1, 1, 1), (1, 1000, 1024), (5, 33, 700), (64, 640, 96), (128, 128, 128), (129, 225, 129),
         (256, 448, 1024), (300, 1000, 2061), (1000, 8, 4096), (2050, 1536, 640), (40, 3000, 513),
         # every tile width, by one CTA and by a pair, several tiles to each
         (1, 32768, 200), (100, 28000, 130), (4096, 4096, 2500), (16384, 672, 200), (5000, 1344, 1024)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_matmul(M, N, K):
    a, b = _pair(M, N, K)
    y = fp8.matmul(a, b)
    _done()
    orc.check_product(y, orc.values(a), orc.values(b))


@pytest.mark.parametrize("fa,fb", [("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
def test_matmul_types(fa, fb):
    a, b = _pair(200, 300, 400, fa, fb)
    y = fp8.matmul(a, b, out_dtype=torch.float32)
    _done()
    orc.check_product(y, orc.values(a), orc.values(b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(384, 256, 8192), (200, 100, 3000), (1536, 1024, 4096), (17, 9, 5000),
                                   (4096, 4096, 300)])
def test_matmul_accumulate(M, N, K, dtype):
    a, b = _pair(M, N, K, "e5m2", "e4m3", spread=1.0)
    base = torch.randn(M, N, device=DEV).to(dtype)
    y = fp8.matmul(a, b, out=base.clone(), accumulate=True)
    _done()
    orc.check_product(y, orc.values(a), orc.values(b), base=base)
    again = fp8.matmul(a, b, out=base.clone(), accumulate=True)
    assert torch.equal(y, again)                                       # no order of summation is left to chance


def test_matmul_block_scales_follow_their_block():
    """Ones times ones with a different power of two in every block: any misplaced scale shows in the sum."""
    M, N, K = 260, 200, 1800
    ka = torch.arange(-(-K // 128))
    for side in range(2):
        one = torch.ones(M, K)
        other = torch.ones(N, K)
        x = (one, other)[side]
        e = (ka[None, :] + torch.arange(x.shape[0])[:, None]) % 7
        x.mul_(torch.pow(2.0, e.float()).repeat_interleave(128, 1)[:, :K])
        a, b = fp8.quantize(one.to(DEV)), fp8.quantize(other.to(DEV))
        y = fp8.matmul(a, b, out_dtype=torch.float32)
        _done()
        assert torch.equal(y.double().cpu(), one.double() @ other.double().t())    # small whole numbers: exact


def test_matmul_out_views_and_untouched_surroundings():
    a, b = _pair(130, 200, 300)
    want = fp8.matmul(a, b)
    for dtype, lo in ((torch.bfloat16, 8), (torch.bfloat16, 3), (torch.float32, 4), (torch.float32, 1)):
        big = torch.full((140, 220), 9.0, dtype=dtype, device=DEV)
        out = big[5:135, lo:lo + 200]
        fp8.matmul(a, b, out=out)
        _done()
        assert torch.equal(out.to(torch.bfloat16), want)
        rest = big.clone()
        rest[5:135, lo:lo + 200] = 9.0
        assert bool((rest == 9).all())


def test_matmul_non_finite_operands_show():
    x = torch.ones(130, 300)
    x[3, 7], x[129, 299] = math.nan, math.inf
    a, b = fp8.quantize(x.to(DEV)), fp8.quantize(torch.ones(40, 300, device=DEV))
    y = fp8.matmul(a, b)
    _done()
    bad = ~torch.isfinite(y).all(1)
    assert bad.nonzero().flatten().tolist() == [3, 129]


def test_matmul_extreme_scales():
    """Scales near both ends: their product is in range although neither operand is near 1."""
    a = fp8.quantize(torch.full((130, 260), 2.0 ** 100, device=DEV))
    b = fp8.quantize(torch.full((20, 260), 2.0 ** -100, device=DEV))
    y = fp8.matmul(a, b, out_dtype=torch.float32)
    _done()
    assert bool((y == 260).all())


def test_matmul_empty():
    b = fp8.quantize(torch.ones(3, 40, device=DEV))
    assert tuple(fp8.matmul(fp8.quantize(torch.ones(0, 40, device=DEV)), b).shape) == (0, 3)
    e0, e1 = fp8.quantize(torch.ones(5, 0, device=DEV)), fp8.quantize(torch.ones(3, 0, device=DEV))
    assert bool((fp8.matmul(e0, e1) == 0).all())
    base = torch.randn(5, 3, device=DEV)
    assert torch.equal(fp8.matmul(e0, e1, out=base.clone(), accumulate=True), base)


# ----------------------------------------------------------------------------- experts
def _segments(counts, pad=1, lead=0):
    o = [lead]
    for c in counts:
        o.append(o[-1] + -(-c // pad) * pad)
    return o


@pytest.mark.parametrize("N,K", [(96, 300), (448, 512), (1344, 1024)])
@pytest.mark.parametrize("counts,lead", [([300, 0, 1, 128, 257], 0), ([0, 0, 0], 0), ([5], 3), ([129] * 20, 0)])
def test_grouped_matmul(counts, lead, N, K):
    o = _segments(counts, lead=lead)
    R = o[-1] + 37
    G = len(counts)
    a = fp8.quantize(_matrix(R, K, R))
    b = fp8.quantize(torch.stack([_matrix(N, K, 50 + s) for s in range(G)]), tiles=True)
    out = torch.full((R, N), 5.0, dtype=torch.bfloat16, device=DEV)
    fp8.grouped_matmul(a, b, torch.tensor(o, dtype=torch.int32, device=DEV), out=out)
    _done()
    va, vb = orc.values(a), orc.values(b).view(G, N, K)
    for g in range(G):
        if o[g + 1] > o[g]:
            orc.check_product(out[o[g]:o[g + 1]], va[o[g]:o[g + 1]], vb[g])
    assert bool((out[:lead] == 5).all()) and bool((out[o[-1]:] == 5).all())


@pytest.mark.parametrize("dtype,acc", [(torch.float32, False), (torch.float32, True), (torch.bfloat16, False),
                                       (torch.bfloat16, True)])
@pytest.mark.parametrize("M,N", [(40, 100), (256, 224), (672, 1024)])
def test_grouped_wgrad(M, N, dtype, acc):
    counts = [300, 0, 1, 128, 700]
    o = _segments(counts, pad=128)
    R = o[-1] + 60
    live = torch.zeros(R, 1)
    for s, c in zip(o, counts):
        live[s:s + c] = 1
    live[o[-1]:] = 1                                     # behind the last segment: anything
    live = live.to(DEV)
    _, at = fp8.quantize(_matrix(R, M, 8, torch.float32) * live, "e5m2", both=True)
    _, bt = fp8.quantize(_matrix(R, N, 9, torch.float32) * live, both=True)
    base = torch.randn(len(counts), M, N, device=DEV).to(dtype)
    out = base.clone()
    fp8.grouped_wgrad(at, bt, torch.tensor(o, dtype=torch.int32, device=DEV), out, accumulate=acc)
    _done()
    va, vb = orc.values(at), orc.values(bt)
    for g in range(len(counts)):
        orc.check_product(out[g], va[:, o[g]:o[g + 1]], vb[:, o[g]:o[g + 1]], base=base[g] if acc else None)


@pytest.mark.parametrize("offs", [[0, 100, 512], [0, 128, 500]])
def test_segments_off_a_block_are_refused_by_the_status_word(offs):
    a, b = _pair(40, 50, 512)
    out = torch.full((2, 40, 50), 3.0, device=DEV)
    fp8.grouped_wgrad(a, b, torch.tensor(offs, dtype=torch.int32, device=DEV), out)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="status"):
        check_status()
    check_status()
    assert bool((out == 3).all())


def test_a_last_segment_that_ends_with_the_matrix():
    a, b = _pair(40, 50, 500)
    out = torch.zeros(2, 40, 50, device=DEV)
    fp8.grouped_wgrad(a, b, torch.tensor([0, 128, 500], dtype=torch.int32, device=DEV), out)
    _done()
    va, vb = orc.values(a), orc.values(b)
    orc.check_product(out[0], va[:, :128], vb[:, :128])
    orc.check_product(out[1], va[:, 128:], vb[:, 128:])


def test_segments_outside_the_rows_are_cut():
    a = fp8.quantize(_matrix(200, 64, 1))
    w = torch.stack([_matrix(32, 64, s) for s in range(3)])
    b = fp8.quantize(w, tiles=True)
    out = torch.full((200, 32), 5.0, dtype=torch.bfloat16, device=DEV)
    fp8.grouped_matmul(a, b, torch.tensor([-10, 90, 50, 400], dtype=torch.int32, device=DEV), out=out)
    _done()
    va, vb = orc.values(a), orc.values(b).view(3, 32, 64)
    orc.check_product(out[:50], va[:50], vb[0])
    orc.check_product(out[90:200], va[90:200], vb[2])       # the third segment starts where the second one said


# ----------------------------------------------------------------------------- as they are used
def test_another_stream_and_a_captured_graph():
    x, w = _matrix(300, 512, 1), _matrix(256, 512, 2)
    side = torch.cuda.Stream()
    dw = torch.zeros(256, 512, device=DEV)

    def layer():
        (xq, xqt), (wq, wqt) = fp8.quantize(x, both=True), fp8.quantize(w, tiles=True, both=True)
        y = fp8.matmul(xq, wq)
        gq, gqt = fp8.quantize(y, "e5m2", both=True)
        return y, fp8.matmul(gq, wqt), fp8.matmul(gqt, xqt, out=dw, accumulate=True)

    want = [t.clone() for t in layer()]
    dw.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in layer()]
    torch.cuda.current_stream().wait_stream(side)
    _done()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    x.copy_(_matrix(300, 512, 11))
    dw.zero_()
    graph.replay()
    replayed = [t.clone() for t in out]
    dw.zero_()
    eager = layer()
    _done()
    assert all(torch.equal(a, b) for a, b in zip(replayed, eager))


def test_two_streams_at_once():
    """Products, split ones among them, on two streams that nothing orders, next to bf16 products."""
    from shift_b200.ops import gemm as G
    cases = [_pair(384, 256, 8192), _pair(1000, 1344, 1024), _pair(1, 4096, 512), _pair(300, 200, 5000)]
    want = [fp8.matmul(a, b, out_dtype=torch.float32) for a, b in cases]
    x, w = _matrix(512, 256, 1, spread=0.1), _matrix(384, 256, 2, spread=0.1)
    plain = G.linear_fwd(x, w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for turn in range(10):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                order = cases if k == 0 else cases[::-1]
                got[k] = [fp8.matmul(a, b, out_dtype=torch.float32) for a, b in order] + [G.linear_fwd(x, w)]
    _done()
    for k in range(2):
        mine = got[k][:-1] if k == 0 else got[k][:-1][::-1]
        assert all(torch.equal(a, b) for a, b in zip(mine, want)) and torch.equal(got[k][-1], plain)


def test_the_same_operand_twice_and_its_own_sum():
    a, _ = _pair(300, 16, 700)
    y = fp8.matmul(a, a, out_dtype=torch.float32)
    _done()
    orc.check_product(y, orc.values(a), orc.values(a))
