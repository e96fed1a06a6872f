"""What the products and the optimizer refuse on the GPU, by the extension's own checks."""
import pytest
import torch

from shift_b200.ops import fp8
from shift_b200.optim import AdamWMany, State8
from test_fp8_refusals_cpu import check_out_rows_apart, check_segments_are_needed, moved

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_products():
    a, b = fp8.quantize(torch.ones(4, 40, device=DEV)), fp8.quantize(torch.ones(6, 40, device=DEV))
    host = fp8.quantize(torch.ones(6, 40))
    for bad in (lambda: fp8.matmul(a, fp8.quantize(torch.ones(6, 41, device=DEV))), lambda: fp8.matmul(a, host),
                lambda: fp8.matmul(a, b, accumulate=True), lambda: fp8.matmul(a, b, out=torch.empty(4, 5, device=DEV)),
                lambda: fp8.matmul(a, b, out=torch.empty(4, 6)),
                lambda: fp8.matmul(a, b, out=torch.empty(4, 6, dtype=torch.float16, device=DEV)),
                lambda: fp8.matmul(a, b, out=torch.empty(6, 4, device=DEV).t()),
                lambda: fp8.matmul(a._replace(cols=400), b), lambda: fp8.matmul(a._replace(cols=-1), b),
                lambda: fp8.matmul(a._replace(scale=a.scale[:, :2]), b),
                lambda: fp8.matmul(a._replace(data=a.data.view(torch.uint8)), b),
                lambda: fp8.grouped_matmul(a, b, torch.zeros(5, dtype=torch.int32, device=DEV)),
                lambda: fp8.grouped_matmul(a, b, torch.zeros(3, device=DEV)),
                lambda: fp8.grouped_matmul(a, b, torch.zeros(1, dtype=torch.int32, device=DEV)),
                lambda: fp8.grouped_matmul(a, b, torch.zeros(4, dtype=torch.int32)),
                lambda: fp8.grouped_wgrad(a, b, torch.tensor([0, 40], dtype=torch.int32, device=DEV),
                                          torch.empty(2, 4, 6, device=DEV))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("eight", [False, True])
def test_optimizer(eight):
    p = torch.ones(300, device=DEV)
    m, v = ((State8.zeros(p), State8.zeros(p)) if eight else (torch.zeros_like(p), torch.zeros_like(p)))
    opt, g = AdamWMany([p], [m], [v]), [torch.ones(300, device=DEV)]
    for bad in (lambda: opt.step([]), lambda: opt.step([g[0][:3]]), lambda: opt.step([g[0].double()]),
                lambda: opt.step([torch.ones(300)]), lambda: opt.step(g, step=0),
                lambda: opt.step([torch.ones(300, 2, device=DEV)[:, 0]]),
                lambda: opt.step(g, skip=torch.zeros(1, device=DEV)),
                lambda: opt.step(g, skip=torch.zeros(1, dtype=torch.int32)),
                lambda: opt.step(g, step_dev=torch.zeros(3, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    assert bool((p == 1).all())
    opt.step(g)
    assert bool((p != 1).all())


def test_segments_are_needed():
    """The extension itself refuses too: it would cut the contraction and sum ranges that nothing wrote."""
    from shift_b200.ops._ext import ext, status_word
    check_segments_are_needed(DEV)
    a, b = fp8.quantize(torch.ones(4, 4096, device=DEV)), fp8.quantize(torch.ones(6, 4096, device=DEV))
    for mode in (1, 2, -1):
        with pytest.raises(ValueError, match="offs"):
            ext().fp8_matmul(a.data, a.scale, a.cols, b.data, b.scale, b.cols, torch.zeros(1, 4, 6, device=DEV), None, mode,
                             False, False, status_word(a.device))


@pytest.mark.parametrize("side", [0, 1])
def test_scales_off_their_words_are_refused(side):
    q = [fp8.quantize(torch.ones(n, 600, device=DEV)) for n in (4, 6)]
    scale = q[side].scale
    for by in (1, 2, 3):
        q[side] = q[side]._replace(scale=moved(scale, by))
        with pytest.raises(ValueError, match="4 bytes"):
            fp8.matmul(*q)
    q[side] = q[side]._replace(scale=moved(scale, 4))
    assert bool((fp8.matmul(*q) == 600).all())


def test_out_rows_apart():
    check_out_rows_apart(DEV)


def test_rows_of_codes_that_overlap():
    """Broadcast or overlapping rows have no tensor map; a single row may have any stride."""
    a, b = fp8.quantize(torch.ones(4, 40, device=DEV)), fp8.quantize(torch.ones(8, 40, device=DEV))
    raw = a.data.view(torch.uint8)
    for bad in (raw[:1].expand(4, 48), raw.as_strided((4, 48), (32, 1))):
        for pair in ((a._replace(data=bad.view(a.data.dtype)), b), (b, a._replace(data=bad.view(a.data.dtype)))):
            with pytest.raises(ValueError, match="overlap"):
                fp8.matmul(*pair)
    one = fp8.BlockFp8(raw.as_strided((1, 48), (0, 1)).view(a.data.dtype), a.scale[:, :1].clone(), 40)
    assert bool((fp8.matmul(one, b) == 40).all())
