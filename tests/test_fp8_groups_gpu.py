"""Contractions by group where a CTA pair takes many tiles and many groups are empty: a tile that issues no product passes
both accumulators on like any other, also where the two share columns (tiles of 256)."""
import pytest
import torch

import fp8_oracle as orc
from shift_b200.ops import fp8
from shift_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"

PATTERNS = {"lead": [0] * 9 + [1, 2, 5] * 5, "every other": [0, 3] * 12, "runs": [2, 0, 0, 0, 1, 1, 0, 0, 6, 0, 0, 0] * 2,
            "last": [4] + [0] * 23, "full": [1, 2, 3, 4] * 6}


# the widths that the host's rule takes for 24 groups: 256, 224, 192, 128 columns by pairs, then single CTAs
@pytest.mark.parametrize("M,N", [(1024, 1024), (1024, 672), (768, 576), (1000, 120), (100, 3000)])
@pytest.mark.parametrize("pattern", list(PATTERNS))
def test_empty_groups_between_full_ones(pattern, M, N):
    blocks = PATTERNS[pattern]
    o = [0]
    for c in blocks:
        o.append(o[-1] + 128 * c)
    g = torch.Generator(device=DEV).manual_seed(M + N)
    a = fp8.quantize(torch.randn(M, o[-1], device=DEV, generator=g), "e5m2")
    b = fp8.quantize(torch.randn(N, o[-1], device=DEV, generator=g))
    offs = torch.tensor(o, dtype=torch.int32, device=DEV)
    out = torch.full((len(blocks), M, N), 7.0, device=DEV)
    fp8.grouped_wgrad(a, b, offs, out)
    twice = out.clone()
    fp8.grouped_wgrad(a, b, offs, twice, accumulate=True)
    half = torch.full_like(out, 7.0, dtype=torch.bfloat16)
    fp8.grouped_wgrad(a, b, offs, half)
    torch.cuda.synchronize()
    check_status()
    va, vb = orc.values(a), orc.values(b)
    for i, c in enumerate(blocks):
        if c == 0:
            assert bool((out[i] == 0).all()) and bool((half[i] == 0).all())
            continue
        x, y = va[:, o[i]:o[i + 1]], vb[:, o[i]:o[i + 1]]
        orc.check_product(out[i], x, y)
        orc.check_product(half[i], x, y)
    assert torch.equal(twice, out + out)                 # the same sums, added to themselves
