"""Rotary positions into another buffer: heads of an odd number of columns, some of them not rotated."""
import pytest
import torch

import packed_oracle as orc
from shift_b200.ops import packed

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot,heads,extra", [(5, 4, 3, 0), (65, 64, 2, 1), (9, 6, 4, 3), (7, 2, 1, 0), (33, 32, 5, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_every_column_of_an_odd_head_is_written(dtype, dim, rot, heads, extra, layout):
    rows = 37
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(rows, heads * dim + extra, generator=g).to(dtype).to(DEV)
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, dtype=torch.int32).to(DEV)
    plan = packed.Rotary(dim, 1.0e4, rot_dim=rot, layout=layout)
    for inverse in (False, True):
        want = orc.rotary(x, pos, plan.freq.to(DEV), heads, dim, rot, layout, 1.0, inverse)
        for out in (torch.full_like(x, 9.0), torch.full((rows, heads * dim + extra + 2), 9.0, dtype=dtype, device=DEV)):
            packed.rotary(x, pos, plan, heads, inverse=inverse, out=out)
            size = 2 * x.abs().double().amax(1, keepdim=True)
            cols = slice(0, heads * dim)
            orc.close(out[:, cols], want[:, cols], torch.finfo(dtype).eps / 2 * want[:, cols].abs() + 2.0 ** -20 * size, inverse)
            same = x[:, cols].view(rows, heads, dim)[..., rot:]
            assert torch.equal(out[:, cols].reshape(rows, heads, dim)[..., rot:], same) and (out[:, heads * dim:] == 9).all()
        here = packed.rotary(x.clone(), pos, plan, heads, inverse=inverse)
        assert torch.equal(here[:, :heads * dim], out[:, :heads * dim]) and torch.equal(here[:, heads * dim:], x[:, heads * dim:])
