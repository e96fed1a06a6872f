"""``optim.AdamW`` on the GPU as scripts handle a torch optimizer."""
import copy

import pytest
import torch

from shift_b200.optim import AdamW
from test_optim_torch_cpu import KINDS, check_layouts, check_stock_state, same, same_state

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits,master", KINDS)
def test_parameters_of_any_layout(bits, master):
    check_layouts(bits, master, DEV)


@pytest.mark.parametrize("bits,master", KINDS)
def test_cleared_replaced_and_copied_state(bits, master):
    def make():
        g = torch.Generator().manual_seed(1)
        ps = [torch.nn.Parameter(torch.randn(s, generator=g).to(torch.bfloat16).to(DEV)) for s in ((70, 9), (130,))]
        return ps, AdamW(ps, lr=1e-2, state_bits=bits, master_weights=master)

    def turn(ps, opt, i):
        g = torch.Generator().manual_seed(50 + i)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(p)
        opt.step()

    (ps, opt), (qs, other) = make(), make()
    turn(ps, opt, 0)
    opt.state.clear()
    for p, q in zip(ps, qs):
        p.data.copy_(q.data)
    turn(ps, opt, 1)
    turn(qs, other, 1)
    assert same(ps, qs)
    same_state(opt, ps, other, qs)
    third = copy.deepcopy(opt)
    rs = third.param_groups[0]["params"]
    for x, o in ((ps, opt), (rs, third)):
        turn(x, o, 2)
    assert same(ps, rs)
    for q in qs:                                       # the state of one is given to the other
        for k, x in other.state[q].items():
            if isinstance(x, torch.Tensor):
                other.state[q][k] = torch.zeros_like(x)
    for p, q, r in zip(ps, qs, rs):
        for k, x in opt.state[p].items():
            other.state[q][k] = x.clone() if isinstance(x, torch.Tensor) else x
        q.data.copy_(p.data)
    for x, o in ((ps, opt), (qs, other)):
        turn(x, o, 3)
    assert same(ps, qs)
    same_state(opt, ps, other, qs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits,master", KINDS)
def test_the_stock_optimizers_saved_state(bits, master, dtype):
    check_stock_state(bits, master, dtype, DEV)


def test_a_captured_step_is_refused():
    """The refusal comes before any launch, so the capture ends as an empty one and the optimizer goes on."""
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    opt = AdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
    assert opt.state[p]["step"] == 1
    opt.step()
    torch.cuda.synchronize()
    assert opt.state[p]["step"] == 2 and bool((x == 0).all())
