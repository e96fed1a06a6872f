"""AdamW over many tensors on the GPU against 64 bits and against the CPU's statement."""
import pytest
import torch

from shift_b200.optim import AdamWMany, State8
from test_optim_cpu import H, SIZES, check, expected, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _host(x):
    return None if x is None else [State8(s.code.cpu(), s.scale.cpu()) if isinstance(s, State8) else s.cpu() for s in x]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype,gdtype,master",
                         [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, True),
                          (torch.bfloat16, torch.float32, False), (torch.float16, torch.float16, True),
                          (torch.float32, torch.bfloat16, True), (torch.float16, torch.float32, False)])
def test_step_against_64_bits(dtype, gdtype, master, eight):
    params, grads, m, v, masters = make(dtype, eight, master, DEV, SIZES + [(4096,), (9999,)])
    grads = [g.clamp(-1e4, 1e4).to(gdtype) for g in grads]
    opt = AdamWMany(params, m, v, masters)
    for step in (1, 2, 50):
        before = [_host(x) for x in (params, grads, m, v, masters)]
        want = expected(*before, *H.values(), step, 0.5)
        opt.step(grads, step=step, grad_scale=0.5, **H)
        torch.cuda.synchronize()
        host = AdamWMany(_host(params), _host(m), _host(v), _host(masters))
        check(host, host.params, before[1], host.masters, want)


def _packed(tensors, lead):
    """The same tensors as views of one buffer, back to back from element `lead`."""
    flat = torch.full((lead + sum(t.numel() for t in tensors) + 5,), 77.0, device=DEV).to(tensors[0].dtype)
    out, at = [], lead
    for t in tensors:
        out.append(flat[at:at + t.numel()].view(t.shape))
        out[-1].copy_(t)
        at += t.numel()
    return flat, out


@pytest.mark.parametrize("eight", [False, True])
def test_views_without_alignment_give_the_same(eight):
    one, two = (make(torch.bfloat16, eight, True, DEV, SIZES + [(2000,)]) for _ in range(2))
    grads = [g.to(torch.bfloat16) for g in one[1]]
    AdamWMany(one[0], one[2], one[3], one[4]).step(grads, step=3, **H)
    flat, params = _packed(two[0], 1)
    _, g = _packed(grads, 3)
    wflat, masters = _packed(two[4], 1)
    if eight:
        code = lambda x: _packed([s.code.view(torch.uint8) for s in x], 1)[1]  # noqa: E731
        m, v = ([State8(c.view(torch.float8_e4m3fn), s.scale) for c, s in zip(code(x), x)] for x in two[2:4])
    else:
        m, v = _packed(two[2], 1)[1], _packed(two[3], 1)[1]
    AdamWMany(params, m, v, masters).step(g, step=3, **H)
    torch.cuda.synchronize()
    for a, b in zip(one[0] + one[4], params + masters):
        assert torch.equal(a, b)
    for a, b in zip(one[2] + one[3], list(m) + list(v)):
        assert torch.equal(a.code.view(torch.uint8), b.code.view(torch.uint8)) if eight else torch.equal(a, b)
    assert float(flat[0]) == 77 and bool((flat[-5:] == 77).all()) and float(wflat[0]) == 77


def test_mixed_types_and_more_tensors_than_one_launch():
    """Parameters of three types in one call; 700 tensors are more than a launch's table holds."""
    params, grads, m, v, _ = make(torch.float32, True, False, DEV, [(1 + 3 * i,) for i in range(700)])
    kinds = (torch.float32, torch.bfloat16, torch.float16)
    params = [p.to(kinds[t % 3]) for t, p in enumerate(params)]
    grads = [g.clamp(-1e4, 1e4).to(kinds[t % 2]) for t, g in enumerate(grads)]
    before = [_host(x) for x in (params, grads, m, v)]
    want = expected(*before, None, *H.values(), 4, 1.0)
    AdamWMany(params, m, v).step(grads, step=4, **H)
    torch.cuda.synchronize()
    host = AdamWMany(_host(params), _host(m), _host(v))
    check(host, host.params, before[1], None, want)


def test_random_bits_match_the_statement():
    """The GPU's codes are the CPU's, but for values within rounding of a border (at most 1 in 10^4)."""
    dev, cpu = make(torch.float32, True, False, DEV, [(50000,)]), make(torch.float32, True, False, "cpu", [(50000,)])
    AdamWMany(dev[0], dev[2], dev[3]).step(dev[1], step=9, seed=123456789012, **H)
    AdamWMany(cpu[0], cpu[2], cpu[3]).step(cpu[1], step=9, seed=123456789012, **H)
    for a, b in ((dev[2][0], cpu[2][0]), (dev[3][0], cpu[3][0])):
        assert float((a.code.view(torch.uint8).cpu() != b.code.view(torch.uint8)).float().mean()) <= 1e-4
        assert torch.equal(a.scale.view(torch.uint8).cpu(), b.scale.view(torch.uint8))


def test_skip_flag_nonfinite_and_a_captured_step():
    params, grads, m, v, masters = make(torch.bfloat16, True, True, DEV)
    opt = AdamWMany(params, m, v, masters)
    skip, flag = torch.ones(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    before = [x.clone() for x in masters]
    opt.step(grads, skip=skip, nonfinite=flag, **H)
    assert all(torch.equal(a, b) for a, b in zip(before, masters)) and int(flag) == 0
    block = torch.zeros(8, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grads, step_dev=block, skip=skip, nonfinite=flag, **H)
    skip.zero_()
    twin = make(torch.bfloat16, True, True, DEV)
    other = AdamWMany(*(twin[i] for i in (0, 2, 3)), masters=twin[4])
    for step in (1, 2):
        scalars = torch.tensor([H["lr"], 1 - H["beta1"] ** step, (1 - H["beta2"] ** step) ** 0.5])
        block.copy_(torch.cat([torch.tensor([step], dtype=torch.int32), scalars.view(torch.int32),
                               torch.zeros(4, dtype=torch.int32)]))
        graph.replay()
        other.step(twin[1], step=step, **H)
    torch.cuda.synchronize()
    for a, b in zip(masters, twin[4]):
        assert torch.equal(a, b)
    grads[4][5] = float("nan")
    opt.step(grads, nonfinite=flag, step=3, **H)
    assert int(flag) == 1


@pytest.mark.parametrize("bits,master", [(8, True), (32, False)])
def test_torch_optimizer_on_the_gpu_follows_the_cpu(bits, master):
    """Ten steps from the same start: weights of both agree to the moments' rounding borders (8 bits: a few values in
    10^4 may take the next code, 2^-3 of a moment, in one step; an update of lr 1e-3 then moves by at most 2.5e-4)."""
    from shift_b200.optim import AdamW

    def run(device):
        torch.manual_seed(5)
        ps = [torch.nn.Parameter(torch.randn(s).to(device)) for s in ((300, 40), (1000,), (3, 5, 7))]
        opt = AdamW(ps, lr=1e-3, state_bits=bits, master_weights=master)
        g = torch.Generator().manual_seed(6)
        for _ in range(10):
            for p in ps:
                p.grad = torch.randn(p.shape, generator=g).to(device)
                if p.dim() == 2:
                    p.grad = p.grad.t().contiguous().t()         # another layout
            opt.step()
        return [p.detach().cpu() for p in ps]

    for a, b in zip(run(DEV), run("cpu")):
        off = (a - b).abs()
        assert float((off > 1e-6 + 16 * 2.0 ** -24 * b.abs()).float().mean()) <= (1e-2 if bits == 8 else 0.0)
        assert float(off.max()) <= (10 * 2.5e-4 if bits == 8 else 1e-5)
