"""``optim.AdamW`` as scripts handle a torch optimizer: state that is cleared, replaced, copied or saved by others."""
import copy
import pickle

import pytest
import torch

from shift_b200.optim import AdamW

KINDS = [(8, False), (8, True), (32, False), (32, True)]


def params(seed=0, dtype=torch.float32, shapes=((40, 7), (130,))):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype)) for s in shapes]


def grads(ps, i):
    g = torch.Generator().manual_seed(100 + i)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).to(p.dtype)


def run(ps, opt, turns):
    for i in turns:
        grads(ps, i)
        opt.step()


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def same_state(a, pa, b, pb):
    for p, q in zip(pa, pb):
        assert a.state[p].keys() == b.state[q].keys()
        for k, x in a.state[p].items():
            assert torch.equal(x, b.state[q][k]) if isinstance(x, torch.Tensor) else x == b.state[q][k]


# ----------------------------------------------------------------------------- state from outside
@pytest.mark.parametrize("bits,master", KINDS)
def test_cleared_state_starts_anew(bits, master):
    ps = params()
    opt = AdamW(ps, lr=1e-2, state_bits=bits, master_weights=master)
    run(ps, opt, range(3))
    opt.state.clear()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = AdamW(qs, lr=1e-2, state_bits=bits, master_weights=master)
    run(ps, opt, [5, 6])
    run(qs, other, [5, 6])
    assert same(ps, qs)
    same_state(opt, ps, other, qs)


@pytest.mark.parametrize("how", ["tensor", "memory"])
@pytest.mark.parametrize("bits,master", KINDS)
def test_replaced_state_is_used_and_updated(bits, master, how):
    ps, qs = params(), params()
    opt, other = (AdamW(x, lr=1e-2, state_bits=bits, master_weights=master) for x in (ps, qs))
    run(ps, opt, range(3))
    run(qs, other, [7])
    for p, q in zip(ps, qs):                           # the other optimizer's state, as it is after one step
        p.data.copy_(q.data)
        for k, x in other.state[q].items():
            if isinstance(x, torch.Tensor) and how == "memory":
                opt.state[p][k].data = x.clone()
            else:
                opt.state[p][k] = x.clone() if isinstance(x, torch.Tensor) else x
    run(ps, opt, [8, 9])
    run(qs, other, [8, 9])
    assert same(ps, qs)
    same_state(opt, ps, other, qs)


def test_state_that_others_add_is_left_alone():
    """Entries of another's making, beside the parameters' and among their state, and state in another order."""
    ps, qs = params(), params()
    opt, other = AdamW(ps, lr=1e-2), AdamW(qs, lr=1e-2)
    for i in range(3):
        run(ps, opt, [i])
        run(qs, other, [i])
        opt.state["note"] = 1.5
        opt.state[ps[0]]["tag"] = 0.5
        opt.state[ps[1]] = dict(reversed(opt.state[ps[1]].items()))
    assert same(ps, qs) and opt.state["note"] == 1.5 and opt.state[ps[0]]["tag"] == 0.5


# ----------------------------------------------------------------------------- copies
@pytest.mark.parametrize("started", [False, True])
@pytest.mark.parametrize("how", [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
@pytest.mark.parametrize("bits,master", KINDS)
def test_copies_go_on_by_themselves(bits, master, how, started):
    ps = params()
    opt = AdamW(ps, lr=1e-2, state_bits=bits, master_weights=master)
    run(ps, opt, range(2 if started else 0))
    other = how(opt)
    qs = other.param_groups[0]["params"]
    before = [p.detach().clone() for p in ps]
    run(qs, other, [5, 6])
    assert same(ps, before)                            # the copy has its own tensors
    run(ps, opt, [5, 6])
    assert same(ps, qs)
    same_state(opt, ps, other, qs)


# ----------------------------------------------------------------------------- refusals
def _double(p):
    p.data = p.data.double()
    p.grad = torch.ones_like(p)


def _sparse(p):
    p.grad = torch.ones_like(p).to_sparse()


@pytest.mark.parametrize("started", [False, True])
@pytest.mark.parametrize("spoil", [_double, _sparse])
def test_a_refused_step_changes_nothing(spoil, started):
    ps, bad = params(), torch.nn.Parameter(torch.randn(30, 4))
    opt = AdamW([{"params": ps, "lr": 1e-2}, {"params": [bad]}], state_bits=8)
    if started:
        run(ps + [bad], opt, range(2))
    kept = bad.data
    grads(ps, 7)
    spoil(bad)
    before, state = [p.detach().clone() for p in ps], copy.deepcopy(opt.state_dict()["state"])
    with pytest.raises(ValueError):
        opt.step()
    assert same(ps, before)
    now = opt.state_dict()["state"]
    assert now.keys() == state.keys()
    for i, x in state.items():
        assert all(torch.equal(y, now[i][k]) if isinstance(y, torch.Tensor) else y == now[i][k] for k, y in x.items())
    bad.grad, bad.data = None, kept
    opt.step()
    assert [opt.state[p]["step"] for p in ps] == [3 if started else 1] * 2


# ----------------------------------------------------------------------------- random bits
@pytest.mark.parametrize("late", [False, True])
def test_groups_do_not_share_random_bits(late):
    """Two equal tensors, in two groups or at two step counts of one: codes that are rounded by independent bits differ
    in about a quarter of the places and more (a value within its step is uniform: 2 u (1 - u), 1/3 in the mean)."""
    w, g = torch.randn(2, 4096, generator=torch.Generator().manual_seed(2)).unbind()
    ps = [torch.nn.Parameter(w.clone()) for _ in range(2)]
    opt = AdamW(ps if late else [{"params": [p]} for p in ps], state_bits=8)
    if late:                                           # the second one has steps of its own from here on
        ps[0].grad = torch.zeros(4096)
        opt.step()
    ps[0].grad, ps[1].grad = g.clone(), g.clone()
    opt.step()
    if late:
        assert [opt.state[p]["step"] for p in ps] == [2, 1]
    off = (opt.state[ps[0]]["exp_avg"] != opt.state[ps[1]]["exp_avg"]).double().mean()
    assert float(off) > 0.2
    # and a parameter alone still takes the bits of its step
    alone = AdamW([torch.nn.Parameter(w.clone())], state_bits=8)
    alone.param_groups[0]["params"][0].grad = g.clone()
    alone.step()
    if not late:
        assert torch.equal(alone.state[alone.param_groups[0]["params"][0]]["exp_avg"], opt.state[ps[0]]["exp_avg"])


# ----------------------------------------------------------------------------- layouts
def check_layouts(bits, master, device="cpu"):
    """Parameters in other layouts are updated like their row-major copies, keep their layout, and state moves between."""
    def make(other):
        g = torch.Generator().manual_seed(4)
        x = [torch.randn(6, 5, 4, 3, generator=g).to(device), torch.randn(40, 30, generator=g).to(device),
             torch.randn(9, generator=g).to(device)]
        if other:
            x[0] = x[0].to(memory_format=torch.channels_last)
            x[1] = x[1].t().contiguous().t()
        ps = [torch.nn.Parameter(y) for y in x]
        return ps, AdamW(ps, lr=1e-2, state_bits=bits, master_weights=master)

    (ps, opt), (qs, other) = make(True), make(False)
    for i in range(2):
        for x, o in ((ps, opt), (qs, other)):
            g = torch.Generator().manual_seed(100 + i)
            for p in x:                                # a gradient in the parameter's layout
                p.grad = torch.empty_like(p).copy_(torch.randn(p.shape, generator=g))
            o.step()
    assert ps[0].is_contiguous(memory_format=torch.channels_last) and not ps[1].is_contiguous()
    assert same(ps, qs)
    same_state(opt, ps, other, qs)
    rs, third = make(True)
    third.load_state_dict(other.state_dict())
    for r, q in zip(rs, qs):
        r.data.copy_(q.data)
    for x, o in ((rs, third), (qs, other)):
        for p in x:
            p.grad = torch.empty_like(p).fill_(0.5)
        o.step()
    assert same(rs, qs)
    rs[1].data = rs[1].data.contiguous()               # and back to row-major in the middle
    for x, o in ((rs, third), (qs, other)):
        o.step()
    assert same(rs, qs)


@pytest.mark.parametrize("bits,master", KINDS)
def test_parameters_of_any_layout(bits, master):
    check_layouts(bits, master)


# ----------------------------------------------------------------------------- another optimizer's state
def stock_state(dtype=torch.float32, device="cpu", **kw):
    ps = [torch.nn.Parameter(p.detach().to(device)) for p in params(1, dtype)]
    ps[0].data = ps[0].data.t().contiguous().t()       # its moments have this layout too
    opt = torch.optim.AdamW(ps, lr=3e-3, weight_decay=0.1, **kw)
    run_on(ps, opt, range(4))
    return ps, opt


def run_on(ps, opt, turns):
    for i in turns:
        g = torch.Generator().manual_seed(100 + i)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(p)
        opt.step()


def check_stock_state(bits, master, dtype, device="cpu"):
    qs, stock = stock_state(dtype, device)
    ps = [torch.nn.Parameter(q.detach().clone(memory_format=torch.contiguous_format)) for q in qs]
    opt = AdamW(ps, state_bits=bits, master_weights=master)
    opt.load_state_dict(stock.state_dict())
    assert opt.param_groups[0]["lr"] == 3e-3 and opt.param_groups[0]["state_bits"] == bits
    for p, q in zip(ps, qs):
        assert opt.state[p]["step"] == 4
        for name in ("exp_avg", "exp_avg_sq"):
            want = stock.state[q][name].double().reshape(-1)
            if bits == 32:
                assert torch.equal(opt.state[p][name].double().reshape(-1), want)
                continue
            want = want if name == "exp_avg" else want.sqrt()
            got = opt._moment(p, name, opt.param_groups[0])
            # half a step: 2^-4 of the value, 2^-10 of the scale below the smallest normal code, and a root's code 1
            low = got.scale.double().repeat_interleave(128)[: p.numel()] * 2.0 ** (-10 if name == "exp_avg" else -9)
            assert bool(((got.values().double() - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, low) * (1 + 1e-6)).all())
    before = [(p.detach().double(), *(stock.state[q][name].double() for name in ("exp_avg", "exp_avg_sq")))
              for p, q in zip(ps, qs)]
    run_on(ps, opt, [9])
    run_on(qs, stock, [9])
    lr, c1, c2 = 3e-3, 1 - 0.9 ** 5, (1 - 0.999 ** 5) ** 0.5
    for p, q, (w, m, v) in zip(ps, qs, before):
        # One step from equal weights.  8 bits: exp_avg off by 1/16 of itself (or 2^-10 of a scale, at most its block's
        # largest / 224), the root by 1/16 of itself.  Then the roundings: the weight to its type on either side, the
        # stock one's bf16 state (half a step of 2^-8 on m and v each), and 32 for fp32.
        g = p.grad.double()
        m1, r1 = 0.9 * m + 0.1 * g, (0.999 * v + 0.001 * g * g).sqrt()
        update = lr / c1 * m1.abs() / (r1 / c2)
        dm = 0.9 * torch.maximum(m.abs() / 16, m.abs().max() / 224 * 2.0 ** -10) if bits == 8 else torch.zeros_like(m)
        tol = lr / c1 * dm / (r1 * 15 / 16 / c2) + (update / 15 if bits == 8 else 0)
        half = torch.finfo(dtype).eps / 2
        tol += 4 * half * (w.abs() + lr) + 3 * half * lr / c1 * (m1.abs() + 0.9 * m.abs()) / (r1 / c2) + 32 * 2.0 ** -24 * (w.abs() + update)
        assert not torch.equal(p.double(), w)
        assert bool(((p.double() - q.double()).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits,master", KINDS)
def test_the_stock_optimizers_saved_state(bits, master, dtype):
    check_stock_state(bits, master, dtype)


def test_saved_state_of_other_rules_is_refused():
    ps = params(1)
    opt = AdamW(ps, lr=1e-2)
    run(ps, opt, [0])
    before = copy.deepcopy(opt.state_dict())
    for sd in (stock_state(amsgrad=True)[1].state_dict(), stock_state(maximize=True)[1].state_dict()):
        with pytest.raises(ValueError):
            opt.load_state_dict(sd)
    adam = torch.optim.Adam(params(1), weight_decay=0.1)
    sgd = torch.optim.SGD(params(1), lr=0.1, momentum=0.9)
    for other in (adam, sgd):
        run(other.param_groups[0]["params"], other, [0])
        with pytest.raises(ValueError):
            opt.load_state_dict(other.state_dict())
    now = opt.state_dict()
    assert now["param_groups"] == before["param_groups"]
    assert all(torch.equal(x, now["state"][i][k]) for i, st in before["state"].items() for k, x in st.items() if k != "step")


def test_a_captured_step_is_refused(monkeypatch):
    ps = params()
    opt = AdamW(ps)
    grads(ps, 0)
    before = [p.detach().clone() for p in ps]
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    monkeypatch.undo()
    assert same(ps, before) and not opt.state
    opt.step()
    assert opt.state[ps[0]]["step"] == 1
