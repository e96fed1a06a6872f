"""AdamW over many tensors on the CPU, and what it refuses."""
import pytest
import torch

from shift_b200.ops import reference as ref
from shift_b200.optim import AdamWMany, State8

SIZES = [(1,), (127,), (128,), (3, 43), (1000,), (5, 0), (700,)]


def make(dtype, eight, master, device="cpu", sizes=SIZES, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = [torch.randn(s, generator=g) for s in sizes]
    params = [x.to(dtype).to(device) for x in w]
    grads = [(torch.randn(s, generator=g) * 10 ** float(torch.randn(1, generator=g))).to(device) for s in sizes]
    m = [torch.randn(s, generator=g) * 0.1 for s in sizes]
    r = [torch.rand(s, generator=g) + 1e-3 for s in sizes]
    if eight:
        m = [State8(*ref.moment_encode(x.reshape(-1), torch.zeros(x.numel(), dtype=torch.int64))) for x in m]
        v = [State8(*ref.moment_encode(x.reshape(-1), torch.zeros(x.numel(), dtype=torch.int64))) for x in r]
        m, v = ([State8(s.code.to(device), s.scale.to(device)) for s in x] for x in (m, v))
    else:
        m, v = [x.to(device) for x in m], [x.square().to(device) for x in r]
    masters = [x.clone().to(device) for x in w] if master else None
    return params, grads, m, v, masters


def expected(params, grads, m, v, masters, lr, b1, b2, eps, wd, step, scale):
    """The update in 64 bits: weights, exp_avg, exp_avg_sq (each flat)."""
    out = []
    for t, p in enumerate(params):
        w = (p if masters is None else masters[t]).double().reshape(-1)
        g = grads[t].double().reshape(-1) * scale
        if isinstance(m[t], State8):
            pad = lambda s: torch.repeat_interleave(s.scale.double(), 128)[: p.numel()]  # noqa: E731
            m0, v0 = m[t].code.double() * pad(m[t]), (v[t].code.double() * pad(v[t])) ** 2
        else:
            m0, v0 = m[t].double().reshape(-1), v[t].double().reshape(-1)
        m1 = b1 * m0 + (1 - b1) * g
        v1 = b2 * v0 + (1 - b2) * g * g
        w1 = w * (1 - lr * wd) - lr * (m1 / (1 - b1 ** step)) / ((v1 / (1 - b2 ** step)).sqrt() + eps)
        # magnitudes of what was added, for the error of cancelling sums
        out.append((w1, m1, v1, w.abs() + lr * (b1 * m0.abs() + (1 - b1) * g.abs()) / (1 - b1 ** step)
                    / ((v1 / (1 - b2 ** step)).sqrt() + eps), b1 * m0.abs() + (1 - b1) * g.abs()))
    return out


H = dict(lr=3e-2, beta1=0.9, beta2=0.99, eps=1e-8, wd=0.1)


def check(opt, params, grads, masters, want):
    """A weight takes about ten roundings to fp32, a moment four: 16 and 8 half steps of 2^-24 of the magnitudes
    that are added, and the float hyper-parameters (2^-24 each) as many again; then half a step of the parameter's
    type: eps / 2 of the value, and of the smallest normal number below that (fp16's steps stay 2^-24 apart under
    2^-14, so half a step is 2^-25 = 2^-14 * 2^-11 for a weight of any smaller size).  An 8-bit moment lies within one step (2^-3 relative, or 2^-9 of its scale) of the exact value."""
    for t, (w1, m1, v1, wmag, mmag) in enumerate(want):
        w = (params[t] if masters is None else masters[t]).double().reshape(-1)
        half, tiny = torch.finfo(params[t].dtype).eps / 2, torch.finfo(params[t].dtype).smallest_normal
        tol = 32 * 2.0 ** -24 * wmag
        assert bool(((w - w1).abs() <= tol + (half * w1.abs().clamp(min=tiny) if masters is None else 0)).all())
        if masters is not None:
            assert torch.equal(params[t], masters[t].to(params[t].dtype))
        if not opt.eight:
            assert bool(((opt.exp_avg[t].double().reshape(-1) - m1).abs() <= 16 * 2.0 ** -24 * mmag).all())
            assert bool(((opt.exp_avg_sq[t].double().reshape(-1) - v1).abs() <= 16 * 2.0 ** -24 * v1).all())
            continue
        for s, x in ((opt.exp_avg[t], m1), (opt.exp_avg_sq[t], v1.sqrt())):
            step = torch.maximum(x.abs() / 8, s.scale.double().repeat_interleave(128)[: x.numel()] * 2.0 ** -9)
            code = s.code.double() * s.scale.double().repeat_interleave(128)[: x.numel()]
            assert bool(((code - x).abs() <= step * (1 + 1e-5)).all())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True), (torch.bfloat16, False),
                                          (torch.float16, True)])
def test_step_against_64_bits(dtype, master, eight):
    params, grads, m, v, masters = make(dtype, eight, master)
    opt = AdamWMany(params, m, v, masters)
    for step in (1, 2, 50):
        want = expected(params, grads, m, v, masters, *H.values(), step, 0.5)
        opt.step(grads, step=step, grad_scale=0.5, **H)
        check(opt, params, grads, masters, want)


def test_rounding_is_unbiased_and_follows_the_seed():
    n = 1 << 16
    x = torch.full((n,), 1.03)
    x[0] = 1.0
    u = ref.moment_draws(n, 5, 0)
    code, scale = ref.moment_encode(x, u & 0xFFFF)
    got = code.double() * float(scale[0].float())
    # two neighbouring codes, 2^-3 apart; the mean of n draws is off by at most 6 standard deviations of step / (2 sqrt n)
    assert set(got[1:].unique().tolist()) == {1.0, 1.125}
    assert abs(float(got[1:].mean()) - 1.03) < 6 * 0.125 / 2 / n ** 0.5
    assert not torch.equal(u, ref.moment_draws(n, 6, 0)) and not torch.equal(u, ref.moment_draws(n, 5, 1))
    assert bool(((u & 0xFFFF).double().mean() / 65535 - 0.5).abs() < 6 * 0.29 / n ** 0.5)
    assert bool(((u >> 16).double().mean() / 65535 - 0.5).abs() < 6 * 0.29 / n ** 0.5)


def test_skip_nonfinite_and_device_scalars():
    import math
    params, grads, m, v, masters = make(torch.float32, True, False)
    opt = AdamWMany(params, m, v)
    before = [p.clone() for p in params]
    opt.step(grads, skip=torch.ones(1, dtype=torch.int32), **H)
    assert all(torch.equal(a, b) for a, b in zip(before, params))
    flag = torch.zeros(1, dtype=torch.int32)
    grads[1][3] = math.inf
    opt.step(grads, skip=torch.zeros(1, dtype=torch.int32), nonfinite=flag, **H)
    assert int(flag) == 1
    one, two = (make(torch.float32, True, False) for _ in range(2))
    AdamWMany(one[0], one[2], one[3]).step(one[1], step=7, seed=3, **H)
    block = torch.zeros(8, dtype=torch.int32)
    block[0] = 3
    block[1:4] = torch.tensor([H["lr"], 1 - H["beta1"] ** 7, math.sqrt(1 - H["beta2"] ** 7)]).view(torch.int32)
    AdamWMany(two[0], two[2], two[3]).step(two[1], step=1, step_dev=block, **{**H, "lr": 9.0})
    assert all(torch.allclose(a, b, rtol=1e-6, atol=0) for a, b in zip(one[0], two[0]))
    assert all(torch.equal(a.code.view(torch.uint8), b.code.view(torch.uint8)) for a, b in zip(one[2], two[2]))


def test_refusals():
    params, grads, m, v, masters = make(torch.float32, False, False)
    m8 = [State8.zeros(p) for p in params]
    for bad in (lambda: AdamWMany(params, m[:-1], v), lambda: AdamWMany(params, m8, v),
                lambda: AdamWMany(params, m, v, masters=params[:-1]),
                lambda: AdamWMany([p.double() for p in params], m, v),
                lambda: AdamWMany(params, [x.half() for x in m], v),
                lambda: AdamWMany([p.t() if p.dim() == 2 else p for p in params],
                                  [x.t() if x.dim() == 2 else x for x in m], v),
                lambda: AdamWMany(params + params[:1], m + m[:1], v + v[:1]), lambda: AdamWMany(params, m, m),
                lambda: AdamWMany(params, m8, [s._replace(scale=s.scale[:0]) for s in m8]),
                lambda: AdamWMany(params, m, v).step(grads[:-1]), lambda: AdamWMany(params, m, v).step(grads, step=0),
                lambda: AdamWMany(params, m, v).step([g.double() for g in grads]),
                lambda: AdamWMany(params, m, v).step(grads, skip=torch.zeros(1)),
                lambda: AdamWMany(params, m, v).step(grads, step_dev=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()
    AdamWMany([], [], []).step([])


@pytest.mark.parametrize("bits,master", [(8, False), (8, True), (32, True)])
def test_torch_optimizer_and_its_saved_state(bits, master):
    from shift_b200.optim import AdamW

    def model():
        torch.manual_seed(3)
        net = torch.nn.Sequential(torch.nn.Linear(40, 30), torch.nn.Linear(30, 7, bias=False)).to(torch.bfloat16)
        return net, AdamW(net.parameters(), lr=1e-2, state_bits=bits, master_weights=master)

    def grads(net, i):
        g = torch.Generator().manual_seed(i)
        for j, p in enumerate(net.parameters()):
            # the second tensor has no gradient in the first step: its count then lags behind
            p.grad = None if i == 0 and j == 1 else torch.randn(p.shape, generator=g).to(p.dtype)

    net, opt = model()
    for i in range(3):
        grads(net, i)
        opt.step()
    steps = [opt.state[p]["step"] for p in net.parameters()]
    assert steps == [3, 2, 3]
    twin, other = model()
    twin.load_state_dict(net.state_dict())
    other.load_state_dict(opt.state_dict())
    for a, b in zip(net.parameters(), twin.parameters()):
        for k, x in opt.state[a].items():
            assert (torch.equal(x, other.state[b][k]) and x.dtype == other.state[b][k].dtype) if k != "step" \
                else x == other.state[b][k]
    for i in range(3, 5):
        for n, o in ((net, opt), (twin, other)):
            grads(n, i)
            o.step()
    assert all(torch.equal(a, b) for a, b in zip(net.parameters(), twin.parameters()))


def test_torch_optimizer_follows_the_stock_one_with_32_bit_state():
    from shift_b200.optim import AdamW
    torch.manual_seed(4)
    a = [torch.nn.Parameter(torch.randn(50, 3)), torch.nn.Parameter(torch.randn(129))]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ours, stock = AdamW(a, lr=1e-2, state_bits=32), torch.optim.AdamW(b, lr=1e-2)
    for i in range(5):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape)
            q.grad = p.grad.clone()
        ours.step()
        stock.step()
    # both round each of five updates of at most 1e-2 and the weight a dozen times in fp32
    for p, q in zip(a, b):
        assert bool(((p - q).abs() <= 5 * 12 * 2.0 ** -24 * (q.abs() + 0.05)).all())
