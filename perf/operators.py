"""The operators of an 8-bit training step, as measured cases.

Three operators, each in a plain form of elementary torch operations
(``own = False``) and through the framework's kernels (``own = True``):

* ``quantize``  bf16/fp16/fp32 matrices to 8-bit floating point with one
  power-of-two scale per block of 128, along the rows, along the columns
  (the transposed copy that a backward pass contracts) or per 128 x 128 tile;
* ``matmul`` / ``experts`` / ``experts_wgrad``  products of two such matrices,
  dense, with rows grouped by expert, and with the contraction grouped by
  expert (the experts' weight gradients);
* ``adamw``  one AdamW update of many tensors, with the moments in 32 bits or
  in 8 bits per value and a scale per block of 128.

The 8-bit matrix is ``data`` [rows, round_up(cols, 16)] with ``scale``
[ceil(cols / 512), rows, 4]: byte j of word (w, r) is the exponent (biased by
127) of the scale of columns [512 w + 128 j, + 128) of row r.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a ragged last batch of gradients, both orientations, range before precision
        dict(name="quantize-ragged-e5m2", op="quantize", groups=1, rows=4093, cols=1000, dtype="bf16", fmt="e5m2",
             tiles=False, both=True),
        # the step's activations (8 x 2048 tokens, hidden 1024): forward and weight-gradient copies in one pass
        dict(name="quantize-activations", op="quantize", groups=1, rows=16384, cols=1024, dtype="bf16", fmt="e4m3",
             tiles=False, both=True),
        # one token against the head's weight: latency and the weight's bytes
        dict(name="matmul-one-token-head", op="matmul", m=1, n=32768, k=1024, fmt_a="e4m3", fmt_b="e4m3", out="bf16",
             accumulate=False),
        # odd sizes on all three sides, gradient type against value type
        dict(name="matmul-odd", op="matmul", m=4093, n=1000, k=2061, fmt_a="e5m2", fmt_b="e4m3", out="bf16",
             accumulate=False),
        # the fused QKV projection over a whole step's tokens
        dict(name="matmul-qkv", op="matmul", m=16384, n=1536, k=1024, fmt_a="e4m3", fmt_b="e4m3", out="bf16",
             accumulate=False),
        # its weight gradient, added to the microbatches' fp32 sum
        dict(name="matmul-qkv-wgrad", op="matmul", m=1536, n=1024, k=16384, fmt_a="e5m2", fmt_b="e4m3", out="f32",
             accumulate=True),
        # the largest product: a square one, bound by the tensor cores
        dict(name="matmul-8192", op="matmul", m=8192, n=8192, k=8192, fmt_a="e4m3", fmt_b="e4m3", out="bf16",
             accumulate=False),
        # the experts' first projection: 16384 tokens to 4 of 16 experts each, uneven bins
        dict(name="experts-w1", op="experts", tokens=16384, top_k=4, experts=16, n=1344, k=1024, skew=0.5),
        # the weight gradient of their second projection
        dict(name="experts-w2-wgrad", op="experts_wgrad", tokens=16384, top_k=4, experts=16, n=1024, k=672, skew=0.5),
        # the tiny model's tensors, 8-bit moments: few elements, many tensors
        dict(name="adamw-tiny-8bit", op="adamw", model="tiny", vocab=1024, hidden=256, layers=2, qkv=768, attn=256,
             experts=8, ffn=256, dtype="bf16", grad="bf16", master=True, bits=8, packed=False),
        # the 0.494B model's tensors with 32-bit moments
        dict(name="adamw-bench-32bit", op="adamw", model="bench", vocab=32768, hidden=1024, layers=12, qkv=1536,
             attn=1024, experts=16, ffn=672, dtype="bf16", grad="bf16", master=True, bits=32, packed=False),
        # the same with 8-bit moments
        dict(name="adamw-bench-8bit", op="adamw", model="bench", vocab=32768, hidden=1024, layers=12, qkv=1536,
             attn=1024, experts=16, ffn=672, dtype="bf16", grad="bf16", master=True, bits=8, packed=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "experts", "experts_wgrad", "adamw"])
    if op == "quantize":
        tiles = rng.random() < 0.4
        groups = rng.choice([1, 1, _log_int(rng, 2, 16)]) if tiles else 1
        while True:
            rows, cols = _log_int(rng, 1, 65536), _log_int(rng, 16, 16384)
            if groups * rows * cols <= 1 << 26:
                break
        return dict(op=op, groups=groups, rows=rows, cols=cols, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    fmt=rng.choice(["e4m3", "e5m2"]), tiles=tiles, both=rng.random() < 0.7)
    if op == "matmul":
        while True:
            m, n, k = _log_int(rng, 1, 32768), _log_int(rng, 16, 32768), _log_int(rng, 16, 32768)
            if m * n <= 1 << 27 and m * k <= 1 << 27 and n * k <= 1 << 27 and m * n * k <= 8192 ** 3:
                break
        out = rng.choice(["bf16", "bf16", "f32"])
        return dict(op=op, m=m, n=n, k=k, fmt_a=rng.choice(["e4m3", "e5m2"]), fmt_b=rng.choice(["e4m3", "e5m2"]),
                    out=out, accumulate=out == "f32" and rng.random() < 0.5)
    if op in ("experts", "experts_wgrad"):
        while True:
            tokens, top_k, experts = _log_int(rng, 1, 16384), rng.randint(1, 8), rng.randint(1, 64)
            n, k = 16 * _log_int(rng, 2, 256), 16 * _log_int(rng, 2, 256)
            rows = tokens * top_k + 128 * experts
            if rows * n * k <= 16384 * 4 * 4096 * 1024 and rows * max(n, k) <= 1 << 28 and experts * n * k <= 1 << 27:
                break
        return dict(op=op, tokens=tokens, top_k=min(top_k, experts), experts=experts, n=n, k=k,
                    skew=round(rng.uniform(0.0, 2.0), 3))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    return dict(op=op, model="mix", tensors=_log_int(rng, 1, 160), numel=_log_int(rng, 4096, 1 << 27),
                spread=round(rng.uniform(0.5, 2.5), 3), mix=rng.randrange(1 << 30), dtype=dtype,
                grad=rng.choice([dtype, "f32"]), master=dtype != "f32" and rng.random() < 0.6,
                bits=rng.choice([8, 32]), packed=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ 8-bit matrices, plain
def _block_scale(amax, fmt):
    """Biased exponent (uint8) of the smallest power of two that brings `amax` (fp32, >= 0) within the type's largest
    value, and the reciprocal of that power of two."""
    top = 8 if fmt == "e4m3" else 15                                        # largest value 1.75 * 2^top
    mant, ex = torch.frexp(amax)                                            # amax = mant * 2^ex, mant in [0.5, 1)
    e = ex - 1 - top + (mant > 0.875).to(torch.int32)
    e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 127)
    inv = ((127 - e) << 23).to(torch.int32).view(torch.float32)
    return (e + 127).to(torch.uint8), inv


def _pack_scales(b):
    """[rows, blocks] bytes -> [ceil(blocks / 4), rows, 4]."""
    rows, nb = b.shape
    b = torch.nn.functional.pad(b, (0, -nb % 4))
    return b.view(rows, -1, 4).permute(1, 0, 2).contiguous().view(torch.float8_e8m0fnu)


def _finite_abs(x):
    a = x.abs()
    return torch.where(torch.isfinite(a), a, torch.zeros_like(a))


def _store_codes(x, inv, fmt):
    """x [rows, cols] fp32 times inv [rows, cols], rounded once, in rows of a multiple of 16 bytes."""
    rows, cols = x.shape
    data = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=x.device).view(F8[fmt])
    data[:, :cols] = (x * inv).to(F8[fmt])
    return data


def _plain_rows(x, fmt):
    """[rows, cols] -> (data, scale), one scale per row and 128 columns."""
    rows, cols = x.shape
    x = x.float()
    nb = -(-cols // 128)
    a = torch.nn.functional.pad(_finite_abs(x), (0, nb * 128 - cols)).view(rows, nb, 128).amax(-1)
    b, inv = _block_scale(a, fmt)
    return _store_codes(x, inv.repeat_interleave(128, 1)[:, :cols], fmt), _pack_scales(b)


def _plain_tiles(x, fmt, both):
    """[groups, rows, cols] -> (data, scale) and, if asked, those of each group's transpose; one scale per 128 x 128."""
    g, rows, cols = x.shape
    x = x.float()
    rb, cb = -(-rows // 128), -(-cols // 128)
    a = torch.nn.functional.pad(_finite_abs(x), (0, cb * 128 - cols, 0, rb * 128 - rows))
    a = a.view(g, rb, 128, cb, 128).amax((2, 4))
    b, inv = _block_scale(a, fmt)
    wide = inv.repeat_interleave(128, 1)[:, :rows].repeat_interleave(128, 2)[:, :, :cols]
    got = [(_store_codes(x.reshape(g * rows, cols), wide.reshape(g * rows, cols), fmt),
            _pack_scales(b.repeat_interleave(128, 1)[:, :rows].reshape(g * rows, cb)))]
    if both:
        bt = b.transpose(1, 2).repeat_interleave(128, 1)[:, :cols]
        got.append((_store_codes(x.transpose(1, 2).reshape(g * cols, rows),
                                 wide.transpose(1, 2).reshape(g * cols, rows), fmt),
                    _pack_scales(bt.reshape(g * cols, rb))))
    return got


def _plain_quantize(x, fmt, tiles, both):
    if tiles:
        return _plain_tiles(x if x.dim() == 3 else x[None], fmt, both)
    got = [_plain_rows(x, fmt)]
    if both:
        got.append(_plain_rows(x.t().contiguous(), fmt))
    return got


def _values(data, scale, cols):
    """The fp32 values that an 8-bit matrix stands for (finite ones exactly)."""
    s = scale.view(torch.uint8).permute(1, 0, 2).reshape(data.shape[0], -1).to(torch.int32)
    s = torch.where(s > 0, s << 23, torch.full_like(s, 1 << 22)).view(torch.float32)      # 2^(byte - 127)
    return data[:, :cols].float() * s.repeat_interleave(128, 1)[:, :cols]


# ------------------------------------------------------------------------------------------------ AdamW, plain
def _mix32(h):
    h = h & MASK32
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & MASK32
    h = ((h ^ (h >> 15)) * 0x846CA68B) & MASK32
    return h ^ (h >> 16)


def _draws(n, seed, tensor, device):
    """32 uniform bits for each element, from the step's seed and the tensor's number."""
    key = _mix32(_mix32(torch.tensor([seed])) ^ (tensor * 0x9E3779B1)).item()
    return _mix32(torch.arange(n, dtype=torch.int64, device=device) * 0x9E3779B1 + key)


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % 128)).view(-1, 128)


def _decode(code, scale):
    s = scale.view(torch.uint8).to(torch.int32)
    s = torch.where(s > 0, s << 23, torch.full_like(s, 1 << 22)).view(torch.float32)
    return code.float() * s.repeat_interleave(128)[: code.numel()]


def _encode(x, bits16, code, scale):
    """x fp32 -> 8-bit codes and block scales, in place, each magnitude rounded up with the probability of its
    distance from the value below (16 random bits each)."""
    n = x.numel()
    b, inv = _block_scale(_blocks(_finite_abs(x)).amax(-1), "e4m3")
    y = (x * inv.repeat_interleave(128)[:n]).abs()
    small = y < 2.0 ** -6
    t = torch.where(small, y + 2.0 ** -6, y)
    t = ((t.view(torch.int32) + (bits16 << 4).to(torch.int32)) & ~0xFFFFF).view(torch.float32)
    t = torch.where(small, t - 2.0 ** -6, t)
    t = torch.where(torch.isfinite(x), torch.copysign(t, x), torch.full_like(t, math.nan))
    code.copy_(t.to(torch.float8_e4m3fn))
    scale.copy_(b.view(torch.float8_e8m0fnu))


HYPER = dict(lr=1.0e-4, beta1=0.9, beta2=0.999, eps=1.0e-8, wd=0.01)


def _plain_adamw(s, step, seed):
    h = HYPER
    bc1, bc2 = 1.0 - h["beta1"] ** step, math.sqrt(1.0 - h["beta2"] ** step)
    for t, (p, g, m, v) in enumerate(zip(s["params"], s["grads"], s["m"], s["v"])):
        w = (s["masters"][t] if s["masters"] else p).float()
        g = g.float() * s["grad_scale"]
        eight = s["bits"] == 8
        m32 = _decode(*m) if eight else m
        v32 = _decode(*v).square() if eight else v
        m32 = m32 + (g - m32) * (1.0 - h["beta1"])
        v32 = v32 * h["beta2"] + (1.0 - h["beta2"]) * g * g
        r = v32.sqrt()
        w = w * (1.0 - h["lr"] * h["wd"]) - (h["lr"] / bc1) * (m32 / (r / bc2 + h["eps"]))
        if eight:
            u = _draws(g.numel(), seed, t, g.device)
            _encode(m32, u & 0xFFFF, *m)
            _encode(r, u >> 16, *v)
        else:
            m.copy_(m32)
            v.copy_(v32)
        if s["masters"]:
            s["masters"][t].copy_(w)
        p.copy_(w.to(p.dtype))


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def _activations(g, *shape, dtype=torch.bfloat16):
    """Rows of very different size, a few loud columns, some rows of padding (zeros)."""
    x = torch.randn(*shape, device=DEV, generator=g)
    x *= torch.exp(torch.randn(*shape[:-1], 1, device=DEV, generator=g))
    x *= 1.0 + 20.0 * (torch.rand(shape[-1], device=DEV, generator=g) < 0.01)
    x *= (torch.rand(*shape[:-1], 1, device=DEV, generator=g) > 0.02) | (shape[-2] < 64)
    return x.to(dtype)


def _bins(case, seed):
    """Segment offsets of the experts' bins, each padded to 128 rows, and the number of valid rows in each."""
    rng = random.Random(seed * 7919 + 17)
    e, total = case["experts"], case["tokens"] * case["top_k"]
    w = [math.exp(rng.gauss(0.0, case["skew"])) for _ in range(e)]
    # no expert has more than the tokens there are; what is cut off goes to the others in turn
    counts = [min(case["tokens"], int(total * x / sum(w))) for x in w]
    left, i = total - sum(counts), 0
    while left > 0:
        add = min(left, case["tokens"] - counts[i % e], -(-left // e))
        counts[i % e] += add
        left, i = left - add, i + 1
    offs = [0]
    for c in counts:
        offs.append(offs[-1] + -(-c // 128) * 128)
    return offs, counts


def _shapes(case):
    if case["model"] == "mix":
        rng = random.Random(case["mix"])
        w = [math.exp(rng.gauss(0.0, case["spread"])) for _ in range(case["tensors"])]
        return [max(1, int(case["numel"] * x / sum(w))) for x in w]
    H, F, E = case["hidden"], case["ffn"], case["experts"]
    layer = [H, case["qkv"] * H, H * case["attn"], H, E * H, E * 2 * F * H, E * H * F]
    return [case["vocab"] * H] + layer * case["layers"] + [H, case["vocab"] * H]


def _prepare_adamw(case, seed):
    g = _gen(seed)
    sizes = _shapes(case)
    step = 1 if case["packed"] else 128
    offs = [0]
    for n in sizes:
        offs.append(offs[-1] + -(-n // step) * step)
    total = offs[-1]
    views = lambda flat: [flat[o:o + n] for o, n in zip(offs, sizes)]  # noqa: E731
    w = _normal(g, total, std=0.02)
    flat = {"param": w.to(TYPES[case["dtype"]])}
    if case["master"]:
        flat["master"] = w
    grad = _normal(g, total, dtype=TYPES[case["grad"]], std=1.0e-2)
    m0 = _normal(g, total, std=3.0e-3)
    r0 = _normal(g, total, std=1.0e-2).abs_() + 1.0e-6
    s = {"bits": case["bits"], "flat": flat, "params": views(flat["param"]), "grads": views(grad),
         "masters": views(flat["master"]) if case["master"] else None, "grad_scale": 0.5, "step": 100, "seed": seed}
    if case["bits"] == 32:
        flat["m"], flat["v"] = m0, r0.square_()
        s["m"], s["v"] = views(flat["m"]), views(flat["v"])
        return s
    nb = [-(-n // 128) for n in sizes]
    at = [sum(nb[:i]) for i in range(len(nb))]
    for name, x in (("m", m0), ("v", r0)):
        flat[name] = torch.zeros(total, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        flat[name + "_scale"] = torch.zeros(sum(nb), dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
        s[name] = [(c, flat[name + "_scale"][a:a + b]) for c, a, b in zip(views(flat[name]), at, nb)]
        for t, (y, (code, scale)) in enumerate(zip(views(x), s[name])):
            _encode(y, _draws(y.numel(), seed + 99, t, DEV) & 0xFFFF, code, scale)
    return s


def prepare(case, seed):
    op = case["op"]
    if op == "adamw":
        return {"op": op, **_prepare_adamw(case, seed)}
    g = _gen(seed)
    if op == "quantize":
        shape = (case["rows"], case["cols"]) if case["groups"] == 1 else (case["groups"], case["rows"], case["cols"])
        make = _normal if case["tiles"] else _activations
        return {"op": op, "x": make(g, *shape, dtype=TYPES[case["dtype"]]), "fmt": case["fmt"],
                "tiles": case["tiles"], "both": case["both"]}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        a = _plain_rows(_activations(g, m, k), case["fmt_a"])
        b = _plain_rows(_normal(g, n, k, std=0.02), case["fmt_b"])
        s = {"op": op, "a": a, "b": b, "k": k, "dtype": TYPES[case["out"]]}
        if case["accumulate"]:
            s["acc"] = _normal(g, m, n)
        return s
    offs, counts = _bins(case, seed)
    cap = case["tokens"] * case["top_k"] + 127 * case["experts"]
    cap = max(cap, offs[-1])
    live = torch.ones(cap, 1, dtype=torch.bool, device=DEV)         # rows behind the last bin hold whatever they hold
    for o, c, end in zip(offs, counts, offs[1:]):
        live[o + c:end] = False
    s = {"op": op, "offs": torch.tensor(offs, dtype=torch.int32, device=DEV), "host_offs": offs}
    x = _activations(g, cap, case["k"]) * live
    if op == "experts":
        w = _normal(g, case["experts"], case["n"], case["k"], std=0.02)
        s.update(a=_plain_rows(x, "e4m3"), b=_plain_tiles(w, "e4m3", False)[0], k=case["k"],
                 out=torch.zeros(cap, case["n"], dtype=torch.bfloat16, device=DEV))
        return s
    dy = _normal(g, cap, case["n"], std=1.0e-3) * live
    s.update(a=_plain_rows(dy.t().contiguous(), "e5m2"), b=_plain_rows(x.t().contiguous(), "e4m3"), k=cap,
             out=torch.zeros(case["experts"], case["n"], case["k"], dtype=torch.bfloat16, device=DEV))
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _run_own(s):
    op = s["op"]
    if op == "adamw":
        from shift_b200.optim import AdamWMany, State8
        if "opt" not in s:
            wrap = (lambda x: [State8(*y) for y in x]) if s["bits"] == 8 else list
            s["opt"] = AdamWMany(s["params"], wrap(s["m"]), wrap(s["v"]), masters=s["masters"])
        s["opt"].step(s["grads"], step=s["step"], grad_scale=s["grad_scale"], seed=s["seed"], **HYPER)
        return s["flat"]
    from shift_b200.ops import fp8
    if op == "quantize":
        q = fp8.quantize(s["x"], s["fmt"], tiles=s["tiles"], both=s["both"])
        return [(t.data[:, :t.cols], t.scale) for t in (q if s["both"] else (q,))]
    a, b = (fp8.BlockFp8(*s[x], s["k"]) for x in "ab")
    if op == "matmul":
        if "acc" in s:
            return fp8.matmul(a, b, out=s["acc"], accumulate=True)
        return fp8.matmul(a, b, out_dtype=s["dtype"])
    if op == "experts":
        return fp8.grouped_matmul(a, b, s["offs"], out=s["out"])
    return fp8.grouped_wgrad(a, b, s["offs"], s["out"])


def _run_plain(s):
    op = s["op"]
    if op == "adamw":
        _plain_adamw(s, s["step"], s["seed"])
        return s["flat"]
    if op == "quantize":
        x = s["x"]
        cols = (x.shape[-1], x.shape[-2])
        return [(d[:, :c], e) for (d, e), c in zip(_plain_quantize(x, s["fmt"], s["tiles"], s["both"]), cols)]
    a, b = _values(*s["a"], s["k"]), _values(*s["b"], s["k"])
    if op == "matmul":
        if "acc" in s:
            return s["acc"].add_(a @ b.t())
        return (a @ b.t()).to(s["dtype"])
    offs, out = s["host_offs"], s["out"]
    if op == "experts":
        n = b.shape[0] // (len(offs) - 1)
        for e in range(len(offs) - 1):
            out[offs[e]:offs[e + 1]] = a[offs[e]:offs[e + 1]] @ b[e * n:(e + 1) * n].t()
        return out
    for e in range(len(offs) - 1):
        out[e] = a[:, offs[e]:offs[e + 1]] @ b[:, offs[e]:offs[e + 1]].t()
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass needs
def _bytes8(rows, cols):
    return rows * cols + rows * 4 * -(-cols // 512)


def work(case):
    op = case["op"]
    if op == "quantize":
        g, r, c = case["groups"], case["rows"], case["cols"]
        size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
        return {"bytes": g * (r * c * size + _bytes8(r, c) + (_bytes8(c, r) if case["both"] else 0)), "flops": 0}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        size = (2 if case["out"] == "bf16" else 4) * (2 if case["accumulate"] else 1)
        return {"bytes": _bytes8(m, k) + _bytes8(n, k) + m * n * size, "flops": 2 * m * n * k}
    if op == "adamw":
        n = sum(_shapes(case))
        size = {"bf16": 2, "f16": 2, "f32": 4}
        state = 16 if case["bits"] == 32 else 4 + 4 / 128
        weights = (8 + size[case["dtype"]]) if case["master"] else 2 * size[case["dtype"]]
        return {"bytes": n * (weights + size[case["grad"]] + state), "flops": 15 * n}
    rows, e, n, k = case["tokens"] * case["top_k"], case["experts"], case["n"], case["k"]
    if op == "experts":
        return {"bytes": _bytes8(rows, k) + _bytes8(e * n, k) + 2 * rows * n, "flops": 2 * rows * n * k}
    return {"bytes": _bytes8(n, rows) + _bytes8(k, rows) + 2 * e * n * k, "flops": 2 * rows * n * k}


# ------------------------------------------------------------------------------------------------ exact answers
def _exact_exponent(amax, top):
    """Smallest e with amax <= 1.75 * 2^top * 2^e, from the quotient's exponent in 64 bits."""
    q, ex = torch.frexp(amax.double() / (1.75 * 2.0 ** top))
    e = torch.where(q > 0.5, ex, ex - 1)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 127)


def _exact_grid(y, fmt):
    """Distance of neighbouring 8-bit values at y."""
    mant, low = (3, -6) if fmt == "e4m3" else (2, -14)
    _, ex = torch.frexp(y.abs())
    return torch.ldexp(torch.ones_like(y), (ex - 1).clamp(min=low) - mant)


def _exact_rows(x, fmt):
    rows, cols = x.shape
    out = torch.empty(rows, cols, dtype=torch.float64, device=x.device)
    words = -(-cols // 512)
    sc = torch.full((words, rows, 4), 2.0 ** -127, dtype=torch.float64, device=x.device)
    for b in range(-(-cols // 128)):
        part = x[:, 128 * b:128 * (b + 1)].double()
        e = _exact_exponent(part.abs().amax(1), 8 if fmt == "e4m3" else 15)
        s = torch.ldexp(torch.ones_like(part[:, 0]), e)
        y = part / s[:, None]
        d = _exact_grid(y, fmt)
        out[:, 128 * b:128 * (b + 1)] = torch.round(y / d) * d
        sc[b // 4, :, b % 4] = s
    return out, sc


def _exact_tiles(x, fmt, transpose):
    g, rows, cols = x.shape
    y = x.double()
    e = torch.empty(g, rows, -(-cols // 128), dtype=torch.int32, device=x.device)
    et = torch.empty(g, cols, -(-rows // 128), dtype=torch.int32, device=x.device)
    for i in range(-(-rows // 128)):
        for j in range(-(-cols // 128)):
            r, c = slice(128 * i, 128 * (i + 1)), slice(128 * j, 128 * (j + 1))
            k = _exact_exponent(y[:, r, c].abs().amax((1, 2)), 8 if fmt == "e4m3" else 15)
            e[:, r, j], et[:, c, i] = k[:, None], k[:, None]
            t = y[:, r, c] / torch.ldexp(torch.ones_like(k, dtype=torch.float64), k)[:, None, None]
            d = _exact_grid(t, fmt)
            y[:, r, c] = torch.round(t / d) * d
    if transpose:
        y, e = y.transpose(1, 2), et
    n, nb = e.shape[0] * e.shape[1], e.shape[2]
    sc = torch.full((-(-nb // 4), n, 4), 2.0 ** -127, dtype=torch.float64, device=x.device)
    for b in range(nb):
        sc[b // 4, :, b % 4] = torch.ldexp(torch.ones(n, dtype=torch.float64, device=x.device),
                                           e.reshape(n, nb)[:, b])
    return y.reshape(n, -1), sc


def _exact_values(data, scale, k):
    """An 8-bit matrix in 64 bits, block by block."""
    v = data[:, :k].double()
    for b in range(-(-k // 128)):
        v[:, 128 * b:128 * (b + 1)] *= scale[b // 4, :, b % 4].double()[:, None]
    return v


def _exact_adamw(case, seed):
    s = _prepare_adamw(case, seed)
    h, t0 = HYPER, s["step"]
    flat = {k: v.double() for k, v in s["flat"].items()}         # gaps between tensors stay as they are
    place = lambda view: slice(view.storage_offset(), view.storage_offset() + view.numel())  # noqa: E731
    for t, p in enumerate(s["params"]):
        at = place(p)
        w = (s["masters"][t] if s["masters"] else p).double()
        g = s["grads"][t].double() * s["grad_scale"]
        old = []
        for name in "mv":
            x = s[name][t]
            if s["bits"] == 8:
                pad = torch.nn.functional.pad(x[0].double(), (0, -p.numel() % 128)).view(-1, 128)
                x = (pad * x[1].double()[:, None]).reshape(-1)[: p.numel()]
                old.append(x if name == "m" else x * x)
            else:
                old.append(x.double())
        m = h["beta1"] * old[0] + (1 - h["beta1"]) * g
        v = h["beta2"] * old[1] + (1 - h["beta2"]) * g ** 2
        update = (m / (1 - h["beta1"] ** t0)) / ((v / (1 - h["beta2"] ** t0)).sqrt() + h["eps"])
        w = w - h["lr"] * h["wd"] * w - h["lr"] * update
        flat["param"][at] = w
        if s["masters"]:
            flat["master"][at] = w
        if s["bits"] == 32:
            flat["m"][at], flat["v"][at] = m, v
            continue
        u = _draws(p.numel(), s["seed"], t, DEV)
        for name, x, r in (("m", m, u & 0xFFFF), ("v", v.sqrt(), u >> 16)):
            b = torch.nn.functional.pad(x, (0, -p.numel() % 128)).view(-1, 128)
            sc = torch.ldexp(torch.ones(b.shape[0], dtype=torch.float64, device=DEV),
                             _exact_exponent(b.abs().amax(1), 8))
            y = (b / sc[:, None]).reshape(-1)[: p.numel()]
            d = _exact_grid(y, "e4m3")
            flat[name][at] = torch.sign(y) * torch.floor(y.abs() / d + r.double() / 65536.0) * d
            scale = s[name][t][1]
            flat[name + "_scale"][place(scale)] = sc
    return flat


def exact(case, seed):
    op = case["op"]
    if op == "adamw":
        return _exact_adamw(case, seed)
    s = prepare(case, seed)
    if op == "quantize":
        x = s["x"]
        if s["tiles"]:
            x = x if x.dim() == 3 else x[None]
            return [_exact_tiles(x, s["fmt"], t) for t in ((False, True) if s["both"] else (False,))]
        return [_exact_rows(y, s["fmt"]) for y in ((x, x.t()) if s["both"] else (x,))]
    a, b = _exact_values(*s["a"], s["k"]), _exact_values(*s["b"], s["k"])
    if op == "matmul":
        y = torch.einsum("mk,nk->mn", a, b)
        return y + s["acc"].double() if "acc" in s else y
    offs = s["host_offs"]
    out = s["out"].double()
    for e, (lo, hi) in enumerate(zip(offs, offs[1:])):
        if op == "experts":
            n = case["n"]
            out[lo:hi] = torch.einsum("mk,nk->mn", a[lo:hi], b[e * n:(e + 1) * n])
        else:
            out[e] = torch.einsum("nt,kt->nk", a[:, lo:hi], b[:, lo:hi])
    return out
