"""The operators of post-training on packed sequences, as measured cases.

A packed buffer holds sequences of different lengths one after the other:
sequence g is rows [offs[g], offs[g + 1]).  Operators, each in a plain form of
elementary torch operations (``own = False``) and through the framework's
kernels (``own = True``):

* ``rotary``      rotary positions of the first heads of every row: halves or
  interleaved, part of the head, frequencies scaled for long contexts
* ``attention``   causal attention with grouped heads inside every sequence;
  ``attention_step`` with its backward pass
* ``logp``        log-probability of every row's label; where a caller's own loss follows, also its gradient at the logits
* ``policy``      clipped policy loss with a KL term, and its gradient at the logits
* ``preference``  loss of pairs of sequences, and its gradient at the logits

Rows that no sequence covers give zeros (log-sum-exp: minus infinity).
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the tiny model's heads, one short batch: latency
        dict(name="rotary-tiny", op="rotary", rows=512, heads=8, others=4, dim=64, rot=64, layout="half", theta=1.0e6,
             scaling="none", factor=1.0, original=512, far=0, dtype="bf16", inverse=False),
        # queries and keys of one step (8 x 2048 tokens), a context stretched 16 times: backward, part of the head
        dict(name="rotary-far-ramp", op="rotary", rows=16384, heads=20, others=4, dim=128, rot=96, layout="interleaved",
             theta=1.0e6, scaling="ramp", factor=16.0, original=4096, far=1000000, dtype="bf16", inverse=True),
        # a handful of short sequences, some of one token
        dict(name="attention-short", op="attention", rows=200, seqs=7, spread=1.5, skip=0, tail=3, q=4, kv=4, dim=64,
             dtype="bf16", mix=5),
        # one long document
        dict(name="attention-long", op="attention", rows=16384, seqs=1, spread=0.0, skip=0, tail=0, q=32, kv=8, dim=128,
             dtype="bf16", mix=1),
        # the 0.494B model's heads, a step's tokens as documents of about 700 tokens
        dict(name="attention-step-documents", op="attention_step", rows=16384, seqs=24, spread=0.9, skip=0, tail=57, q=16,
             kv=4, dim=64, dtype="bf16", mix=2),
        # every head with keys of its own, odd sizes, padding on both sides
        dict(name="attention-step-odd", op="attention_step", rows=5003, seqs=5, spread=0.7, skip=3, tail=100, q=5, kv=5,
             dim=128, dtype="f16", mix=3),
        # a reference model's log-probability of one row: latency
        dict(name="logp-one", op="logp", rows=1, vocab=32768, dtype="bf16", live=1.0, grad=False),
        # a caller's own loss of the log-probabilities over a large odd vocabulary
        dict(name="logp-odd-vocabulary", op="logp", rows=2048, vocab=100003, dtype="bf16", live=0.9, grad=True),
        # the tiny model's rollouts
        dict(name="policy-tiny", op="policy", rows=96, vocab=1024, dtype="bf16", live=0.8, kl=0.05, low=0.2, high=0.28),
        # a step's tokens over the whole vocabulary
        dict(name="policy-step", op="policy", rows=16384, vocab=32768, dtype="bf16", live=0.9, kl=0.05, low=0.2, high=0.2),
        # three pairs, fp32 logits, odd vocabulary
        dict(name="preference-odd", op="preference", rows=301, vocab=1021, pairs=3, spread=0.8, tail=5, dtype="f32",
             live=0.7, beta=0.1, mix=4),
        # sixteen pairs of answers
        dict(name="preference-step", op="preference", rows=8192, vocab=32768, pairs=16, spread=0.6, tail=0, dtype="bf16",
             live=0.7, beta=0.1, mix=6),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_PAIRS = 16384 * 16384 * 32 * 128


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention_step", "attention_step", "logp", "policy", "preference"])
    mix = rng.randrange(1 << 30)
    if op == "rotary":
        while True:
            dim = 2 * rng.randint(8, 128)
            rows, heads, others = _log_int(rng, 1, 65536), _log_int(rng, 1, 64), rng.randint(0, 16)
            if rows * (heads + others) * dim <= 1 << 26:
                break
        scaling = rng.choice(["none", "linear", "base", "ramp"])
        return dict(op=op, rows=rows, heads=heads, others=others, dim=dim, rot=rng.choice([dim, 2 * rng.randint(4, dim // 2)]),
                    layout=rng.choice(["half", "interleaved"]), theta=rng.choice([1.0e4, 5.0e5, 1.0e6]), scaling=scaling,
                    factor=1.0 if scaling == "none" else round(rng.uniform(1.5, 40.0), 2), original=_log_int(rng, 512, 32768),
                    far=rng.choice([0, _log_int(rng, 1000, 1 << 30)]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    inverse=rng.random() < 0.5)
    if op in ("attention", "attention_step"):
        while True:
            kv, group, dim = rng.randint(1, 8), rng.randint(1, 8), rng.choice([64, 128])
            case = dict(op=op, rows=_log_int(rng, 1, 32768), seqs=_log_int(rng, 1, 200), spread=round(rng.uniform(0.0, 2.0), 3),
                        skip=rng.choice([0, 0, rng.randint(1, 200)]), tail=rng.choice([0, rng.randint(1, 300)]), q=kv * group,
                        kv=kv, dim=dim, dtype=rng.choice(["bf16", "bf16", "f16"]), mix=mix)
            pairs = sum((b - a) ** 2 for a, b in zip(_offsets(case), _offsets(case)[1:])) * case["q"] * dim
            if pairs <= MOST_PAIRS // (1 if op == "attention" else 4):
                return case
    while True:
        rows, vocab, dtype = _log_int(rng, 1, 16384), _log_int(rng, 16, 200000), rng.choice(["bf16", "bf16", "f16", "f32"])
        if rows * vocab * SIZE[dtype] <= 16384 * 32768 * 2:
            break
    case = dict(op=op, rows=rows, vocab=vocab, dtype=dtype, live=round(rng.uniform(0.3, 1.0), 2))
    if op == "logp":
        case.update(grad=rng.random() < 0.6)
    if op == "policy":
        case.update(kl=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]), low=0.2, high=round(rng.uniform(0.1, 0.4), 3))
    if op == "preference":
        case.update(pairs=_log_int(rng, 1, 64), spread=round(rng.uniform(0.0, 1.5), 3), tail=rng.choice([0, rng.randint(1, 40)]),
                    beta=round(rng.uniform(0.02, 0.5), 3), mix=mix)
    return case


def _offsets(case):
    """Rows where the sequences begin, and where the last one ends; some may be empty, and rows on both sides covered
    by none."""
    n = 2 * case["pairs"] if case["op"] == "preference" else case["seqs"]
    rng = random.Random(case["mix"])
    lo = min(case.get("skip", 0), case["rows"])
    hi = max(lo, case["rows"] - case["tail"])
    w = [math.exp(rng.gauss(0.0, case["spread"])) for _ in range(n)]
    offs, run = [lo], 0.0
    for x in w:
        run += x
        offs.append(lo + int(round((hi - lo) * run / sum(w))))
    return offs


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def _logits(g, case):
    """Logits that favour the label by a few units, and the labels; some rows have none (-100)."""
    rows, vocab = case["rows"], case["vocab"]
    z = torch.randn(rows, vocab, device=DEV, generator=g).mul_(2.0)
    labels = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    z.scatter_add_(1, labels[:, None], torch.randn(rows, 1, device=DEV, generator=g) * 2 + 6)
    z = z.to(TYPES[case["dtype"]])
    logp = torch.cat([(p.gather(1, b[:, None])[:, 0].double() - p.double().exp().sum(1).log())
                      for p, b in zip(z.split(512), labels.split(512))]).float()
    live = torch.rand(rows, device=DEV, generator=g) < case["live"]
    return z, torch.where(live, labels, torch.full_like(labels, -100)).int(), logp


def prepare(case, seed):
    op, g = case["op"], _gen(seed)
    s = {"op": op, "case": case}
    if op == "rotary":
        rows, width = case["rows"], (case["heads"] + case["others"]) * case["dim"]
        s["x"] = _normal(g, rows, width, dtype=TYPES[case["dtype"]])
        # documents of some hundred rows, each at a place of its own in a long context
        pos = torch.arange(rows, device=DEV, dtype=torch.int32)
        s["pos"] = (pos - pos // 700 * 700 + case["far"] // 700 * (pos // 700 % 701)).int()
        s["out"] = s["x"].clone()
        return s
    if op in ("attention", "attention_step"):
        rows, dim = case["rows"], case["dim"]
        s["host_offs"] = _offsets(case)
        s["offs"] = torch.tensor(s["host_offs"], dtype=torch.int32, device=DEV)
        s["qkv"] = _normal(g, rows, (case["q"] + 2 * case["kv"]) * dim, dtype=TYPES[case["dtype"]])
        if op == "attention_step":
            s["do"] = _normal(g, rows, case["q"] * dim, dtype=TYPES[case["dtype"]])
        return s
    s["logits"], s["labels"], logp = _logits(g, case)
    if op == "logp" and case["grad"]:
        s["dlogp"] = _normal(g, case["rows"], std=1.0 / case["rows"])
    if op != "logp":
        s["ref"] = logp + _normal(g, case["rows"], std=0.2)
        s["scale"] = 1.0 / case["rows"] if op == "policy" else 1.0 / case["pairs"]
    if op == "policy":
        s["old"] = logp + _normal(g, case["rows"], std=0.15)
        s["adv"] = _normal(g, case["rows"])
    if op == "preference":
        s["host_offs"] = _offsets(case)
        s["offs"] = torch.tensor(s["host_offs"], dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------------------------------------ one pass, own
def _slowest(case):
    """How often a pair turns within the original context that is slowed all the way: once, or as often as the last pair does,
    at which a case's ramp ends at the latest."""
    last = case["original"] / (2 * math.pi) * case["theta"] ** (2.0 / case["rot"] - 1.0) * (1 + 1e-9)
    return last if 1.0 < last < 32.0 else 1.0


def _run_own(s):
    case, op = s["case"], s["op"]
    if op in ("logp", "policy", "preference"):
        from shift_b200.ops import objectives
        if op == "logp":
            logp, lse = objectives.token_logp_fwd(s["logits"], s["labels"])
            if "dlogp" in s:
                objectives.token_logp_bwd(s["logits"], s["labels"], lse, s["dlogp"])
            return {"logp": logp, "lse": lse, **({"dlogits": s["logits"]} if "dlogp" in s else {})}
        if op == "policy":
            loss, logp = objectives.policy_loss_fwd_bwd(s["logits"], s["labels"], s["old"], s["adv"], ref_logp=s["ref"],
                                                        clip_low=case["low"], clip_high=case["high"], kl_coef=case["kl"],
                                                        scale=s["scale"])
            return {"loss": loss, "logp": logp, "dlogits": s["logits"]}
        loss, margin = objectives.preference_loss_fwd_bwd(s["logits"], s["labels"], s["ref"], s["offs"],
                                                          beta=case["beta"], scale=s["scale"])
        return {"loss": loss, "margin": margin, "dlogits": s["logits"]}
    from shift_b200.ops import packed
    if op == "rotary":
        if "plan" not in s:
            scaling = None if case["scaling"] == "none" else packed.RotaryScaling(case["scaling"], case["factor"],
                                                                                  case["original"], slow=_slowest(case))
            s["plan"] = packed.Rotary(case["dim"], case["theta"], rot_dim=case["rot"], layout=case["layout"],
                                      scaling=scaling, device=s["x"].device)
        return packed.rotary(s["x"], s["pos"], s["plan"], case["heads"], inverse=case["inverse"], out=s["out"])
    heads = (case["q"], case["kv"], case["dim"], case["dim"] ** -0.5)
    seqs = packed.sequences(s["offs"], case["rows"])
    o, lse = packed.attention_fwd(s["qkv"], seqs, *heads)
    if op == "attention":
        return {"o": o, "lse": lse}
    return {"o": o, "lse": lse, "dqkv": packed.attention_bwd(s["qkv"], o, lse, s["do"], seqs, *heads)}


# ------------------------------------------------------------------------------------------------ one pass, plain
def _frequencies(case):
    """Angle per position of each rotated pair (64 bits), and what the rotated values are multiplied by."""
    rot, theta, factor = case["rot"], case["theta"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    if case["scaling"] == "base":
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] != "ramp":
        return f, 1.0
    place = lambda turns: rot * math.log(case["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low, high = max(math.floor(place(32.0)), 0), min(math.ceil(place(1.0)), rot // 2 - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


def _plain_rotary(s):
    case, x = s["case"], s["x"]
    f, size = _frequencies(case)
    angle = s["pos"].double()[:, None] * f
    c, n = (angle.cos() * size).float()[:, None, :], (angle.sin() * size).float()[:, None, :]
    n = -n if case["inverse"] else n
    y = x[:, :case["heads"] * case["dim"]].view(-1, case["heads"], case["dim"]).float()
    r = y[..., :case["rot"]]
    if case["layout"] == "half":
        a, b = r.chunk(2, -1)
        r = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    y = torch.cat([r, y[..., case["rot"]:]], -1)
    s["out"][:, :case["heads"] * case["dim"]] = y.flatten(1).to(x.dtype)
    return s["out"]


def _plain_attention(s):
    case, x = s["case"], s["qkv"]
    rows, q, kv, dim = x.shape[0], case["q"], case["kv"], case["dim"]
    group, scale = q // kv, dim ** -0.5
    step = "do" in s
    xq = x[:, :q * dim].view(rows, kv, group, dim)
    xk, xv = x[:, q * dim:].view(rows, 2, kv, 1, dim).unbind(1)
    o = torch.zeros(rows, kv, group, dim, device=DEV, dtype=x.dtype)
    lse = torch.full((kv, group, rows), -math.inf, device=DEV)
    grad = torch.zeros_like(x)
    gq, (gk, gv) = grad[:, :q * dim].view(rows, kv, group, dim), grad[:, q * dim:].view(rows, 2, kv, 1, dim).unbind(1)
    for lo, hi in zip(s["host_offs"], s["host_offs"][1:]):
        if lo == hi:
            continue
        hidden = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=DEV).triu(1)
        some = max(1, min(kv, (1 << 29) // (group * (hi - lo) ** 2)))       # key heads at once: scores of 2 GB
        for h in range(0, kv, some):
            heads = slice(h, h + some)
            qs, ks, vs = (t[lo:hi, heads].permute(1, 2, 0, 3).float() for t in (xq, xk, xv))
            p = (qs @ ks.transpose(-1, -2)).mul_(scale).masked_fill_(hidden, -math.inf)
            top = p.amax(-1, keepdim=True)
            p = p.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            p = p.div_(total)
            lse[heads, :, lo:hi] = (top + total.log())[..., 0]
            os = p @ vs
            o[lo:hi, heads] = os.permute(2, 0, 1, 3).to(x.dtype)
            if not step:
                continue
            do = s["do"].view(rows, kv, group, dim)[lo:hi, heads].permute(1, 2, 0, 3).float()
            gv[lo:hi, heads] = (p.transpose(-1, -2) @ do).sum(1, keepdim=True).permute(2, 0, 1, 3).to(x.dtype)
            ds = (do @ vs.transpose(-1, -2)).sub_((do * os).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            gq[lo:hi, heads] = (ds @ ks).permute(2, 0, 1, 3).to(x.dtype)
            gk[lo:hi, heads] = (ds.transpose(-1, -2) @ qs).sum(1, keepdim=True).permute(2, 0, 1, 3).to(x.dtype)
    out = {"o": o.view(rows, q * dim), "lse": lse.view(q, rows)}
    return {**out, "dqkv": grad} if step else out


def _label_logp(z, labels):
    """Softmax of every row and the label's log-probability (64 bits: the clip decides next to a border), 0 without one."""
    z = z.float()
    top = z.amax(1, keepdim=True)
    p = (z - top).exp_()
    total = p.sum(1, keepdim=True, dtype=torch.float64)
    live = labels >= 0
    at = labels.long().clamp(min=0)[:, None]
    logp = ((z.gather(1, at) - top).double() - total.log())[:, 0]
    return p.div_(total.float()), live, at, torch.where(live, logp, torch.zeros_like(logp)), (top + total.log())[:, 0].float()


def _spread(p, at, d):
    """d (onehot - softmax) over p's memory."""
    p = p.mul_(-d[:, None])
    return p.scatter_add_(1, at, d[:, None])


def _plain_loss(s):
    case, op, z = s["case"], s["op"], s["logits"]
    p, live, at, logp, lse = _label_logp(z, s["labels"])
    if op == "logp":
        got = {"logp": logp.float(), "lse": lse}
        if "dlogp" in s:
            z.copy_(_spread(p, at, torch.where(live, s["dlogp"], torch.zeros_like(s["dlogp"]))))
            got["dlogits"] = z
        return got
    if op == "policy":
        ratio = (logp - s["old"].double()).exp()
        adv, gap = s["adv"].double(), s["ref"].double() - logp
        clipped = ratio.clamp(1 - case["low"], 1 + case["high"])
        loss = -torch.minimum(ratio * adv, clipped * adv) + case["kl"] * (gap.exp() - gap - 1)
        d = -torch.where(ratio * adv <= clipped * adv, ratio * adv, torch.zeros_like(adv)) + case["kl"] * (1 - gap.exp())
        loss, d = (torch.where(live, t, torch.zeros_like(t)) for t in (loss, d))
        z.copy_(_spread(p, at, (d * s["scale"]).float()))
        return {"loss": loss.float(), "logp": logp.float(), "dlogits": z}
    gap = torch.where(live, logp - s["ref"].double(), torch.zeros_like(logp))
    run = torch.cat([gap.new_zeros(1), gap.cumsum(0)])
    offs = s["offs"].long()
    sums = (run[offs[1:]] - run[offs[:-1]]).view(-1, 2)
    margin = case["beta"] * (sums[:, 0] - sums[:, 1])
    weight = case["beta"] * s["scale"] / (1 + margin.exp())
    index = torch.arange(case["rows"], device=DEV)
    which = torch.searchsorted(offs, index, right=True) - 1
    inside = live & (which >= 0) & (which < offs.numel() - 1)
    sign = torch.where(which % 2 == 0, -1.0, 1.0)
    d = torch.where(inside, sign * weight[(which // 2).clamp(0, case["pairs"] - 1)], torch.zeros_like(gap))
    z.copy_(_spread(p, at, d.float()))
    loss = (-margin).clamp(min=0) + (-margin.abs()).exp().log1p()
    return {"loss": loss.float(), "margin": margin.float(), "dlogits": z}


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "rotary":
        return _plain_rotary(state)
    return _plain_attention(state) if "qkv" in state else _plain_loss(state)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    op, size = case["op"], SIZE[case["dtype"]]
    if op == "rotary":
        return {"bytes": case["rows"] * (2 * case["heads"] * case["dim"] * size + 4), "flops": 0}
    if op in ("attention", "attention_step"):
        offs = _offsets(case)
        seen = sum((b - a) * (b - a + 1) // 2 for a, b in zip(offs, offs[1:])) * case["q"] * case["dim"]
        rows, wide = case["rows"], (case["q"] + 2 * case["kv"]) * case["dim"]
        moved = rows * (wide * size + case["q"] * (case["dim"] * size + 4))
        if op == "attention":
            return {"bytes": moved, "flops": 4 * seen}
        return {"bytes": moved + rows * (wide + case["q"] * case["dim"]) * size, "flops": 14 * seen}
    n = case["rows"] * case["vocab"] * size
    return {"bytes": n if op == "logp" and not case["grad"] else 2 * n, "flops": 0}


# ------------------------------------------------------------------------------------------------ exact answers
def _exact_rotary(case, s):
    out = s["x"].double()
    half = case["rot"] // 2
    factor, base, scaling = case["factor"], case["theta"], case["scaling"]
    if scaling == "base":
        base *= factor ** (case["rot"] / (case["rot"] - 2))
    view = out[:, :case["heads"] * case["dim"]].view(case["rows"], case["heads"], case["dim"])
    old = view.clone()
    size = 1 + 0.1 * math.log(factor) if scaling == "ramp" else 1.0
    for i in range(half):
        f = math.exp(-math.log(base) * i / half)
        if scaling == "linear":
            f /= factor
        if scaling == "ramp":
            edge = [case["rot"] * math.log(case["original"] / (2 * math.pi * t)) / (2 * math.log(base)) for t in (32, 1)]
            low, high = max(0, math.floor(edge[0])), min(half - 1, math.ceil(edge[1]))
            share = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            f = share * f / factor + (1 - share) * f
        angle = s["pos"].double() * f * (-1 if case["inverse"] else 1)
        turn = torch.polar(torch.full_like(angle, size), angle)[:, None]
        a, b = (i, half + i) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        z = torch.complex(old[..., a], old[..., b]) * turn
        view[..., a], view[..., b] = z.real, z.imag
    return out


def _exact_attention(case, s):
    rows, dim, group = case["rows"], case["dim"], case["q"] // case["kv"]
    x = s["qkv"].double().view(rows, -1, dim)
    out = torch.zeros(rows, case["q"], dim, dtype=torch.float64, device=DEV)
    lse = torch.full((case["q"], rows), -math.inf, dtype=torch.float64, device=DEV)
    dx = torch.zeros_like(x)
    for a, b in zip(s["host_offs"], s["host_offs"][1:]):
        for h in range(case["q"]):
            kh, vh = case["q"] + h // group, case["q"] + case["kv"] + h // group
            for lo in range(a, b, 4096):                        # some queries at a time, the keys up to the last of them
                hi = min(b, lo + 4096)
                q, k, v = x[lo:hi, h], x[a:hi, kh], x[a:hi, vh]
                z = torch.einsum("qd,kd->qk", q, k) / math.sqrt(dim)
                late = torch.arange(a, hi, device=DEV)[None, :] > torch.arange(lo, hi, device=DEV)[:, None]
                z[late] = -math.inf
                lse[h, lo:hi] = z.logsumexp(1)
                w = (z - lse[h, lo:hi, None]).exp()
                out[lo:hi, h] = torch.einsum("qk,kd->qd", w, v)
                if "do" not in s:
                    continue
                g = s["do"][lo:hi, h * dim:(h + 1) * dim].double()
                dx[a:hi, vh] += torch.einsum("qk,qd->kd", w, g)
                dw = torch.einsum("qd,kd->qk", g, v)
                dz = w * (dw - (w * dw).sum(1, keepdim=True)) / math.sqrt(dim)
                dx[lo:hi, h] = torch.einsum("qk,kd->qd", dz, k)
                dx[a:hi, kh] += torch.einsum("qk,qd->kd", dz, q)
    got = {"o": out.view(rows, -1), "lse": lse}
    return {**got, "dqkv": dx.view(rows, -1)} if "do" in s else got


def _exact_loss(case, s):
    rows, offs, op = case["rows"], s.get("host_offs"), case["op"]
    labels = s["labels"].long()
    parts = [z.double().log_softmax(1) for z in s["logits"].split(1024)]
    lse = torch.cat([z.double().logsumexp(1) for z in s["logits"].split(1024)])
    logp = torch.cat([q.gather(1, b.clamp(min=0)[:, None])[:, 0] for q, b in zip(parts, labels.split(1024))])
    logp = logp * (labels >= 0)
    extra = {"logp": logp}
    if op == "logp":
        if "dlogp" not in s:
            return {"logp": logp, "lse": lse}
        d, first = s["dlogp"].double() * (labels >= 0), {"lse": lse}
    elif op == "policy":
        log_r, u = logp - s["old"].double(), s["ref"].double() - logp
        adv, up = s["adv"].double(), s["adv"] >= 0
        limit = up.double() * math.log1p(case["high"]) + (~up).double() * math.log1p(-case["low"])
        open_ = torch.where(up, log_r <= limit, log_r >= limit)
        gain = torch.where(open_, log_r.exp(), limit.exp()) * adv
        first = {"loss": (case["kl"] * (torch.expm1(u) - u) - gain) * (labels >= 0)}
        d = -case["kl"] * torch.expm1(u) - open_ * log_r.exp() * adv
        d = d * (labels >= 0) * s["scale"]
    else:
        d, loss, margin = torch.zeros_like(logp), [], []
        for k in range(case["pairs"]):
            won, lost = (slice(offs[2 * k + i], offs[2 * k + 1 + i]) for i in (0, 1))
            total = [((logp - s["ref"].double()) * (labels >= 0))[part].sum() for part in (won, lost)]
            margin.append(case["beta"] * (total[0] - total[1]))
            loss.append(-torch.nn.functional.logsigmoid(margin[-1]))
            pull = case["beta"] * s["scale"] * torch.sigmoid(-margin[-1])
            d[won], d[lost] = -pull, pull
        d, first, extra = d * (labels >= 0), {"loss": torch.stack(loss)}, {"margin": torch.stack(margin)}
    z = torch.empty(rows, case["vocab"], dtype=torch.float64, device=DEV)
    for k, q in enumerate(parts):
        at = slice(1024 * k, 1024 * k + q.shape[0])
        z[at] = -q.exp() * d[at, None]
        z[at].scatter_add_(1, labels[at].clamp(min=0)[:, None], d[at, None])
    return {**first, **extra, "dlogits": z}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "rotary":
        return _exact_rotary(case, s)
    return _exact_attention(case, s) if "qkv" in s else _exact_loss(case, s)
