"""64-bit statements of the packed-sequence operators, row by row from their definitions, with bounds on what a kernel that
rounds its operands to the input type may be off."""
import math

import torch


def cut(offs, rows):
    """Offsets as they count: within the buffer, none below the one before."""
    out, top = [], 0
    for o in offs:
        top = max(top, min(max(o, 0), rows))
        out.append(top)
    return out


def attention(qkv, offs, Hq, Hkv, D, scale, do=None):
    """{"o", "lse"} and with `do` {"dqkv"}, each with its bound under "..._tol"; rows of no sequence: 0 and -inf."""
    rows, g, half = qkv.shape[0], Hq // Hkv, torch.finfo(qkv.dtype).eps / 2
    x = qkv.double().view(rows, -1, D)
    o, o_tol = torch.zeros(2, rows, Hq, D, dtype=torch.float64, device=qkv.device)
    lse = torch.full((Hq, rows), -math.inf, dtype=torch.float64, device=qkv.device)
    dx, tol = torch.zeros(2, *x.shape, dtype=torch.float64, device=qkv.device)
    bounds = cut(offs, rows)
    for a, b in zip(bounds, bounds[1:]):
        if a == b:
            continue
        late = torch.ones(b - a, b - a, dtype=torch.bool, device=qkv.device).triu(1)
        for h in range(Hq):
            kh, vh = Hq + h // g, Hq + Hkv + h // g
            q, k, v = x[a:b, h], x[a:b, kh], x[a:b, vh]
            s = (q @ k.t() * scale).masked_fill(late, -math.inf)
            lse[h, a:b] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[h, a:b, None])
            o[a:b, h] = p @ v
            # P is rounded to the inputs' type (half a step, relative), the result once more; fp32 score and exponential
            # errors are bounded by 2^-21 of the score's absolute products (D products cut off at 2^-24, and the exponent)
            soft = 2.0 ** -21 * (scale * q.abs() @ k.abs().t() + 1) * 1.4427 + 2.0 ** -20
            o_tol[a:b, h] = (p * (half + soft)) @ v.abs() + half * o[a:b, h].abs() + tiny(qkv.dtype)
            if do is None:
                continue
            gr = do[a:b].double().view(b - a, Hq, D)[:, h]
            delta = (gr * o[a:b, h]).sum(1, keepdim=True)
            ds = p * (gr @ v.t() - delta)
            dx[a:b, vh] += p.t() @ gr
            dx[a:b, h] = scale * ds @ k
            dx[a:b, kh] += scale * ds.t() @ q
            # delta is taken from the rounded o
            off = ((gr.abs() * o_tol[a:b, h]).sum(1, keepdim=True) + 2.0 ** -21 * (gr.abs() @ v.abs().t()))
            e = ds.abs() * (half + soft) + p * off + tiny(qkv.dtype)
            tol[a:b, vh] += (p * (half + soft) + tiny(qkv.dtype)).t() @ gr.abs()
            tol[a:b, h] = scale * e @ k.abs()
            tol[a:b, kh] += scale * e.t() @ q.abs()
    got = {"o": o.view(rows, -1), "o_tol": o_tol.view(rows, -1), "lse": lse}
    if do is not None:
        got.update(dqkv=dx.view(rows, -1), dqkv_tol=(tol + half * dx.abs() + tiny(qkv.dtype)).view(rows, -1))
    return got


def tiny(dtype):
    """Half of the smallest step of the type: what a value below its normal range may be off."""
    info = torch.finfo(dtype)
    return info.smallest_normal * info.eps / 2


def close(got, want, tol, what=""):
    """|got - want| <= tol everywhere; where `want` is infinite or NaN, `got` is the same."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.nan_to_num(got[~fine], nan=7.0), torch.nan_to_num(want[~fine], nan=7.0)), what
    over = (got - want).abs()[fine] - (tol[fine] if isinstance(tol, torch.Tensor) else tol)
    assert not torch.isnan(over).any() and (over.numel() == 0 or over.max() <= 0), \
        f"{what}: {int((over > 0).sum())} of {over.numel()} values off, worst by {float(over.max()):.3e} over its bound"


def rotary(x, pos, freq, heads, dim, rot, layout, size, inverse):
    y = x.double().clone()
    view = y[:, :heads * dim].unflatten(1, (heads, dim))
    old = view.clone()
    for i in range(rot // 2):
        a, b = (i, rot // 2 + i) if layout == "half" else (2 * i, 2 * i + 1)
        angle = pos.double() * freq[i] * (-1 if inverse else 1)
        z = torch.complex(old[..., a], old[..., b]) * torch.polar(torch.full_like(angle, size), angle)[:, None]
        view[..., a], view[..., b] = z.real, z.imag
    y[:, :heads * dim] = view.flatten(1)
    return y


def label_logp(logits, labels):
    z = logits.double()
    lse = torch.logsumexp(z, 1)
    live = (labels >= 0) & (labels < z.shape[1])
    at = torch.where(live, labels, torch.zeros_like(labels)).long()
    logp = z.gather(1, at[:, None])[:, 0] - lse
    return torch.where(live, logp, torch.zeros_like(logp)), lse, live, at


def logits_grad(logits, labels, d):
    """d (onehot - softmax), zeros in rows without a label."""
    _, lse, live, at = label_logp(logits, labels)
    g = -torch.exp(logits.double() - lse[:, None]) * d.double()[:, None]
    g.scatter_add_(1, at[:, None], d.double()[:, None])
    return torch.where((live & (d != 0))[:, None], g, torch.zeros_like(g))
