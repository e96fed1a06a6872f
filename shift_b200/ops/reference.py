"""Plain fp32 PyTorch statements of every op of the model.

These are the numerical oracle of the kernel tests and the compute path for
CPU tensors (the CPU/gloo fault-tolerance harness).  Backward passes of the
CPU path re-run these forwards under autograd (``grad_of``), so each op has a
single definition.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    rs = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * rs * w.float()).to(x.dtype)


def rope_tables(max_pos: int, head_dim: int, theta: float, device=None):
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    pos = torch.arange(max_pos, dtype=torch.float64)
    ang = torch.outer(pos, inv)
    return ang.cos().float().to(device), ang.sin().float().to(device)


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, S: int) -> torch.Tensor:
    """x: [T, H, D] with T = B*S; rotate-half convention."""
    T, H, D = x.shape
    pos = torch.arange(T, device=x.device) % S
    c = cos[pos][:, None, :]
    s = sin[pos][:, None, :]
    x1, x2 = x[..., : D // 2].float(), x[..., D // 2:].float()
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).to(x.dtype)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, B: int, S: int, scale: float) -> torch.Tensor:
    """Causal GQA attention.  q [T, Hq, D], k/v [T, Hkv, D] -> [T, Hq, D]."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    g = Hq // Hkv
    qf = q.float().view(B, S, Hq, D).transpose(1, 2)
    kf = k.float().view(B, S, Hkv, D).transpose(1, 2).repeat_interleave(g, dim=1)
    vf = v.float().view(B, S, Hkv, D).transpose(1, 2).repeat_interleave(g, dim=1)
    s = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    mask = torch.ones(S, S, dtype=torch.bool, device=q.device).triu(1)
    s = s.masked_fill(mask, float("-inf"))
    p = torch.softmax(s, dim=-1)
    o = torch.matmul(p, vf)
    return o.transpose(1, 2).reshape(T, Hq, D).to(q.dtype)


def router(x: torch.Tensor, wr: torch.Tensor, k: int, normalize: bool):
    logits = x.float() @ wr.float().t()
    probs = torch.softmax(logits, dim=-1)
    # deterministic top-k: highest prob first, ties to the lower expert index
    order = torch.argsort(-probs, dim=-1, stable=True)[:, :k]
    sel = torch.gather(probs, 1, order)
    w = sel / sel.sum(-1, keepdim=True) if normalize else sel
    return probs, order.to(torch.int32), w


def swiglu_interleaved(h: torch.Tensor) -> torch.Tensor:
    """h: [R, 2F] with blocks of 16 gate then 16 up columns."""
    R, F2 = h.shape
    hv = h.float().view(R, F2 // 32, 2, 16)
    g, u = hv[:, :, 0, :], hv[:, :, 1, :]
    return (F.silu(g) * u).reshape(R, F2 // 2).to(h.dtype)


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """[F, H] gate and up -> [2F, H] rows in blocks of 16 gate / 16 up."""
    Fd, H = gate.shape
    return torch.stack([gate.view(Fd // 16, 16, H), up.view(Fd // 16, 16, H)], dim=1).reshape(2 * Fd, H)


def moe_experts(x: torch.Tensor, idx: torch.Tensor, w: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor,
                e_lo: int = 0) -> torch.Tensor:
    """Reference MoE: x [T, H], idx/w [T, k], w1 [E, 2F, H] (interleaved), w2 [E, H, F].
    Only experts [e_lo, e_lo + E) contribute."""
    T, H = x.shape
    E = w1.shape[0]
    out = torch.zeros(T, H, dtype=torch.float32, device=x.device)
    for e in range(E):
        tok, slot = torch.nonzero(idx == (e + e_lo), as_tuple=True)
        if tok.numel() == 0:
            continue
        h = x[tok].float() @ w1[e].float().t()
        a = swiglu_interleaved(h)
        y = a.float() @ w2[e].float().t()
        out.index_add_(0, tok, y * w[tok, slot].float()[:, None])
    return out.to(x.dtype)


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    return F.cross_entropy(logits.float(), labels.long(), reduction="none", ignore_index=-100)


def adamw(master, m, v, grad, lr, beta1, beta2, eps, wd, step):
    """torch.optim.AdamW single-tensor arithmetic, fp32."""
    master = master * (1 - lr * wd)
    m = m.lerp(grad, 1 - beta1)
    v = v * beta2 + (1 - beta2) * grad * grad
    bc1 = 1 - beta1 ** step
    bc2 = 1 - beta2 ** step
    denom = (v.sqrt() / math.sqrt(bc2)) + eps
    master = master - (lr / bc1) * (m / denom)
    return master, m, v


# ------------------------------------------------------------- 8-bit floating point, a scale per block of 128
def fp8_block_scale(amax: torch.Tensor, fmt: str):
    """Scale byte (exponent + 127) and reciprocal scale of blocks with largest finite magnitude ``amax``."""
    top = 8 if fmt == "e4m3" else 15
    frac, ex = torch.frexp(amax.float())
    e = ex - 1 - top + (frac > 0.875).int()
    e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 127)
    return (e + 127).to(torch.uint8), ((127 - e) << 23).to(torch.int32).view(torch.float32)


def _finite_abs(x: torch.Tensor) -> torch.Tensor:
    a = x.abs()
    return torch.where(torch.isfinite(a), a, torch.zeros_like(a))


def _fp8_pack_scales(b: torch.Tensor) -> torch.Tensor:
    b = F.pad(b, (0, -b.shape[1] % 4))
    return b.view(b.shape[0], -1, 4).permute(1, 0, 2).contiguous()


def _fp8_codes(x: torch.Tensor, inv: torch.Tensor, fmt: str) -> torch.Tensor:
    dt = torch.float8_e4m3fn if fmt == "e4m3" else torch.float8_e5m2
    out = torch.zeros(x.shape[0], -(-x.shape[1] // 16) * 16, dtype=torch.uint8)
    out[:, :x.shape[1]] = (x * inv).to(dt).view(torch.uint8)
    return out


def fp8_quantize(x: torch.Tensor, fmt: str, tiles: bool, both: bool) -> list:
    """Codes and scales (uint8) of [rows, cols] or [G, rows, cols], and of the transposes."""
    x = (x if x.dim() == 3 else x[None]).float()
    G, R, C = x.shape
    if x.numel() == 0:
        got = [torch.zeros(G * R, -(-C // 16) * 16), torch.zeros(-(-C // 512), G * R, 4)]
        if both:
            got += [torch.zeros(G * C, -(-R // 16) * 16), torch.zeros(-(-R // 512), G * C, 4)]
        return [t.to(torch.uint8) for t in got]
    rb, cb = -(-R // 128), -(-C // 128)
    a = F.pad(_finite_abs(x), (0, cb * 128 - C, 0, rb * 128 - R)).view(G, rb, 128, cb, 128)
    full = a.amax((2, 4), keepdim=True) if tiles else None
    got = []
    for t in range(2 if both else 1):
        m = full if tiles else a.amax(2 if t else 4, keepdim=True)
        b, inv = fp8_block_scale(m, fmt)
        inv = inv.expand(G, rb, 128, cb, 128).reshape(G, rb * 128, cb * 128)[:, :R, :C]
        xt, it = (x.transpose(1, 2), inv.transpose(1, 2)) if t else (x, inv)
        n, k = (C, R) if t else (R, C)
        if t:
            b = b.permute(0, 3, 4, 1, 2)                     # [G, cb, 128 or 1, rb, 1]
        b = b.expand(G, b.shape[1], 128, b.shape[3], 1).reshape(G, -1, b.shape[3])[:, :n]
        got += [_fp8_codes(xt.reshape(G * n, k), it.reshape(G * n, k), fmt), _fp8_pack_scales(b.reshape(G * n, -1))]
    return got


def fp8_scales(scale: torch.Tensor) -> torch.Tensor:
    """Scale bytes as fp32 powers of two."""
    b = scale.view(torch.uint8).int()
    return torch.where(b > 0, b << 23, torch.full_like(b, 1 << 22)).view(torch.float32)


def fp8_values(data: torch.Tensor, scale: torch.Tensor, cols: int) -> torch.Tensor:
    """fp32 values of an 8-bit matrix (``ops.fp8.BlockFp8``)."""
    s = fp8_scales(scale).permute(1, 0, 2).reshape(data.shape[0], 4 * scale.shape[0]).repeat_interleave(128, 1)
    return data[:, :cols].float() * s[:, :cols]


def segments(offs: torch.Tensor, limit: int):
    """(lo, hi) of each segment, cut to [0, limit]; an offset below the one before counts as that one."""
    o = [min(max(x, 0), limit) for x in offs.tolist()]
    for g in range(1, len(o)):
        o[g] = max(o[g], o[g - 1])
    return list(zip(o, o[1:]))


# ------------------------------------------------------------- 8-bit moments
_M32 = 0xFFFFFFFF


def mix32(h):
    """Two multiply-and-fold rounds over 32 bits (ints or int64 tensors); the constants are those that Chris Wellons
    published ("Prospecting for hash functions", 2018)."""
    h = h & _M32
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & _M32
    h = ((h ^ (h >> 15)) * 0x846CA68B) & _M32
    return h ^ (h >> 16)


def moment_draws(n: int, seed: int, number: int, device=None) -> torch.Tensor:
    """32 random bits per element of tensor ``number``: the low half rounds exp_avg, the high half exp_avg_sq."""
    key = mix32(mix32(seed & _M32) ^ ((number * 0x9E3779B1) & _M32))
    return mix32(torch.arange(n, dtype=torch.int64, device=device) * 0x9E3779B1 + key)


def moment_decode(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return code.float() * fp8_scales(scale).repeat_interleave(128)[: code.numel()]


def moment_encode(x: torch.Tensor, bits16: torch.Tensor, root: bool = False):
    """x fp32 [n] -> (codes float8_e4m3fn [n], scales float8_e8m0fnu [ceil(n / 128)]); a magnitude goes to the
    code above with the probability of its distance from the one below.  ``root``: x are roots of second moments, of
    which those above zero get code 1 at least (an update is divided by them)."""
    n = x.numel()
    b, inv = fp8_block_scale(F.pad(_finite_abs(x), (0, -n % 128)).view(-1, 128).amax(-1), "e4m3")
    y = (x * inv.repeat_interleave(128)[:n]).abs()
    if root:
        y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
    shift = torch.where(y < 2.0 ** -6, 2.0 ** -6, 0.0)
    t = (((y + shift).view(torch.int32) + (bits16 << 4).int()) & ~0xFFFFF).view(torch.float32) - shift
    t = torch.where(torch.isfinite(x), torch.copysign(t, x), torch.full_like(t, math.nan))
    return t.to(torch.float8_e4m3fn), b.view(torch.float8_e8m0fnu)


def grad_of(fn, inputs, grad_out):
    """Gradients of fn(*inputs) w.r.t. the floating inputs, via autograd."""
    # cloned: an input may be a view of a buffer another rank's thread writes
    # into meanwhile (tensor-parallel emulation), which autograd would reject
    leaves = [t.detach().clone().requires_grad_(t.is_floating_point()) if isinstance(t, torch.Tensor) else t
              for t in inputs]
    with torch.enable_grad():
        out = fn(*leaves)
    diff = [t for t in leaves if isinstance(t, torch.Tensor) and t.requires_grad]
    grads = torch.autograd.grad(out, diff, grad_out, allow_unused=True)
    it = iter(grads)
    res = []
    for t in leaves:
        if isinstance(t, torch.Tensor) and t.requires_grad:
            g = next(it)
            res.append(torch.zeros_like(t) if g is None else g)
        else:
            res.append(None)
    return res
