"""Packed sequences: sequences of different lengths one after the other in one buffer.

Sequence g is rows [offs[g], offs[g + 1]) (int32, on the device, rising; cut to
the buffer, and one below the one before counts as that one).  Rows that none
covers take part in nothing.

* ``sequences``      what the offsets say of every row; made once a batch
* ``rotary``         rotary positions: given per row, halves or interleaved,
  part of the head, frequencies scaled for long contexts; ``inverse`` is the
  backward pass
* ``attention_fwd`` / ``attention_bwd``  causal attention with grouped heads
  inside every sequence

They stand beside ``ops.functional.rope_`` and ``attention_fwd``, which want
sequences of one length and read positions from that::

    seqs = sequences(offs, qkv.shape[0])
    rotary(qkv, seqs.pos, plan, Hq + Hkv)                      # in place
    o, lse = attention_fwd(qkv, seqs, Hq, Hkv, D, D ** -0.5)
    dqkv = attention_bwd(qkv, o, lse, do, seqs, Hq, Hkv, D, D ** -0.5)
    rotary(dqkv, seqs.pos, plan, Hq + Hkv, inverse=True)

CPU tensors take the fp32 statements of ``ops.reference``.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import reference as ref
from ._ext import ext, status_word

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


class Sequences(NamedTuple):
    """What the offsets say of every row of a buffer, in one int32 tensor: ``start``, the first row of its sequence, ``pos``,
    its place in it, and ``stop``, the row behind its end.  A row that no sequence covers has ``start`` row + 1, ``pos`` -1
    and ``stop`` row.  ``ends``: the first covered row and the one behind the last.  (On the GPU orders follow in which the
    attention kernels take their tiles.)"""
    offs: torch.Tensor
    plan: torch.Tensor
    rows: int

    @property
    def start(self) -> torch.Tensor:
        return self.plan[:self.rows]

    @property
    def pos(self) -> torch.Tensor:
        return self.plan[self.rows:2 * self.rows]

    @property
    def stop(self) -> torch.Tensor:
        return self.plan[2 * self.rows:3 * self.rows]

    @property
    def ends(self) -> torch.Tensor:
        return self.plan[3 * self.rows:3 * self.rows + 2]


def sequences(offs: torch.Tensor, rows: int) -> Sequences:
    """The plan of a buffer of ``rows`` rows.  It reads ``offs`` on the device, now: it can be captured into a graph, and
    is made again for other offsets."""
    if offs.is_cuda:
        return Sequences(offs, ext().packed_sequences(offs, rows), rows)
    if offs.dtype != torch.int32 or offs.dim() != 1 or offs.numel() < 2 or not offs.is_contiguous():
        raise ValueError(f"sequences: offs are int32 [sequences + 1], contiguous, got {tuple(offs.shape)} of {offs.dtype}")
    if not 0 <= rows <= 1 << 29:
        raise ValueError(f"sequences: 0 to 2^29 rows, got {rows}")
    return Sequences(offs, torch.cat(ref.packed_rows(offs, rows)), rows)


# ----------------------------------------------------------------------------- rotary positions
class RotaryScaling(NamedTuple):
    """How frequencies change for contexts ``factor`` times as long.

    ``"linear"``: all divided by factor.  ``"base"``: theta becomes theta * factor^(rot / (rot - 2)), so that the
    slowest pair is stretched by factor and the fastest stays.  ``"ramp"``: pairs that turn more than ``fast`` times
    within ``original`` positions stay, those that turn less than ``slow`` times are divided by factor, a ramp over the
    pairs between; rotated values are multiplied by ``magnitude`` (``None``: 0.1 ln(factor) + 1, at least 1)."""
    kind: str
    factor: float
    original: int = 0
    fast: float = 32.0
    slow: float = 1.0
    magnitude: float | None = None


class Rotary:
    """Frequencies of a head of ``head_dim`` columns, of which the first ``rot_dim`` are rotated (default: all).

    ``layout``: pair i is columns (i, rot_dim / 2 + i) (``"half"``) or (2 i, 2 i + 1) (``"interleaved"``).  Angles are
    pos * theta^(-2 i / rot_dim), for any int32 position, kept as 64-bit fractions of a turn."""

    def __init__(self, head_dim: int, theta: float = 1.0e4, rot_dim: int | None = None, layout: str = "half",
                 scaling: RotaryScaling | None = None, device="cuda"):
        rot = head_dim if rot_dim is None else rot_dim
        if not 2 <= rot <= head_dim or rot % 2:
            raise ValueError(f"Rotary: {rot} of {head_dim} columns; an even number, from 2 to the head's")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"Rotary: layout {layout!r}, expected 'half' or 'interleaved'")
        if not (math.isfinite(theta) and theta > 0):
            raise ValueError(f"Rotary: theta {theta}")
        if scaling is not None and not isinstance(scaling, RotaryScaling):
            scaling = RotaryScaling(*scaling)              # as a configuration file gives it
        self.head_dim, self.rot_dim, self.layout, self.theta, self.scaling = head_dim, rot, layout, theta, scaling
        freq, self.magnitude = self._frequencies()
        self.freq = torch.tensor(freq, dtype=torch.float64)
        turns = [int(f / (2 * math.pi) * 2.0 ** 64) & (2 ** 64 - 1) for f in freq]
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=device)

    def _frequencies(self):
        s, rot, theta = self.scaling, self.rot_dim, self.theta
        plain = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
        if s is None:
            return plain, 1.0
        if not (math.isfinite(s.factor) and s.factor > 0):
            raise ValueError(f"Rotary: scaled by {s.factor}")
        if s.kind == "linear":
            return [f / s.factor for f in plain], 1.0 if s.magnitude is None else s.magnitude
        if s.kind == "base":
            if rot < 4:
                raise ValueError("Rotary: a scaled base needs two pairs or more")
            theta *= s.factor ** (rot / (rot - 2))
            return [theta ** (-2.0 * i / rot) for i in range(rot // 2)], 1.0 if s.magnitude is None else s.magnitude
        if s.kind != "ramp":
            raise ValueError(f"Rotary: scaling {s.kind!r}, expected 'linear', 'base' or 'ramp'")
        if s.original < 1 or not s.fast > s.slow > 0 or theta <= 1:
            raise ValueError(f"Rotary: a ramp needs the original context, fast > slow > 0 and theta > 1, got {s}, {theta}")
        place = [rot * math.log(s.original / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (s.fast, s.slow)]
        # The ramp's end may lie behind the last pair, which then keeps a part of its speed; it is held to the columns, the
        # guard that scaled models are trained with.
        low, high = max(math.floor(place[0]), 0), min(math.ceil(place[1]), rot - 1)
        ramp = [1.0 if i >= place[1] else min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        size = 0.1 * math.log(max(s.factor, 1.0)) + 1.0 if s.magnitude is None else s.magnitude
        return [f * (1 - r) + f / s.factor * r for f, r in zip(plain, ramp)], size


def _share_memory(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether two matrices (inner stride 1, rows that do not overlap) share a byte, as csrc/apart.h says it."""
    if x.numel() == 0 or y.numel() == 0:
        return False
    (a, a_end, a_row, a_step), (b, b_end, b_row, b_step) = (
        (t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * step + t.shape[1]) * t.element_size(),
         t.shape[1] * t.element_size(), step * t.element_size())
        for t in (x, y) for step in [t.stride(0) if t.shape[0] > 1 else t.shape[1]])
    if a_end <= b or b_end <= a:
        return False
    if a_step != b_step:
        return True
    shift = (b - a) % a_step                               # columns of one buffer, side by side?
    return not (shift >= a_row and shift + b_row <= a_step)


def _check_apart(out, who, **others):
    for name, t in others.items():
        if _share_memory(out, t):
            raise ValueError(f"{who}: out overlaps {name}")


def rotary(x: torch.Tensor, pos: torch.Tensor, plan: Rotary, heads: int, inverse: bool = False,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotates the first ``heads`` heads of every row of x [T, >= heads * head_dim] (bf16, fp16 or fp32, any row stride)
    to its position (int32 [T]), in place, or into ``out``, whose columns behind those heads are left as they were.

    ``inverse`` turns back, with the same magnitude: applied to a gradient it is the backward pass.  A row that no
    sequence covers (position -1) is rotated like any other."""
    out = x if out is None else out
    if x.is_cuda:
        ext().rotary(x, out, pos, plan.turns, heads, plan.head_dim, plan.rot_dim, plan.layout == "interleaved",
                     plan.magnitude, inverse)
        return out
    n = heads * plan.head_dim
    if x.dim() != 2 or out.dim() != 2 or out.shape[0] != x.shape[0] or heads < 0 or min(x.shape[1], out.shape[1]) < n:
        raise ValueError(f"rotary: {heads} heads of {plan.head_dim} columns do not fit x {tuple(x.shape)} or out "
                         f"{tuple(out.shape)}")
    if x.dtype not in _FLOATS or out.dtype != x.dtype:
        raise ValueError(f"rotary: bf16, fp16 or fp32, x and out alike, got {x.dtype} and {out.dtype}")
    if pos.dtype != torch.int32 or tuple(pos.shape) != (x.shape[0],):
        raise ValueError(f"rotary: positions are int32, one for each of the {x.shape[0]} rows")
    for t in (x, out):
        if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
            raise ValueError("rotary: rows of stride 1 inside that do not overlap")
    same = x.data_ptr() == out.data_ptr() and (x.shape[0] <= 1 or x.stride(0) == out.stride(0))
    if not same:
        _check_apart(out, "rotary", x=x)
    y = ref.rotary(x[:, :n].reshape(-1, heads, plan.head_dim), pos, plan.freq, plan.rot_dim, plan.layout, plan.magnitude,
                   inverse)
    out[:, :n] = y.reshape(-1, n)
    return out


# ----------------------------------------------------------------------------- attention
# The CUDA entry points check their arguments themselves (csrc/attention_packed_host.cpp); this is for CPU tensors.
def _check(x, width, seqs, Hq, Hkv, D, scale, who):
    if Hq < 1 or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"{who}: {Hq} query heads for {Hkv} key heads")
    if D not in (64, 128):
        raise ValueError(f"{who}: heads of 64 or 128 columns, got {D}")
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError(f"{who}: scale {scale}, a number above 0 is expected")
    if x.dtype not in _FLOATS:
        raise ValueError(f"{who}: bf16, fp16 or fp32, got {x.dtype}")
    _check_rows(x, x, seqs.rows, width, who, "qkv")


def _check_rows(t, qkv, rows, cols, who, what):
    if t.dim() != 2 or tuple(t.shape) != (rows, cols) or t.dtype != qkv.dtype or t.device != qkv.device:
        raise ValueError(f"{who}: {what} [{rows}, {cols}] of {qkv.dtype} beside qkv, got {tuple(t.shape)} of {t.dtype}")


def attention_fwd(qkv: torch.Tensor, seqs: Sequences, Hq: int, Hkv: int, D: int, scale: float,
                  out: torch.Tensor | None = None):
    """Causal attention inside every sequence: qkv [T, (Hq + 2 Hkv) * D] -> (o [T, Hq * D], lse [Hq, T] fp32).

    Query head h takes key head h / (Hq / Hkv); D is 64 or 128, qkv bf16 or fp16 (on the CPU also fp32) with rows a
    multiple of 16 bytes apart.  ``lse`` is the natural logarithm of the sum of exp(scale q k).  Rows that no sequence
    covers get zeros (with ``out``: are left as they were) and an lse of minus infinity; what they hold is not looked
    at.  A row's result hangs on the rows it sees and on no other, also where others are not finite (such rows are
    computed one by one, slowly).  A score of NaN or plus infinity makes its row NaN, on the GPU its lse too."""
    if qkv.is_cuda:
        return tuple(ext().packed_attn_fwd(qkv, seqs.plan, seqs.rows, Hq, Hkv, D, scale, out, status_word(qkv.device)))
    _check(qkv, (Hq + 2 * Hkv) * D, seqs, Hq, Hkv, D, scale, "attention_fwd")
    if out is not None:
        _check_rows(out, qkv, seqs.rows, Hq * D, "attention_fwd", "out")
        _check_apart(out, "attention_fwd", qkv=qkv)
    o, lse = ref.packed_attention(qkv, ref.segments(seqs.offs, seqs.rows), Hq, Hkv, D, scale)
    if out is not None:
        live = seqs.pos >= 0
        out[live] = o[live].to(out.dtype)
        return out, lse
    return o.to(qkv.dtype), lse


def attention_bwd(qkv: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, do: torch.Tensor, seqs: Sequences, Hq: int,
                  Hkv: int, D: int, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """dqkv of ``attention_fwd``, from its results and do [T, Hq * D] (rows a multiple of 16 bytes apart).

    Deterministic: no sum's order hangs on timing.  Rows that no sequence covers get zeros (with ``out``: are left as
    they were).  fp16 scales what it rounds by powers of two, each row by the gradients that are in its own sums; the
    scaled values stay below fp16's largest where the magnitudes of a row of v add up to less than 16000."""
    if qkv.is_cuda:
        return ext().packed_attn_bwd(qkv, o, lse, do, seqs.plan, seqs.rows, Hq, Hkv, D, scale, out,
                                     status_word(qkv.device))
    who = "attention_bwd"
    _check(qkv, (Hq + 2 * Hkv) * D, seqs, Hq, Hkv, D, scale, who)
    _check_rows(o, qkv, seqs.rows, Hq * D, who, "o")
    _check_rows(do, qkv, seqs.rows, Hq * D, who, "do")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (Hq, seqs.rows) or lse.device != qkv.device:
        raise ValueError(f"{who}: lse [{Hq}, {seqs.rows}] fp32 beside qkv, got {tuple(lse.shape)} of {lse.dtype}")
    if out is not None:
        _check_rows(out, qkv, seqs.rows, qkv.shape[1], who, "out")
        _check_apart(out, who, qkv=qkv, o=o, do=do)
    segs = ref.segments(seqs.offs, seqs.rows)
    if all(lo == hi for lo, hi in segs):
        return torch.zeros_like(qkv) if out is None else out
    (g,) = ref.grad_of(lambda x: ref.packed_attention(x, segs, Hq, Hkv, D, scale)[0], [qkv], do.float())
    if out is not None:
        live = seqs.pos >= 0
        out[live] = g[live].to(out.dtype)
        return out
    return g.to(qkv.dtype)
