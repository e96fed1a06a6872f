"""8-bit matrices with a scale per block of 128, and their products.

A value is ``code * 2^e``: the code is an 8-bit float (``"e4m3"``: 448 largest,
3 fraction bits; ``"e5m2"``: 57344 largest, 2 fraction bits) and ``2^e`` the
smallest power of two that brings the block's largest finite magnitude within
the type.  Power-of-two scales multiply exactly, so quantising rounds once and
a product needs no rescaling of partial sums: the tensor cores apply the
exponents themselves.

* ``quantize``        matrix -> ``BlockFp8``; with ``both`` also of its transpose,
  from one read (a backward pass contracts along the other side); with
  ``tiles`` one scale per 128 x 128, the same in both orientations (weights)
* ``dequantize``      the values a ``BlockFp8`` stands for
* ``matmul``          D = a @ b^T, both with the contraction inside
* ``grouped_matmul``  rows of ``a`` in segments ``offs``, segment g with b's group g
* ``grouped_wgrad``   contraction in segments ``offs``: D[g] = a[:, seg] @ b[:, seg]^T

They stand beside ``ops.gemm`` and mirror it for a linear layer y = x @ w^T::

    xq, xqt = quantize(x, both=True)              # [T, K], [K, T]
    wq, wqt = quantize(w, tiles=True, both=True)  # [N, K], [K, N]
    y = matmul(xq, wq)
    gq, gqt = quantize(dy, "e5m2", both=True)     # [T, N], [N, T]
    dx = matmul(gq, wqt)
    matmul(gqt, xqt, out=dw, accumulate=True)

Non-finite values stay non-finite: infinities and NaN are left out of a
block's maximum and stored as NaN (an infinity stays one in e5m2, which has
it), so a product shows them.  CPU tensors take the fp32 statements of
``ops.reference``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import reference as ref
from ._ext import ext, status_word

FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
BLOCK = 128


class BlockFp8(NamedTuple):
    """``data`` [rows, round_up(cols, 16)] codes, of which the first ``cols`` count; ``scale``
    [ceil(cols / 512), rows, 4] powers of two (float8_e8m0fnu): entry (w, r, j) scales
    columns [512 w + 128 j, + 128) of row r.  A batch of G matrices has their rows one
    after the other."""
    data: torch.Tensor
    scale: torch.Tensor
    cols: int

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def device(self) -> torch.device:
        return self.data.device


def _fail(cond: bool, text: str):
    if not cond:
        raise ValueError(text)


def quantize(x: torch.Tensor, fmt: str = "e4m3", tiles: bool = False, both: bool = False):
    """x [rows, cols] or [G, rows, cols], bf16 / fp16 / fp32, inner stride 1.

    Returns the ``BlockFp8`` of x (rows G * rows), or with ``both`` the pair
    of it and that of each matrix's transpose (rows G * cols)."""
    _fail(fmt in FORMATS, f"quantize: 8-bit type {fmt!r}, expected one of {sorted(FORMATS)}")
    _fail(x.dim() in (2, 3), f"quantize: a matrix or a batch of matrices, got {x.dim()} dimensions")
    _fail(x.dtype in (torch.bfloat16, torch.float16, torch.float32), f"quantize: bf16, fp16 or fp32, got {x.dtype}")
    rows, cols = x.shape[-2:]
    if x.is_cuda:
        got = ext().fp8_quantize(x, 0 if fmt == "e4m3" else 1, tiles, both)
    else:
        got = ref.fp8_quantize(x, fmt, tiles, both)
    q = BlockFp8(got[0].view(FORMATS[fmt]), got[1].view(torch.float8_e8m0fnu), cols)
    if not both:
        return q
    return q, BlockFp8(got[2].view(FORMATS[fmt]), got[3].view(torch.float8_e8m0fnu), rows)


def dequantize(q: BlockFp8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [rows, cols]; exact in fp32 and bf16 down to their smallest values."""
    _check(q, "dequantize")
    return ref.fp8_values(q.data, q.scale, q.cols).to(dtype)


def _check(q: BlockFp8, who: str):
    _fail(q.data.dim() == 2 and q.data.dtype in FORMATS.values(),
          f"{who}: codes are a matrix of float8_e4m3fn or float8_e5m2, got {q.data.dtype}")
    _fail(q.cols >= 0 and q.data.shape[1] >= q.cols, f"{who}: {q.data.shape[1]} columns of codes, {q.cols} are said")
    _fail(q.scale.dtype == torch.float8_e8m0fnu and q.scale.is_contiguous()
          and tuple(q.scale.shape) == (-(-q.cols // 512), q.data.shape[0], 4),
          f"{who}: scales [{-(-q.cols // 512)}, {q.data.shape[0]}, 4] of float8_e8m0fnu, contiguous, got "
          f"{tuple(q.scale.shape)} of {q.scale.dtype}")
    _fail(q.scale.device == q.data.device, f"{who}: codes and scales on one device")


def _check_pair(a: BlockFp8, b: BlockFp8, who: str):
    _check(a, who)
    _check(b, who)
    _fail(a.cols == b.cols, f"{who}: the operands contract {a.cols} and {b.cols} values")
    _fail(a.device == b.device, f"{who}: operands on {a.device} and {b.device}")


def _check_out(out: torch.Tensor, shape: tuple, a: BlockFp8, who: str):
    _fail(tuple(out.shape) == shape, f"{who}: out {tuple(out.shape)}, expected {shape}")
    _fail(out.dtype in (torch.bfloat16, torch.float32), f"{who}: out in bf16 or fp32, got {out.dtype}")
    _fail(out.device == a.device, f"{who}: out on {out.device}, operands on {a.device}")
    _fail(out.shape[-1] <= 1 or out.stride(-1) == 1, f"{who}: out's inner stride must be 1")


def _check_offs(offs: torch.Tensor, a: BlockFp8, who: str):
    _fail(offs.dim() == 1 and offs.numel() >= 2 and offs.dtype == torch.int32 and offs.is_contiguous(),
          f"{who}: offs are int32 [groups + 1]")
    _fail(offs.device == a.device, f"{who}: offs on {offs.device}, operands on {a.device}")


def _run(a, b, out, offs, M, N, K, G, mode, accumulate):
    ext().fp8_matmul(a.data, a.scale, b.data, b.scale, out, offs, M, N, K, G, mode, accumulate,
                     status_word(a.device))
    return out


def matmul(a: BlockFp8, b: BlockFp8, out: torch.Tensor | None = None, accumulate: bool = False,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """D [a.rows, b.rows] = a @ b^T, summed in fp32 and rounded once to
    ``out``'s type (bf16 or fp32; ``out_dtype`` where no ``out`` is given).
    ``accumulate`` adds to what ``out`` holds."""
    _check_pair(a, b, "matmul")
    M, N, K = a.rows, b.rows, a.cols
    if out is None:
        _fail(not accumulate, "matmul: accumulate needs out")
        out = torch.empty(M, N, dtype=out_dtype, device=a.device)
    _check_out(out, (M, N), a, "matmul")
    if a.data.is_cuda:
        return _run(a, b, out, None, M, N, K, 1, 0, accumulate)
    y = ref.fp8_values(a.data, a.scale, K) @ ref.fp8_values(b.data, b.scale, K).t()
    return out.copy_(out.float() + y if accumulate else y)


def grouped_matmul(a: BlockFp8, b: BlockFp8, offs: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """D[r] = a[r] @ b[g]^T for the rows r in [offs[g], offs[g + 1]).

    ``b`` holds the groups' matrices one after the other (``quantize`` of
    [G, N, K]); ``offs`` is int32 [G + 1] on the device, rising.  Rows of
    ``out`` that no segment covers are left as they were (unwritten memory
    where no ``out`` is given)."""
    _check_pair(a, b, "grouped_matmul")
    _check_offs(offs, a, "grouped_matmul")
    G = offs.numel() - 1
    _fail(b.rows % G == 0, f"grouped_matmul: {b.rows} rows of b for {G} groups")
    R, N, K = a.rows, b.rows // G, a.cols
    if out is None:
        out = torch.empty(R, N, dtype=torch.bfloat16, device=a.device)
    _check_out(out, (R, N), a, "grouped_matmul")
    if a.data.is_cuda:
        return _run(a, b, out, offs, R, N, K, G, 0, False)
    x, w = ref.fp8_values(a.data, a.scale, K), ref.fp8_values(b.data, b.scale, K).view(G, N, K)
    for g, (lo, hi) in enumerate(ref.segments(offs, R)):
        out[lo:hi] = (x[lo:hi] @ w[g].t()).to(out.dtype)
    return out


def grouped_wgrad(a: BlockFp8, b: BlockFp8, offs: torch.Tensor, out: torch.Tensor,
                  accumulate: bool = False) -> torch.Tensor:
    """out[g] (+)= a[:, seg g] @ b[:, seg g]^T with seg g = [offs[g], offs[g + 1]).

    For expert weight gradients: ``a`` of dy^T [N, rows], ``b`` of x^T
    [K, rows], ``out`` [G, N, K].  Segments start and end on a multiple of 128
    (the last may end with the matrix), so that no block of 128 is shared by
    two of them: rows that pad a segment belong to it and have to be zero
    (``ops.functional.gather_rows`` leaves them so).  Other segments are
    refused, on the GPU through the status word (``ops._ext.check_status``)
    with ``out`` left as it was.  An empty segment gives zeros (or leaves
    ``out[g]`` with ``accumulate``)."""
    _check_pair(a, b, "grouped_wgrad")
    _check_offs(offs, a, "grouped_wgrad")
    G, M, N, K = offs.numel() - 1, a.rows, b.rows, a.cols
    _check_out(out, (G, M, N), a, "grouped_wgrad")
    _fail(out.is_contiguous(), "grouped_wgrad: out must be contiguous")
    if a.data.is_cuda:
        _run(a, b, out.view(G * M, N), offs, M, N, K, G, 1, accumulate)
        return out
    x, y = ref.fp8_values(a.data, a.scale, K), ref.fp8_values(b.data, b.scale, K)
    segs = ref.segments(offs, K)
    _fail(all(hi == lo or (lo % BLOCK == 0 and (hi % BLOCK == 0 or hi == K)) for lo, hi in segs),
          f"grouped_wgrad: segments {segs} cut a block of {BLOCK}")
    for g, (lo, hi) in enumerate(segs):
        d = x[:, lo:hi] @ y[:, lo:hi].t()
        out[g] = (out[g].float() + d if accumulate else d).to(out.dtype)
    return out
