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
    after the other.  Products on the GPU want codes that start on 16 bytes in rows a multiple
    of 16 bytes apart (none over another), and scales that start on 4 bytes, as ``quantize`` makes them: views of a
    byte buffer that lie otherwise are refused and have to be cloned."""
    data: torch.Tensor
    scale: torch.Tensor
    cols: int

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def device(self) -> torch.device:
        return self.data.device


def quantize(x: torch.Tensor, fmt: str = "e4m3", tiles: bool = False, both: bool = False):
    """x [rows, cols] or [G, rows, cols], bf16 / fp16 / fp32, inner stride 1.

    Returns the ``BlockFp8`` of x (rows G * rows), or with ``both`` the pair
    of it and that of each matrix's transpose (rows G * cols)."""
    if fmt not in FORMATS:
        raise ValueError(f"quantize: 8-bit type {fmt!r}, expected one of {sorted(FORMATS)}")
    if x.dim() not in (2, 3):
        raise ValueError(f"quantize: a matrix or a batch of matrices, got {x.dim()} dimensions")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"quantize: bf16, fp16 or fp32, got {x.dtype}")
    rows, cols = x.shape[-2:]
    if x.is_cuda:
        got = ext().fp8_quantize(x, fmt == "e5m2", tiles, both)
    else:
        got = ref.fp8_quantize(x, fmt, tiles, both)
        got = [t.view(torch.float8_e8m0fnu if i % 2 else FORMATS[fmt]) for i, t in enumerate(got)]
    q = BlockFp8(got[0], got[1], cols)
    return (q, BlockFp8(got[2], got[3], rows)) if both else q


def dequantize(q: BlockFp8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [rows, cols], each rounded once to ``dtype`` (fp32 and bf16 hold them exactly, but for those that
    were rounded up past the type's largest value, which become infinite, or lie below its smallest)."""
    _check(q, "dequantize")
    return ref.fp8_values(q.data, q.scale, q.cols).to(dtype)


# The CUDA entry point checks its arguments itself (csrc/gemm_fp8.cu); these are for CPU tensors.
def _check(q: BlockFp8, who: str):
    if q.data.dim() != 2 or q.data.dtype not in FORMATS.values():
        raise ValueError(f"{who}: codes are a matrix of float8_e4m3fn or float8_e5m2, got {q.data.dtype}")
    if q.cols < 0 or q.data.shape[1] < q.cols:
        raise ValueError(f"{who}: {q.data.shape[1]} columns of codes, {q.cols} are said")
    if (q.scale.dtype != torch.float8_e8m0fnu or not q.scale.is_contiguous() or q.scale.device != q.data.device
            or tuple(q.scale.shape) != (-(-q.cols // 512), q.data.shape[0], 4)):
        raise ValueError(f"{who}: scales [{-(-q.cols // 512)}, {q.data.shape[0]}, 4] of float8_e8m0fnu, contiguous, "
                         f"beside the codes, got {tuple(q.scale.shape)} of {q.scale.dtype}")


def _check_pair(a: BlockFp8, b: BlockFp8, who: str):
    _check(a, who)
    _check(b, who)
    if a.cols != b.cols:
        raise ValueError(f"{who}: the operands contract {a.cols} and {b.cols} values")
    if a.device != b.device:
        raise ValueError(f"{who}: operands on {a.device} and {b.device}")


def _check_out(out: torch.Tensor, shape: tuple, a: BlockFp8, who: str):
    if tuple(out.shape) != shape or (out.shape[-1] > 1 and out.stride(-1) != 1):
        raise ValueError(f"{who}: out {tuple(out.shape)}, expected {shape} with inner stride 1")
    if out.shape[-2] > 1 and out.stride(-2) < out.shape[-1]:
        raise ValueError(f"{who}: rows of out overlap")
    if out.dtype not in (torch.bfloat16, torch.float32) or out.device != a.device:
        raise ValueError(f"{who}: out in bf16 or fp32 beside the operands, got {out.dtype} on {out.device}")


def _need_offs(offs, who: str):
    if offs is None:                       # the extension takes none for a dense product
        raise ValueError(f"{who}: offs are int32 [groups + 1] beside the operands")


def _check_offs(offs: torch.Tensor, a: BlockFp8, who: str):
    if offs.dim() != 1 or offs.numel() < 2 or offs.dtype != torch.int32 or offs.device != a.device:
        raise ValueError(f"{who}: offs are int32 [groups + 1] beside the operands")


def _run(a, b, out, offs, mode, accumulate, make_f32=False):
    return ext().fp8_matmul(a.data, a.scale, a.cols, b.data, b.scale, b.cols, out, offs, mode, accumulate, make_f32,
                            status_word(a.data.device))


def matmul(a: BlockFp8, b: BlockFp8, out: torch.Tensor | None = None, accumulate: bool = False,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """D [a.rows, b.rows] = a @ b^T, summed in fp32 and rounded once to
    ``out``'s type (bf16 or fp32; ``out_dtype`` where no ``out`` is given).
    ``accumulate`` adds to what ``out`` holds.

    On the GPU the sum is the tensor cores', which cut off where an fp32
    addition rounds: K products of mixed signs ended about 1e-10 K of the
    result's size from the exact sum (1.2e-6 at K = 16384; one by one in fp32
    2e-7), sums of one sign up to 7e-10 K of themselves too small."""
    if out is None and out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"matmul: out in bf16 or fp32, got {out_dtype}")
    if a.data.is_cuda:
        return _run(a, b, out, None, 0, accumulate, out_dtype == torch.float32)
    _check_pair(a, b, "matmul")
    if out is None:
        if accumulate:
            raise ValueError("matmul: accumulate needs out")
        out = torch.empty(a.rows, b.rows, dtype=out_dtype)
    _check_out(out, (a.rows, b.rows), a, "matmul")
    y = ref.fp8_values(a.data, a.scale, a.cols) @ ref.fp8_values(b.data, b.scale, b.cols).t()
    return out.copy_(out.float() + y if accumulate else y)


def grouped_matmul(a: BlockFp8, b: BlockFp8, offs: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """D[r] = a[r] @ b[g]^T for the rows r in [offs[g], offs[g + 1]).

    ``b`` holds the groups' matrices one after the other (``quantize`` of
    [G, N, K]); ``offs`` is int32 [G + 1] on the device, rising (cut to the
    rows; one below the one before counts as that one), of at most 512 groups
    on the GPU.  Rows of ``out`` that no segment covers are left as they were
    (unwritten memory where no ``out`` is given)."""
    _need_offs(offs, "grouped_matmul")
    if a.data.is_cuda:
        return _run(a, b, out, offs, 0, False)
    _check_pair(a, b, "grouped_matmul")
    _check_offs(offs, a, "grouped_matmul")
    G = offs.numel() - 1
    if b.rows % G:
        raise ValueError(f"grouped_matmul: {b.rows} rows of b for {G} groups")
    R, N, K = a.rows, b.rows // G, a.cols
    if out is None:
        out = torch.empty(R, N, dtype=torch.bfloat16)
    _check_out(out, (R, N), a, "grouped_matmul")
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
    _need_offs(offs, "grouped_wgrad")
    if a.data.is_cuda:
        return _run(a, b, out, offs, 1, accumulate)
    _check_pair(a, b, "grouped_wgrad")
    _check_offs(offs, a, "grouped_wgrad")
    G, K = offs.numel() - 1, a.cols
    _check_out(out, (G, a.rows, b.rows), a, "grouped_wgrad")
    if not out.is_contiguous():
        raise ValueError("grouped_wgrad: out must be contiguous")
    x, y = ref.fp8_values(a.data, a.scale, K), ref.fp8_values(b.data, b.scale, K)
    segs = ref.segments(offs, K)
    if not all(hi == lo or (lo % BLOCK == 0 and (hi % BLOCK == 0 or hi == K)) for lo, hi in segs):
        raise ValueError(f"grouped_wgrad: segments {segs} cut a block of {BLOCK}")
    for g, (lo, hi) in enumerate(segs):
        d = x[:, lo:hi] @ y[:, lo:hi].t()
        out[g] = (out[g].float() + d if accumulate else d).to(out.dtype)
    return out
