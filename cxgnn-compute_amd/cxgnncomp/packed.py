"""Rows held in 8 bits: what a layer keeps of its input for the backward pass.

128 consecutive columns of a row share a power of two; a value is that times an int8 or an e4m3
code (csrc/packed_rows.hip).  ``pack_rows`` makes them, ``PackedRows.unpack`` reads them back,
``packed_weight_grad`` multiplies them with a gradient without unpacking them (csrc/packed_wgrad.hip)
-- which is what ``linear(..., checkpoint=...)``, ``TypedLinearE2EOP`` and the layers' ``checkpoint``
use.  No counterpart upstream.
"""
import torch

from cxgnncomp_backend import _ops

FORMATS = {"int8": 0, "e4m3": 1}


def check_format(fmt):
    """``fmt`` if it is a format or None."""
    if fmt is not None and fmt not in FORMATS:
        raise ValueError("checkpoint must be None, 'int8' or 'e4m3', got %r" % (fmt, ))
    return fmt


def _format(fmt):
    if fmt not in FORMATS:
        raise ValueError("format must be 'int8' or 'e4m3', got %r" % (fmt, ))
    return FORMATS[fmt]


class PackedRows:
    """``codes`` uint8 [N, cols rounded up to 16], ``exps`` uint8 [N, cols / 128 rounded up] (exponent
    byte b: scale 2^(b - 127), 255: the group was not finite), ``cols``, ``fmt`` and the ``dtype`` the
    rows had."""

    __slots__ = ("codes", "exps", "cols", "fmt", "dtype")

    def __init__(self, codes, exps, cols, fmt="int8", dtype=torch.float32):
        _format(fmt)
        self.codes, self.exps, self.cols, self.fmt, self.dtype = codes, exps, int(cols), fmt, dtype

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.cols))

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def unpack(self, dtype=None):
        """The rows [N, cols] in ``dtype`` (the one they had): exact in float32 and bfloat16.  In float16 a magnitude
        of 65536, as which values next to the largest float16 are held, reads back as 65504: finite float16
        rows stay finite.  Larger ones (of rows that had a wider dtype) become infinities."""
        return _ops._C.unpack_rows(self.codes, self.exps, self.cols, FORMATS[self.fmt], dtype or self.dtype)

    def __repr__(self):
        return "PackedRows(%d x %d, %s, %s)" % (self.codes.shape[0], self.cols, self.fmt, self.dtype)


def pack_rows(x, fmt="int8"):
    """x [N, C] (CUDA, float32 / bfloat16 / float16, rows may be strided) in 8 bits per value and one
    byte per 128 columns.  Codes are x / 2^k rounded to the nearest, ties to even, 2^k the smallest power
    of two (2^-111 at least) with which the group's largest magnitude stays within 127 ("int8") or
    448 ("e4m3"): an int8 value is off by at most 2^(k-1), which is 1/127 of the group's largest magnitude or less
    (k > -111), an e4m3 value by at most 1/16 of itself or 2^(k-10) (a value that rounds up to 2^128 reads back
    as an infinity).  Not differentiable; packing unpacked rows gives the same codes."""
    codes, exps = _ops._C.pack_rows(x, _format(fmt))
    return PackedRows(codes, exps, x.shape[1], fmt, x.dtype)


def packed_weight_grad(packed, g, seg_ptr=None, src_idx=None, dst_idx=None, want_sums=False):
    """gW[r] = sum over the rows i of segment r of A[src_idx[i]]^T g[dst_idx[i]] -> fp32 [R, C, N], A the rows
    ``packed`` stands for, g [*, N] float32 / bfloat16 / float16.

    ``seg_ptr`` [R + 1] (int64, non-decreasing): rows seg_ptr[r] .. seg_ptr[r + 1] - 1 are segment r's; None: one
    segment of all rows.  The row maps (int64) may be missing: row i.  An entry outside its matrix
    (padding) leaves the row out.  ``want_sums``: returns (gW, gB), gB [R, N] the sums of the same rows of g (the
    bias gradient), from the same pass.  Products are exact up to fp32 accumulation, in a fixed order: results
    repeat bit for bit.  Not differentiable."""
    gw, gb = _ops._C.packed_wgrad(packed.codes, packed.exps, packed.cols, FORMATS[packed.fmt], g, seg_ptr, src_idx, dst_idx,
                                  want_sums)
    return (gw, gb) if want_sums else gw
