"""Operators of a wide dense trunk on torch tensors, over the C ABI (include/bullet_b200.h has each one's definition).

    y, total, rstd = rms_norm(x, weight, residual=r, out_dtype=torch.float8_e4m3fn)   # y: Packed8
    w8 = pack8(w, by_column=True)
    h = dense(y, w8, bias=b, act=ACT_CRELU)
    h8 = pack8(h, act=ACT_CRELU)                                                      # all that the backward keeps of h
    dx, dw, db = dense_backward(dh, y, w, y=h8, act=ACT_CRELU)
    dx, dweight = rms_norm_backward(dx, total, rstd, weight, dtotal=dtotal)
    h = dense(pack4(x), pack4(w, by_column=True), bias=b, act=ACT_CRELU)              # in 4 bits
    delta = embed(table, ids)                                                         # rows by feature or bucket
    dtable = embed_backward(ddelta, ids, len(table))
    gradients, norm = clip_gradients(gradients, 1.0, out=gradients)

Weights are [in, out], which is the networks' column-major out x in matrix.  Matrices may have any distance between rows, the
elements of a row are consecutive.  Calls enqueue on torch's current stream of their tensors' device and do not wait; new
tensors come from torch's allocator.  Arguments that do not fit raise ValueError, what the library refuses B200Error, want of
memory torch.OutOfMemoryError.  Nothing is recorded for autograd: gradients are the *_backward calls', and a tensor that requires
one is refused while torch records.  The checks and allocations are compiled (csrc/tensor_calls.cpp).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .configs import ACT_CRELU, ACT_NONE, ACT_RELU, ACT_SCRELU  # noqa: F401

_lib.load()
try:
    from . import _tensor_calls as _calls
except ImportError as e:
    raise ImportError(f"bullet_b200._tensor_calls is missing or not built for this torch: build it with `python -m bullet_b200.build` ({e})") from e
_calls.set_errors(_lib.B200Error, torch.OutOfMemoryError)


class Packed8(NamedTuple):
    """Codes of 8 bits and their scales: one per row, or with `by_column` one per column.  The scales that pack8 and rms_norm make are powers
    of two, which leaves the values exact in bf16; with others dense_backward rounds a checkpoint's values to bf16 for dw."""

    codes: torch.Tensor
    scale: torch.Tensor
    by_column: bool = False


class Packed4(NamedTuple):
    """Codes of 4 bits (e2m1) along the axis that a product sums over, `length` of them a row in whole groups of 32, and their scales, a power of
    two for each group: torch.uint8 both, laid out as include/bullet_b200.h says.  `by_column`: a row of codes is a column of the matrix."""

    codes: torch.Tensor
    scale: torch.Tensor
    length: int
    by_column: bool = False


def _of_rows(p, what: str):
    """(matrix, scales) of a matrix (None) or of codes with a scale per row."""
    if p.__class__ is not Packed8:
        return p, None
    if p.by_column:
        raise ValueError(f"{what}: a scale per row is wanted")
    return p.codes, p.scale


def rms_norm(x, weight=None, residual=None, eps: float = 1e-5, out_dtype=None):
    """(y, total, rstd): y = total * rstd * weight with total = x + residual and rstd = 1 / sqrt(mean(total^2) + eps) per row.
    `out_dtype` torch.float8_e4m3fn gives y as Packed8; default: x's type.  Without a residual total is x itself."""
    y, scale, total, rstd = _calls.rms_norm(x, weight, residual, eps, out_dtype)
    return y if scale is None else Packed8(y, scale), x if total is None else total, rstd


def rms_norm_backward(dy, total, rstd, weight=None, dtotal=None):
    """(dx, dweight): the gradients at x (and the residual), in total's type, and at the weight (None without one).  `dtotal` is
    the gradient that reaches the total by itself."""
    return _calls.rms_norm_backward(dy, total, rstd, weight, dtotal)


def pack8(x, act: int = ACT_NONE, by_column: bool = False) -> Packed8:
    """x in 8 bits with a scale per row (weights: per column).  `act` names the activation that x came out of, whose gradient
    then stays where it was."""
    codes, scale = _calls.pack8(x, act, by_column)
    return Packed8(codes, scale, by_column)


def unpack8(packed: Packed8, dtype=torch.bfloat16):
    """The values that codes stand for."""
    return _calls.unpack8(packed.codes, packed.scale, packed.by_column, dtype)


def pack4(x, by_column: bool = False) -> Packed4:
    """x in 4 bits with a scale for every 32 elements of a row (weights [in, out]: of a column).  A group with an infinity or a NaN becomes NaN."""
    codes, scale = _calls.pack4(x, by_column)
    return Packed4(codes, scale, x.shape[0 if by_column else 1], bool(by_column))


def unpack4(packed: Packed4, dtype=torch.bfloat16):
    """The values that codes stand for (exact in bf16 and fp32): a matrix as pack4 was given."""
    return _calls.unpack4(packed.codes, packed.scale, packed.length, packed.by_column, dtype)


def dense(x, w, bias=None, act: int = ACT_NONE, residual=None, out_dtype=None):
    """act(x @ w + bias) + residual.  x and w: matrices of one 16-bit type, or both Packed8, or both Packed4 (w by column).  `out_dtype`: fp32 or 16
    bits; default x's type, bf16 for codes.  The gradient of a layer on Packed4 is dense_backward's at unpack4's values.  dense_backward wants act(x @ w + bias) by
    itself: to train a layer that has both, call without the residual, and add it behind (rms_norm does, on its way)."""
    if x.__class__ is Packed4 or w.__class__ is Packed4:
        if x.__class__ is not w.__class__:
            raise ValueError("x and w: both in 4 bits or neither")
        if x.by_column or not w.by_column:
            raise ValueError("x and w: codes of x by row and of w by column are wanted")
        return _calls.dense4(x.codes, x.scale, x.length, w.codes, w.scale, w.length, bias, act, residual, out_dtype)
    x, x_scale = _of_rows(x, "x")
    w_scale = None
    if w.__class__ is Packed8:
        if not w.by_column:
            raise ValueError("w: a scale per column is wanted")
        w, w_scale, _ = w
    return _calls.dense(x, x_scale, w, w_scale, bias, act, residual, out_dtype)


def dense_backward(dy, x, w, y=None, act: int = ACT_NONE, dskip=None, dw_dtype=torch.float32, need_dx: bool = True, need_dw: bool = True,
                   need_dbias: bool = True):
    """(dx, dw, dbias) of act(x @ w + bias); None for what is not needed.  x and y (the layer's output before a residual; not
    needed with ACT_NONE) are matrices of dy's type or 8-bit checkpoints; dskip is added to dx.  The gradient at the pre-activation
    enters both products in dy's type: behind ACT_SCRELU it is rounded to 16 bits (2^-9 of itself in bf16), also where dw is fp32;
    dbias is of the values before that."""
    x, x_scale = _of_rows(x, "x")
    y, y_scale = _of_rows(y, "y")
    return _calls.dense_backward(dy, x, x_scale, w, y, y_scale, act, dskip, dw_dtype, need_dx, need_dw, need_dbias)


def embed(table, ids, scale: float = 1.0, out_dtype=None):
    """scale (finite) * the sum of table[ids[r][s]] over s, for every list r of `ids`: [rows, slots], or [rows] for one each, in int32 or int64.  Ids outside
    [0, len(table)), as -1, name no row and add nothing.  Sums are of 32 bits; `out_dtype`: default the table's type."""
    return _calls.embed(table, ids, scale, out_dtype)


def embed_backward(dy, ids, n: int, scale: float = 1.0, dtype=torch.float32):
    """The gradient of embed at its table, [n, cols]: row t is scale * the sum of dy[r] over all ids[r][s] == t, in their order, 0 where there are none."""
    return _calls.embed_backward(dy, ids, n, scale, dtype)


def gradient_norm(gradients):
    """The norm of all elements of tensors (fp32, bf16, fp16, of any shape, their elements side by side) together: a tensor of no dimension."""
    return _calls.clip_gradients(gradients, None, None)[1]


def clip_gradients(gradients, max_norm: float, out=None):
    """([tensors], norm): the gradients times max_norm / norm where their norm together is above max_norm (and finite), else as they are.  max_norm
    is taken in 64 bits; past fp32's numbers it is infinity.  `out`:
    where they go; may be `gradients`, or any of them, themselves, which are then written only if they change.  To torch all of `out` is written in place:
    a backward that has kept one of them raises."""
    if max_norm is None:
        raise TypeError("max_norm: a number is wanted")
    return _calls.clip_gradients(gradients, max_norm, out)


def gave_up(device: int) -> bool:
    """Whether a wait of dense kernels on a device gave up since this was last asked, or reported by a call: the outputs of what ran
    there are not valid then.  For programs that replay graphs, behind a synchronisation; other calls report by B200Error."""
    word = ctypes.POINTER(ctypes.c_int32)()
    _lib.check(_lib.load().b200_op_dense_gave_up(device, ctypes.byref(word)))
    if not word or not word[0]:
        return False
    word[0] = 0
    return True
