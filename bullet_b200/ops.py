"""Operators of a wide dense trunk on torch tensors, over the C ABI (include/bullet_b200.h has each one's definition).

    y, total, rstd = rms_norm(x, weight, residual=r, out_dtype=torch.float8_e4m3fn)   # y: Packed8
    w8 = pack8(w, by_column=True)
    h = dense(y, w8, bias=b, act=ACT_CRELU)
    h8 = pack8(h, act=ACT_CRELU)                                                      # all that the backward keeps of h
    dx, dw, db = dense_backward(dh, y, w, y=h8, act=ACT_CRELU)
    dx, dweight = rms_norm_backward(dx, total, rstd, weight, dtotal=dtotal)

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


def dense(x, w, bias=None, act: int = ACT_NONE, residual=None, out_dtype=None):
    """act(x @ w + bias) + residual.  x and w: matrices of one 16-bit type, or both Packed8 (w by column).  `out_dtype`: fp32 or 16
    bits; default x's type, bf16 for codes.  dense_backward wants act(x @ w + bias) by itself: to train a layer that has both, call
    without the residual, and add it behind (rms_norm does, on its way)."""
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


def gave_up(device: int) -> bool:
    """Whether a wait of dense kernels on a device gave up since this was last asked, or reported by a call: the outputs of what ran
    there are not valid then.  For programs that replay graphs, behind a synchronisation; other calls report by B200Error."""
    word = ctypes.POINTER(ctypes.c_int32)()
    _lib.check(_lib.load().b200_op_dense_gave_up(device, ctypes.byref(word)))
    if not word or not word[0]:
        return False
    word[0] = 0
    return True
