"""Operators of a wide dense trunk on torch tensors, over the C ABI (include/bullet_b200.h has each one's definition).

    y, total, rstd = rms_norm(x, weight, residual=r, out_dtype=torch.float8_e4m3fn)   # y: Packed8
    w8 = pack8(w, by_column=True)
    h = dense(y, w8, bias=b, act=ACT_CRELU)
    h8 = pack8(h, act=ACT_CRELU)                                                      # all that the backward keeps of h
    dx, dw, db = dense_backward(dh, y, w, y=h8, act=ACT_CRELU)
    dx, dweight = rms_norm_backward(dx, total, rstd, weight, dtotal=dtotal)

Weights are [in, out], which is the networks' column-major out x in matrix.  Matrices may have any distance between rows, the
elements of a row are consecutive.  Calls enqueue on torch's current stream of their tensors' device and do not wait; new
tensors come from torch's allocator.  Arguments that do not fit raise ValueError, what the library refuses B200Error.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .configs import ACT_CRELU, ACT_NONE, ACT_RELU, ACT_SCRELU  # noqa: F401

TYPE_F32, TYPE_BF16, TYPE_F16, TYPE_E4M3 = 0, 1, 2, 3
_TYPES = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16, torch.float8_e4m3fn: TYPE_E4M3}
_ref = ctypes.byref


class Packed8(NamedTuple):
    """Codes of 8 bits and their scales, powers of two: one per row, or with `by_column` one per column."""

    codes: torch.Tensor
    scale: torch.Tensor
    by_column: bool = False


def _matrix(t: torch.Tensor, what: str, device=None, shape=None, types=_TYPES) -> int:
    """Checks a matrix and returns the distance of its rows."""
    if t.dtype in types and t.is_cuda and t.dim() == 2 and t.is_contiguous() and (device is None or t.device == device) and (shape is None or t.shape == shape):
        return t.shape[1]
    if t.dim() != 2 or not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{what}: a matrix on {device or 'a CUDA device'} is wanted, not {tuple(t.shape)} on {t.device}")
    if t.dtype not in types:
        raise ValueError(f"{what}: type {t.dtype} is not taken here")
    rows, cols = t.shape
    if shape is not None and (rows, cols) != shape:
        raise ValueError(f"{what}: shape {(rows, cols)} where {shape} is wanted")
    ld = t.stride(0)
    if (t.stride(1) != 1 and cols > 1) or (ld < cols and rows > 1):
        raise ValueError(f"{what}: the elements of a row must be consecutive and rows must not overlap")
    return ld if rows > 1 else max(ld, cols)


def _vector(t: torch.Tensor | None, what: str, device, n: int):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: {n} consecutive fp32 values on {device} are wanted")
    return t.data_ptr()


def _codes(p: Packed8, what: str, device=None, shape=None, by_column=False):
    """(distance of rows, address of the scales)"""
    ld = _matrix(p.codes, what, device, shape, (torch.float8_e4m3fn,))
    if bool(p.by_column) != by_column:
        raise ValueError(f"{what}: a scale per {'column' if by_column else 'row'} is wanted")
    return ld, _vector(p.scale, f"{what}'s scales", p.codes.device, p.codes.shape[1 if by_column else 0])


_16_BITS = (torch.bfloat16, torch.float16)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _like(t: torch.Tensor, dtype):
    """An empty matrix without gaps, of t's shape (empty_like is the quicker way to one, where t has none)."""
    if t.is_contiguous():
        return torch.empty_like(t, dtype=dtype)
    return torch.empty(t.shape, dtype=dtype, device=t.device)


def _act(act: int) -> int:
    if act not in (ACT_NONE, ACT_CRELU, ACT_SCRELU, ACT_RELU):
        raise ValueError(f"act: {act} names no activation")
    return act


try:  # (the public way makes a stream object: 2.2 us instead of 0.1)
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


def _call(entry, device, op) -> None:
    rc = entry(device.index, _raw_stream(device.index), _ref(op))
    if rc < 0:
        _lib.check(rc)


def _space(query, op, device):
    """The call's workspace, set in `op`; held by the caller until the call is enqueued."""
    n = ctypes.c_int64()
    _lib.check(query(_ref(op), _ref(n)))
    if not n.value:
        return None
    space = torch.empty(n.value, dtype=torch.uint8, device=device)
    op.workspace, op.workspace_bytes = space.data_ptr(), n.value
    return space


def rms_norm(x, weight=None, residual=None, eps: float = 1e-5, out_dtype=None):
    """(y, total, rstd): y = total * rstd * weight with total = x + residual and rstd = 1 / sqrt(mean(total^2) + eps) per row.
    `out_dtype` torch.float8_e4m3fn gives y as Packed8; default: x's type.  Without a residual total is x itself."""
    ldx = _matrix(x, "x", types=_FLOATS)
    rows, cols = x.shape
    device = x.device
    out_dtype = out_dtype or x.dtype
    if out_dtype not in _TYPES:
        raise ValueError(f"out_dtype: {out_dtype} is not taken here")
    w = _vector(weight, "weight", device, cols)
    total, ldr, r, s = x, 0, None, None
    if residual is not None:
        ldr, r = _matrix(residual, "residual", device, (rows, cols), (x.dtype,)), residual.data_ptr()
        total = _like(x, x.dtype)
        s = total.data_ptr()
    y = _like(x, out_dtype)
    rstd = torch.empty(rows, dtype=torch.float32, device=device)
    packed = out_dtype is torch.float8_e4m3fn
    scale = torch.empty(rows, dtype=torch.float32, device=device) if packed else None
    op = _lib.CRmsNorm(rows, cols, _TYPES[x.dtype], _TYPES[out_dtype], ldx, ldr, cols, cols, x.data_ptr(), r, w, s, y.data_ptr(),
                       scale.data_ptr() if packed else None, rstd.data_ptr(), eps)
    _call(_lib.load().b200_op_rms_norm, device, op)
    return (Packed8(y, scale) if packed else y), total, rstd


def rms_norm_backward(dy, total, rstd, weight=None, dtotal=None):
    """(dx, dweight): the gradients at x (and the residual), in total's type, and at the weight (None without one).  `dtotal` is
    the gradient that reaches the total by itself."""
    lds = _matrix(total, "total", types=_FLOATS)
    rows, cols = total.shape
    device = total.device
    lddy = _matrix(dy, "dy", device, (rows, cols), _FLOATS)
    ldds, ds = 0, None
    if dtotal is not None:
        ldds, ds = _matrix(dtotal, "dtotal", device, (rows, cols), (total.dtype,)), dtotal.data_ptr()
    dx = _like(total, total.dtype)
    dweight = torch.empty(cols, dtype=torch.float32, device=device) if weight is not None else None
    op = _lib.CRmsNormGrad(rows, cols, _TYPES[total.dtype], _TYPES[dy.dtype], lddy, lds, ldds, cols, dy.data_ptr(), total.data_ptr(),
                           _vector(rstd, "rstd", device, rows), _vector(weight, "weight", device, cols), ds, dx.data_ptr(),
                           dweight.data_ptr() if dweight is not None else None)
    lib = _lib.load()
    space = _space(lib.b200_op_rms_norm_backward_workspace, op, device)  # noqa: F841
    _call(lib.b200_op_rms_norm_backward, device, op)
    return dx, dweight


def pack8(x, act: int = ACT_NONE, by_column: bool = False) -> Packed8:
    """x in 8 bits with a scale per row (weights: per column).  `act` names the activation that x came out of, whose gradient
    then stays where it was."""
    ldx = _matrix(x, "x", types=_FLOATS)
    rows, cols = x.shape
    codes = _like(x, torch.float8_e4m3fn)
    scale = torch.empty(cols if by_column else rows, dtype=torch.float32, device=x.device)
    op = _lib.CPack8(rows, cols, _TYPES[x.dtype], _act(act), int(by_column), ldx, cols, x.data_ptr(), codes.data_ptr(), scale.data_ptr())
    _call(_lib.load().b200_op_pack8, x.device, op)
    return Packed8(codes, scale, by_column)


def unpack8(packed: Packed8, dtype=torch.bfloat16):
    """The values that codes stand for."""
    ldq, scale = _codes(packed, "packed", by_column=bool(packed.by_column))
    if dtype not in _FLOATS:
        raise ValueError(f"dtype: {dtype} is not taken here")
    rows, cols = packed.codes.shape
    y = _like(packed.codes, dtype)
    op = _lib.CUnpack8(rows, cols, _TYPES[dtype], int(packed.by_column), ldq, cols, packed.codes.data_ptr(), scale, y.data_ptr())
    _call(_lib.load().b200_op_unpack8, y.device, op)
    return y


def dense(x, w, bias=None, act: int = ACT_NONE, residual=None, out_dtype=None):
    """act(x @ w + bias) + residual.  x and w: matrices of one 16-bit type, or both Packed8 (w by column).  `out_dtype`: fp32 or 16
    bits; default x's type, bf16 for codes."""
    x_scale = w_scale = None
    if isinstance(x, Packed8) != isinstance(w, Packed8):
        raise ValueError("x and w: both in 8 bits or neither")
    if isinstance(x, Packed8):
        ldx, x_scale = _codes(x, "x")
        x = x.codes
        ldw, w_scale = _codes(w, "w", x.device, by_column=True)
        w = w.codes
        out_dtype = out_dtype or torch.bfloat16
    else:
        ldx = _matrix(x, "x", types=_16_BITS)
        ldw = _matrix(w, "w", x.device, types=(x.dtype,))
        out_dtype = out_dtype or x.dtype
    rows, n_in = x.shape
    if w.shape[0] != n_in:
        raise ValueError(f"w: {w.shape[0]} inputs where x has {n_in}")
    if out_dtype not in _FLOATS:
        raise ValueError(f"out_dtype: {out_dtype} is not taken here")
    n_out, device = w.shape[1], x.device
    ldr, r = 0, None
    if residual is not None:
        ldr, r = _matrix(residual, "residual", device, (rows, n_out), (out_dtype,)), residual.data_ptr()
    y = torch.empty((rows, n_out), dtype=out_dtype, device=device)
    op = _lib.CDense(rows, n_in, n_out, _TYPES[x.dtype], _TYPES[out_dtype], _act(act), ldx, ldw, ldr, n_out, x.data_ptr(), x_scale, w.data_ptr(), w_scale,
                     _vector(bias, "bias", device, n_out), r, y.data_ptr())
    lib = _lib.load()
    space = _space(lib.b200_op_dense_workspace, op, device)  # noqa: F841
    _call(lib.b200_op_dense, device, op)
    return y


def dense_backward(dy, x, w, y=None, act: int = ACT_NONE, dskip=None, dw_dtype=torch.float32, need_dx: bool = True, need_dw: bool = True,
                   need_dbias: bool = True):
    """(dx, dw, dbias) of act(x @ w + bias); None for what is not needed.  x and y (the layer's output before a residual; not
    needed with ACT_NONE) are matrices of dy's type or 8-bit checkpoints; dskip is added to dx."""
    lddy = _matrix(dy, "dy", types=_16_BITS)
    rows, n_out = dy.shape
    device, kind = dy.device, dy.dtype
    n_in = (w if need_dx else x.codes if isinstance(x, Packed8) else x).shape[0 if need_dx else 1]

    def checkpoint(t, what, width):
        if isinstance(t, Packed8):
            return (*_codes(t, what, device, (rows, width)), t.codes.data_ptr(), TYPE_E4M3)
        return _matrix(t, what, device, (rows, width), (kind,)), None, t.data_ptr(), _TYPES[kind]

    ldx, x_scale, x_at, x_type = checkpoint(x, "x", n_in) if need_dw else (0, None, None, _TYPES[kind])
    if _act(act) != ACT_NONE and y is None:
        raise ValueError("y: the gradient of an activation needs its output")
    ldy, y_scale, y_at, y_type = checkpoint(y, "y", n_out) if act != ACT_NONE else (0, None, None, _TYPES[kind])
    ldw, w_at, ldskip, skip_at, dx, dw, dbias = 0, None, 0, None, None, None, None
    if need_dx:
        ldw, w_at = _matrix(w, "w", device, (n_in, n_out), (kind,)), w.data_ptr()
        dx = torch.empty((rows, n_in), dtype=kind, device=device)
        if dskip is not None:
            ldskip, skip_at = _matrix(dskip, "dskip", device, (rows, n_in), (kind,)), dskip.data_ptr()
    if need_dw:
        if dw_dtype not in (torch.float32, kind):
            raise ValueError(f"dw_dtype: {dw_dtype} is not taken here")
        dw = torch.empty((n_in, n_out), dtype=dw_dtype, device=device)
    if need_dbias:
        dbias = torch.empty(n_out, dtype=torch.float32, device=device)
    op = _lib.CDenseGrad(rows, n_in, n_out, _TYPES[kind], x_type, y_type, _TYPES[dw_dtype], act, lddy, ldx, ldy, ldw, ldskip, n_in, n_out,
                         dy.data_ptr(), x_at, x_scale, y_at, y_scale, w_at, skip_at, dx.data_ptr() if need_dx else None,
                         dw.data_ptr() if need_dw else None, dbias.data_ptr() if need_dbias else None)
    lib = _lib.load()
    space = _space(lib.b200_op_dense_backward_workspace, op, device)  # noqa: F841
    _call(lib.b200_op_dense_backward, device, op)
    return dx, dw, dbias
