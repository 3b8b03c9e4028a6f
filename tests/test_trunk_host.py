"""CPU tests of the dense trunk's operators: what they refuse, and that the ctypes structures are the header's."""
import ctypes
import os
import re

import pytest

from bullet_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"b200_rms_norm_op": _lib.CRmsNorm, "b200_rms_norm_grad_op": _lib.CRmsNormGrad, "b200_pack8_op": _lib.CPack8,
           "b200_unpack8_op": _lib.CUnpack8, "b200_dense_op": _lib.CDense, "b200_dense_grad_op": _lib.CDenseGrad}


def header_fields(header, name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, re.S).group(1)
    fields = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        m = re.match(r"\s*(?:const\s+)?(\w+)(\*)?\s+(.*)", decl, re.S)
        if m:
            kind = ctypes.c_void_p if m.group(2) else {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}[m.group(1)]
            fields += [(n.strip().replace("in", "in_") if n.strip() == "in" else n.strip(), kind) for n in m.group(3).split(",")]
    return fields


@pytest.mark.parametrize("name", STRUCTS)
def test_structures_are_the_headers(name):
    header = open(os.path.join(ROOT, "include", "bullet_b200.h")).read()
    assert header_fields(header, name) == list(STRUCTS[name]._fields_)
    rust = open(os.path.join(ROOT, "bindings", "rust", "b200-sys", "src", "lib.rs")).read()
    body = re.search(r"pub struct %s \{(.*?)\n\}" % name, rust, re.S).group(1)
    assert [n.replace("r#in", "in_") for n in re.findall(r"pub ([\w#]+):", body)] == [n for n, _ in STRUCTS[name]._fields_]


A = 1 << 20  # an address that no call here gets as far as to use
NORM = dict(rows=4, cols=8, x_type=1, y_type=1, ldx=8, ldr=8, lds=8, ldy=8, x=A, y=A, eps=1e-5)
NORM_GRAD = dict(rows=4, cols=8, x_type=1, dy_type=1, lddy=8, lds=8, ldds=8, lddx=8, dy=A, sum=A, rstd=A, dx=A)
PACK = dict(rows=4, cols=8, x_type=1, act=0, by_column=0, ldx=8, ldq=8, x=A, q=A, scale=A)
UNPACK = dict(rows=4, cols=8, y_type=1, by_column=0, ldq=8, ldy=8, q=A, scale=A, y=A)
DENSE = dict(rows=4, in_=8, out=16, x_type=1, y_type=1, act=0, ldx=8, ldw=16, ldr=16, ldy=16, x=A, w=A, y=A)
GRAD = dict(rows=4, in_=8, out=16, dy_type=1, x_type=1, y_type=1, dw_type=0, act=1, lddy=16, ldx=8, ldy=16, ldw=16, ldskip=8, lddx=8, lddw=16,
            dy=A, x=A, y=A, w=A, dx=A, dw=A, dbias=A, workspace=A, workspace_bytes=1 << 30)
ARG, UNSUPPORTED = -1, -5
REFUSED = [
    ("b200_op_rms_norm", NORM, dict(rows=-1), ARG), ("b200_op_rms_norm", NORM, dict(cols=0), ARG), ("b200_op_rms_norm", NORM, dict(x_type=3), UNSUPPORTED),
    ("b200_op_rms_norm", NORM, dict(y_type=4), UNSUPPORTED), ("b200_op_rms_norm", NORM, dict(x=0), ARG), ("b200_op_rms_norm", NORM, dict(y=0), ARG),
    ("b200_op_rms_norm", NORM, dict(ldx=7), ARG), ("b200_op_rms_norm", NORM, dict(x=A + 1), ARG), ("b200_op_rms_norm", NORM, dict(eps=-1.0), ARG),
    ("b200_op_rms_norm", NORM, dict(eps=float("nan")), ARG), ("b200_op_rms_norm", NORM, dict(y_type=3), ARG),  # no scale
    ("b200_op_rms_norm", NORM, dict(residual=A, ldr=4), ARG), ("b200_op_rms_norm", NORM, dict(weight=A + 2), ARG), ("b200_op_rms_norm", NORM, dict(sum=A, lds=1), ARG),
    ("b200_op_rms_norm_backward", NORM_GRAD, dict(rows=-1), ARG), ("b200_op_rms_norm_backward", NORM_GRAD, dict(dy_type=3), UNSUPPORTED),
    ("b200_op_rms_norm_backward", NORM_GRAD, dict(dy=0), ARG), ("b200_op_rms_norm_backward", NORM_GRAD, dict(sum=0), ARG),
    ("b200_op_rms_norm_backward", NORM_GRAD, dict(rstd=0), ARG), ("b200_op_rms_norm_backward", NORM_GRAD, dict(lddx=2), ARG),
    ("b200_op_rms_norm_backward", NORM_GRAD, dict(dsum=A, ldds=2), ARG), ("b200_op_rms_norm_backward", NORM_GRAD, dict(dweight=A), ARG),  # no workspace
    ("b200_op_pack8", PACK, dict(act=4), ARG), ("b200_op_pack8", PACK, dict(x_type=3), UNSUPPORTED), ("b200_op_pack8", PACK, dict(scale=0), ARG),
    ("b200_op_pack8", PACK, dict(ldq=7), ARG), ("b200_op_pack8", PACK, dict(cols=0), ARG), ("b200_op_pack8", PACK, dict(q=0), ARG),
    ("b200_op_unpack8", UNPACK, dict(y_type=3), UNSUPPORTED), ("b200_op_unpack8", UNPACK, dict(q=0), ARG), ("b200_op_unpack8", UNPACK, dict(scale=0), ARG),
    ("b200_op_unpack8", UNPACK, dict(ldy=7), ARG),
    ("b200_op_dense", DENSE, dict(x_type=0), UNSUPPORTED), ("b200_op_dense", DENSE, dict(y_type=3), UNSUPPORTED), ("b200_op_dense", DENSE, dict(act=-1), ARG),
    ("b200_op_dense", DENSE, dict(in_=0), ARG), ("b200_op_dense", DENSE, dict(out=0), ARG), ("b200_op_dense", DENSE, dict(w=0), ARG),
    ("b200_op_dense", DENSE, dict(ldw=15), ARG), ("b200_op_dense", DENSE, dict(x_type=3), ARG),  # no scales
    ("b200_op_dense", DENSE, dict(residual=A, ldr=15), ARG), ("b200_op_dense", DENSE, dict(bias=A + 1), ARG), ("b200_op_dense", DENSE, dict(w=A + 1), ARG),
    ("b200_op_dense_backward", GRAD, dict(dy_type=0), UNSUPPORTED), ("b200_op_dense_backward", GRAD, dict(x_type=2), UNSUPPORTED),
    ("b200_op_dense_backward", GRAD, dict(dy_type=2, x_type=3, y_type=2), UNSUPPORTED), ("b200_op_dense_backward", GRAD, dict(dw_type=2), UNSUPPORTED),
    ("b200_op_dense_backward", GRAD, dict(act=9), ARG), ("b200_op_dense_backward", GRAD, dict(y=0), ARG), ("b200_op_dense_backward", GRAD, dict(x=0), ARG),
    ("b200_op_dense_backward", GRAD, dict(w=0), ARG), ("b200_op_dense_backward", GRAD, dict(x_type=3), ARG), ("b200_op_dense_backward", GRAD, dict(y_type=3), ARG),
    ("b200_op_dense_backward", GRAD, dict(workspace_bytes=16), ARG), ("b200_op_dense_backward", GRAD, dict(workspace=A + 8), ARG),
    ("b200_op_dense_backward", GRAD, dict(dskip=A, ldskip=4), ARG), ("b200_op_dense_backward", GRAD, dict(lddw=8), ARG),
]
KINDS = {"b200_op_rms_norm": _lib.CRmsNorm, "b200_op_rms_norm_backward": _lib.CRmsNormGrad, "b200_op_pack8": _lib.CPack8, "b200_op_unpack8": _lib.CUnpack8,
         "b200_op_dense": _lib.CDense, "b200_op_dense_backward": _lib.CDenseGrad}


@pytest.mark.parametrize("entry,good,change,code", REFUSED, ids=[f"{e[8:]}-{'-'.join(c)}-{k}" for k, (e, _, c, _) in enumerate(REFUSED)])
def test_what_does_not_fit_is_refused_before_anything_runs(entry, good, change, code):
    lib = _lib.load()
    assert getattr(lib, entry)(0, None, ctypes.byref(KINDS[entry](**{**good, **change}))) == code
    assert lib.b200_last_error().startswith(entry[5:].encode())


@pytest.mark.parametrize("entry", KINDS)
def test_null_descriptions_are_refused(entry):
    lib = _lib.load()
    assert getattr(lib, entry)(0, None, None) == ARG
    if hasattr(lib, entry + "_workspace"):
        assert getattr(lib, entry + "_workspace")(None, ctypes.byref(ctypes.c_int64())) == ARG


@pytest.mark.parametrize("entry,good", [("b200_op_rms_norm", NORM), ("b200_op_pack8", PACK), ("b200_op_unpack8", UNPACK), ("b200_op_dense", DENSE)])
def test_no_rows_need_no_memory_and_no_device(entry, good):
    empty = {k: (0 if k in ("x", "q", "y", "w", "scale", "rows") else v) for k, v in good.items()}
    assert getattr(_lib.load(), entry)(0, None, ctypes.byref(KINDS[entry](**empty))) == 0


def test_tensor_calls_name_what_is_wrong():
    torch = pytest.importorskip("torch")
    from bullet_b200 import ops

    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="x: "):
        ops.rms_norm(x)
    with pytest.raises(ValueError, match="both in 8 bits"):
        ops.dense(ops.Packed8(x, x), x)
    with pytest.raises(ValueError, match="dy: "):
        ops.dense_backward(x, x, x)


def test_tensors_whose_gradient_would_be_lost_are_refused():
    torch = pytest.importorskip("torch")
    from bullet_b200 import ops

    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(8, 8, dtype=torch.bfloat16, requires_grad=True)
    of_w = w * 2
    for call in (lambda: ops.rms_norm(w), lambda: ops.rms_norm(x, torch.ones(8, requires_grad=True)), lambda: ops.rms_norm(x, residual=of_w), lambda: ops.dense(x, w),
                 lambda: ops.dense(of_w, x), lambda: ops.pack8(w), lambda: ops.dense_backward(x, x, w), lambda: ops.rms_norm_backward(x, of_w, x),
                 lambda: ops.unpack8(ops.Packed8(x, torch.ones(4, requires_grad=True)))):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="a matrix on a CUDA device is wanted|this type is not taken here"):  # (on to the next check)
            call()
