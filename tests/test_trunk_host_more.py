"""CPU tests of the operators in 4 bits, of embedded rows and of the norm of gradients: what they refuse, and that the ctypes structures are the
header's."""
import ctypes
import os
import re

import pytest

from bullet_b200 import _lib
from tests.test_trunk_host import A, ARG, UNSUPPORTED, header_fields

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"b200_pack4_op": _lib.CPack4, "b200_unpack4_op": _lib.CUnpack4, "b200_dense4_op": _lib.CDense4}
KINDS = {"b200_op_pack4": _lib.CPack4, "b200_op_unpack4": _lib.CUnpack4, "b200_op_dense4": _lib.CDense4}
PACK = dict(rows=4, cols=40, x_type=1, by_column=0, ldx=40, ldq=32, x=A, q=A, scale=A)
UNPACK = dict(rows=4, cols=40, y_type=1, by_column=0, ldq=32, ldy=40, q=A, scale=A, y=A)
DENSE = dict(rows=4, in_=40, out=16, y_type=1, act=0, ldx=32, ldw=32, ldr=16, ldy=16, x=A, x_scale=A, w=A, w_scale=A, y=A)
REFUSED = [
    ("b200_op_pack4", PACK, dict(rows=-1), ARG), ("b200_op_pack4", PACK, dict(cols=0), ARG), ("b200_op_pack4", PACK, dict(x_type=3), UNSUPPORTED),
    ("b200_op_pack4", PACK, dict(by_column=2), ARG), ("b200_op_pack4", PACK, dict(x=0), ARG), ("b200_op_pack4", PACK, dict(q=0), ARG), ("b200_op_pack4", PACK, dict(scale=0), ARG),
    ("b200_op_pack4", PACK, dict(ldx=39), ARG), ("b200_op_pack4", PACK, dict(ldq=16), ARG), ("b200_op_pack4", PACK, dict(ldq=40), ARG), ("b200_op_pack4", PACK, dict(q=A + 8), ARG),
    ("b200_op_pack4", PACK, dict(scale=A + 4), ARG), ("b200_op_pack4", PACK, dict(x=A + 1), ARG), ("b200_op_pack4", PACK, dict(by_column=1, rows=40, ldq=16), ARG),
    ("b200_op_unpack4", UNPACK, dict(y_type=3), UNSUPPORTED), ("b200_op_unpack4", UNPACK, dict(q=0), ARG), ("b200_op_unpack4", UNPACK, dict(scale=0), ARG),
    ("b200_op_unpack4", UNPACK, dict(ldy=39), ARG), ("b200_op_unpack4", UNPACK, dict(ldq=-16), ARG), ("b200_op_unpack4", UNPACK, dict(y=A + 1), ARG),
    ("b200_op_dense4", DENSE, dict(rows=-1), ARG), ("b200_op_dense4", DENSE, dict(in_=0), ARG), ("b200_op_dense4", DENSE, dict(out=0), ARG), ("b200_op_dense4", DENSE, dict(y_type=3), UNSUPPORTED),
    ("b200_op_dense4", DENSE, dict(act=4), ARG), ("b200_op_dense4", DENSE, dict(x=0), ARG), ("b200_op_dense4", DENSE, dict(w=0), ARG), ("b200_op_dense4", DENSE, dict(x_scale=0), ARG),
    ("b200_op_dense4", DENSE, dict(w_scale=0), ARG), ("b200_op_dense4", DENSE, dict(ldx=16), ARG), ("b200_op_dense4", DENSE, dict(ldw=16), ARG), ("b200_op_dense4", DENSE, dict(ldw=40), ARG),
    ("b200_op_dense4", DENSE, dict(w=A + 8), ARG), ("b200_op_dense4", DENSE, dict(ldy=15), ARG), ("b200_op_dense4", DENSE, dict(residual=A, ldr=15), ARG),
    ("b200_op_dense4", DENSE, dict(bias=A + 1), ARG), ("b200_op_dense4", DENSE, dict(y=0), ARG),
]


@pytest.mark.parametrize("name", STRUCTS)
def test_structures_are_the_headers(name):
    header = open(os.path.join(ROOT, "include", "bullet_b200.h")).read()
    header = header.replace("uint8_t*", "float*")  # (pointers all)
    assert header_fields(header, name) == list(STRUCTS[name]._fields_)
    rust = open(os.path.join(ROOT, "bindings", "rust", "b200-sys", "src", "lib.rs")).read()
    body = re.search(r"pub struct %s \{(.*?)\n\}" % name, rust, re.S).group(1)
    assert [n.replace("r#in", "in_") for n in re.findall(r"pub ([\w#]+):", body)] == [n for n, _ in STRUCTS[name]._fields_]


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


@pytest.mark.parametrize("entry,good", [("b200_op_pack4", PACK), ("b200_op_unpack4", UNPACK), ("b200_op_dense4", DENSE)])
def test_no_rows_need_no_memory_and_no_device(entry, good):
    empty = {k: (0 if v == A or k == "rows" else v) for k, v in good.items()}
    assert getattr(_lib.load(), entry)(0, None, ctypes.byref(KINDS[entry](**empty))) == 0


def test_tensor_calls_name_what_is_wrong():
    torch = pytest.importorskip("torch")
    from bullet_b200 import ops

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    p = ops.Packed4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), 64)
    with pytest.raises(ValueError, match="x: "):
        ops.pack4(x)
    with pytest.raises(ValueError, match="packed: "):
        ops.unpack4(p)
    with pytest.raises(ValueError, match="both in 4 bits"):
        ops.dense(p, x)
    with pytest.raises(ValueError, match="of x by row and of w by column"):
        ops.dense(p, p)
    w = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="requires a gradient"):
        ops.pack4(w)
    with pytest.raises(ValueError, match="requires a gradient"):
        ops.dense(p, p._replace(by_column=True), residual=w)
