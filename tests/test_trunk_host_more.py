"""CPU tests of the operators in 4 bits, of embedded rows and of the norm of gradients: what they refuse, and that the ctypes structures are the
header's."""
import ctypes
import os
import re

import pytest

from bullet_b200 import _lib
from tests.test_trunk_host import A, ARG, UNSUPPORTED, header_fields

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"b200_pack4_op": _lib.CPack4, "b200_unpack4_op": _lib.CUnpack4, "b200_dense4_op": _lib.CDense4, "b200_embed_op": _lib.CEmbed, "b200_embed_grad_op": _lib.CEmbedGrad,
           "b200_gradient": _lib.CGradient, "b200_clip_op": _lib.CClip}
KINDS = {"b200_op_pack4": _lib.CPack4, "b200_op_unpack4": _lib.CUnpack4, "b200_op_dense4": _lib.CDense4, "b200_op_embed": _lib.CEmbed, "b200_op_embed_backward": _lib.CEmbedGrad,
         "b200_op_clip_gradients": _lib.CClip}
EMBED = dict(rows=4, slots=3, n=10, cols=8, table_type=1, y_type=0, wide_ids=0, ldids=3, ldt=8, ldy=8, ids=A, table=A, y=A, scale=1.0)
EMBED_GRAD = dict(rows=4, slots=3, n=10, cols=8, dy_type=1, dtable_type=0, wide_ids=0, ldids=3, lddy=8, lddt=8, ids=A, dy=A, dtable=A, workspace=A, scale=1.0, workspace_bytes=1 << 30)


def gradients(*of):
    """An array of b200_gradient and its address as the field of a call; the array is kept."""
    array = (_lib.CGradient * len(of))(*(_lib.CGradient(*t) for t in of))
    KEPT.append(array)
    return dict(count=len(of), gradients=ctypes.addressof(array))


KEPT = []
CLIP = dict(**gradients((A, A, 100, 0), (A + 4096, A + 4096, 100, 1)), norm=A + 8192, workspace=A + 16384, max_norm=1.0, workspace_bytes=1 << 20)
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
    ("b200_op_embed", EMBED, dict(rows=-1), ARG), ("b200_op_embed", EMBED, dict(slots=0), ARG), ("b200_op_embed", EMBED, dict(n=0), ARG), ("b200_op_embed", EMBED, dict(cols=0), ARG),
    ("b200_op_embed", EMBED, dict(wide_ids=2), ARG), ("b200_op_embed", EMBED, dict(table_type=3), UNSUPPORTED), ("b200_op_embed", EMBED, dict(y_type=4), UNSUPPORTED),
    ("b200_op_embed", EMBED, dict(rows=1 << 30, slots=2), UNSUPPORTED), ("b200_op_embed", EMBED, dict(ids=0), ARG), ("b200_op_embed", EMBED, dict(ids=A + 4, wide_ids=1), ARG),
    ("b200_op_embed", EMBED, dict(ldids=2), ARG), ("b200_op_embed", EMBED, dict(table=0), ARG), ("b200_op_embed", EMBED, dict(ldt=7), ARG), ("b200_op_embed", EMBED, dict(y=A + 2), ARG),
    ("b200_op_embed_backward", EMBED_GRAD, dict(rows=-1), ARG), ("b200_op_embed_backward", EMBED_GRAD, dict(dy_type=3), UNSUPPORTED),
    ("b200_op_embed_backward", EMBED_GRAD, dict(dtable_type=3), UNSUPPORTED), ("b200_op_embed_backward", EMBED_GRAD, dict(dtable=0), ARG),
    ("b200_op_embed_backward", EMBED_GRAD, dict(dy=0), ARG), ("b200_op_embed_backward", EMBED_GRAD, dict(lddy=7), ARG), ("b200_op_embed_backward", EMBED_GRAD, dict(lddt=7), ARG),
    ("b200_op_embed_backward", EMBED_GRAD, dict(ids=A + 2), ARG), ("b200_op_embed_backward", EMBED_GRAD, dict(workspace_bytes=16), ARG),
    ("b200_op_embed_backward", EMBED_GRAD, dict(workspace=A + 8), ARG), ("b200_op_embed_backward", EMBED_GRAD, dict(wide_ids=-1), ARG),
    ("b200_op_embed", EMBED, dict(scale=float("inf")), ARG), ("b200_op_embed_backward", EMBED_GRAD, dict(scale=float("nan")), ARG),
    ("b200_op_clip_gradients", CLIP, dict(count=-1), ARG), ("b200_op_clip_gradients", CLIP, dict(gradients=0), ARG), ("b200_op_clip_gradients", CLIP, dict(norm=0), ARG),
    ("b200_op_clip_gradients", CLIP, dict(workspace=0), ARG), ("b200_op_clip_gradients", CLIP, dict(workspace_bytes=64), ARG), ("b200_op_clip_gradients", CLIP, dict(max_norm=-1.0), ARG),
    ("b200_op_clip_gradients", CLIP, dict(max_norm=float("nan")), ARG), ("b200_op_clip_gradients", CLIP, gradients((A, A, 100, 3)), UNSUPPORTED),
    ("b200_op_clip_gradients", CLIP, gradients((A, A, -1, 0)), ARG), ("b200_op_clip_gradients", CLIP, gradients((A, A, 1 << 60, 0)), ARG),
    ("b200_op_clip_gradients", CLIP, gradients((0, A, 5, 0)), ARG), ("b200_op_clip_gradients", CLIP, gradients((A + 2, A, 5, 0)), ARG),
    ("b200_op_clip_gradients", CLIP, gradients((A, A, 100, 0), (A, A, 100, 0)), ARG),
    ("b200_op_clip_gradients", CLIP, gradients((A, A + 40, 100, 0)), ARG), ("b200_op_clip_gradients", CLIP, gradients((A, A + 4096, 100, 0), (A + 4400, 0, 100, 1)), ARG),
    ("b200_op_clip_gradients", CLIP, gradients((A, A + 4096, 100, 0), (A + 8192, A + 4400, 100, 1)), ARG),
]


@pytest.mark.parametrize("name", STRUCTS)
def test_structures_are_the_headers(name):
    header = open(os.path.join(ROOT, "include", "bullet_b200.h")).read()
    header = header.replace("uint8_t*", "float*")  # (pointers all)
    assert header_fields(header, name) == list(STRUCTS[name]._fields_)
    rust = open(os.path.join(ROOT, "bindings", "rust", "b200-sys", "src", "lib.rs")).read()
    body = re.search(r"pub struct %s \{(.*?)\n\}" % name, rust, re.S).group(1)
    assert [n.replace("r#in", "in_").replace("r#", "") for n in re.findall(r"pub ([\w#]+):", body)] == [n for n, _ in STRUCTS[name]._fields_]


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


@pytest.mark.parametrize("entry,good", [("b200_op_pack4", PACK), ("b200_op_unpack4", UNPACK), ("b200_op_dense4", DENSE), ("b200_op_embed", EMBED)])
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
    ids = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="table: "):
        ops.embed(x, ids)
    with pytest.raises(ValueError, match="dy: "):
        ops.embed_backward(x, ids, 7)
    with pytest.raises(ValueError, match=r"gradients\[0\]: "):
        ops.gradient_norm([x])
    with pytest.raises(ValueError, match=r"gradients\[0\]: a tensor is wanted"):
        ops.clip_gradients([None], 1.0)
    with pytest.raises(ValueError, match="at least one"):
        ops.clip_gradients([], 1.0)
    with pytest.raises(TypeError):
        ops.clip_gradients([x], None)
    for call in (lambda: ops.embed(w, ids), lambda: ops.embed_backward(w, ids, 7), lambda: ops.clip_gradients([w], 1.0)):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
