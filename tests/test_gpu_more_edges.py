"""Edges of the operators in 4 bits, of embedded rows and of the gradients' norm, over the C ABI where tensors do not get there: results inside larger matrices, what lies
around them, first calls of a process that a stream captures, calls of several threads and streams at once."""
import ctypes
import os
import subprocess
import sys
import threading

import pytest
import torch

from bullet_b200 import _lib, ops

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPE = {F32: 0, BF16: 1, F16: 2}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GUARD = 77


def normal(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g)


def call(entry, op):
    _lib.check(getattr(_lib.load(), entry)(0, torch.cuda.current_stream().cuda_stream, ctypes.byref(op)))


def guarded(rows, cols, kind, pad, at):
    """(buffer, view): rows of `cols` with `pad` elements of GUARD between them, `at` in front, more behind."""
    raw = torch.full((at + rows * (cols + pad) + 64,), GUARD, device="cuda").to(kind)
    return raw, raw[at:at + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]


def around(raw, view, at):
    """What is not of the view is as it was."""
    kept = torch.ones(raw.shape, dtype=torch.bool, device="cuda")
    rows, cols = view.shape
    kept[at:at + rows * view.stride(0)].view(rows, view.stride(0))[:, :cols] = False
    return bool((raw[kept] == GUARD).all())


LAYOUTS = [(0, 0), (8, 0), (3, 0), (0, 1), (5, 3), (16, 16)]


@pytest.mark.parametrize("rows,n_in,n_out", [(1, 64, 23), (3, 96, 8), (9, 64, 40), (130, 300, 264), (300, 64, 7), (257, 128, 33), (1000, 96, 520)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("pad,at", LAYOUTS)
def test_layers_write_their_rows_alone(rows, n_in, n_out, kind, pad, at):
    x, w = ops.pack4(normal(1, rows, n_in)), ops.pack4(normal(2, n_in, n_out), by_column=True)
    r = normal(3, rows, n_out).to(kind)
    raw, y = guarded(rows, n_out, kind, pad, at)
    op = _lib.CDense4(rows=rows, in_=n_in, out=n_out, y_type=TYPE[kind], act=1, ldx=x.codes.stride(0), ldw=w.codes.stride(0), ldr=n_out, ldy=n_out + pad, x=x.codes.data_ptr(),
                      x_scale=x.scale.data_ptr(), w=w.codes.data_ptr(), w_scale=w.scale.data_ptr(), residual=r.data_ptr(), y=y.data_ptr())
    call("b200_op_dense4", op)
    assert torch.equal(y, ops.dense(x, w, act=1, residual=r, out_dtype=kind)) and around(raw, y, at)


@pytest.mark.parametrize("rows,cols", [(1, 33), (5, 64), (130, 200), (33, 16)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("by_column", [0, 1])
@pytest.mark.parametrize("pad,at", LAYOUTS)
def test_packing_there_and_back_writes_its_rows_alone(rows, cols, kind, by_column, pad, at):
    x = normal(4, rows, cols).to(kind)
    want = ops.pack4(x, by_column=bool(by_column))
    lists, width = want.codes.shape
    raw_q, q = guarded(lists, width, torch.uint8, 32, 16)
    scale = torch.full((want.scale.numel() + 64,), GUARD, device="cuda", dtype=torch.uint8)
    call("b200_op_pack4", _lib.CPack4(rows=rows, cols=cols, x_type=TYPE[kind], by_column=by_column, ldx=cols, ldq=width + 32, x=x.data_ptr(), q=q.data_ptr(), scale=scale.data_ptr()))
    assert torch.equal(q, want.codes) and around(raw_q, q, 16)
    assert torch.equal(scale[:want.scale.numel()], want.scale) and (scale[want.scale.numel():] == GUARD).all()
    raw, y = guarded(rows, cols, kind, pad, at)
    call("b200_op_unpack4", _lib.CUnpack4(rows=rows, cols=cols, y_type=TYPE[kind], by_column=by_column, ldq=width + 32, ldy=cols + pad, q=q.data_ptr(), scale=scale.data_ptr(),
                                          y=y.data_ptr()))
    assert torch.equal(y, ops.unpack4(want, kind)) and around(raw, y, at)


@pytest.mark.parametrize("rows,slots,n,cols", [(1, 3, 5, 7), (70, 1, 9, 24), (3000, 2, 50, 33), (2000, 1, 3, 136), (9000, 1, 5, 40), (600, 9, 800, 64)])
@pytest.mark.parametrize("kind,out", [(BF16, F32), (F32, F16), (F16, BF16)])
@pytest.mark.parametrize("pad,at", LAYOUTS)
def test_embedded_rows_and_their_gradient_write_their_rows_alone(rows, slots, n, cols, kind, out, pad, at):
    table, dy = normal(5, n, cols).to(kind), normal(6, rows, cols).to(kind)
    ids = torch.randint(-1, n, (rows, slots), device="cuda", dtype=torch.int32)
    raw, y = guarded(rows, cols, out, pad, at)
    call("b200_op_embed", _lib.CEmbed(rows=rows, slots=slots, n=n, cols=cols, table_type=TYPE[kind], y_type=TYPE[out], ldids=slots, ldt=cols, ldy=cols + pad, ids=ids.data_ptr(),
                                      table=table.data_ptr(), y=y.data_ptr(), scale=0.5))
    assert torch.equal(y, ops.embed(table, ids, scale=0.5, out_dtype=out)) and around(raw, y, at)
    raw, d = guarded(n, cols, out, pad, at)
    op = _lib.CEmbedGrad(rows=rows, slots=slots, n=n, cols=cols, dy_type=TYPE[kind], dtable_type=TYPE[out], ldids=slots, lddy=cols, lddt=cols + pad, ids=ids.data_ptr(), dy=dy.data_ptr(),
                         dtable=d.data_ptr(), scale=0.5)
    need = ctypes.c_int64()
    _lib.check(_lib.load().b200_op_embed_backward_workspace(ctypes.byref(op), ctypes.byref(need)))
    # (what the workspace holds before does not count, and nothing is written behind it)
    space = torch.full((need.value + 256,), GUARD, device="cuda", dtype=torch.uint8)
    op.workspace, op.workspace_bytes = space.data_ptr(), need.value
    for fill in (GUARD, 255, 0):
        space[:need.value] = fill
        call("b200_op_embed_backward", op)
        assert torch.equal(d, ops.embed_backward(dy, ids, n, scale=0.5, dtype=out)) and around(raw, d, at) and (space[need.value:] == GUARD).all()


def test_no_rows_leave_what_lies_between_a_gradients_rows():
    raw, d = guarded(6, 20, F32, 4, 1)
    call("b200_op_embed_backward", _lib.CEmbedGrad(rows=0, slots=1, n=6, cols=20, dy_type=0, dtable_type=0, ldids=1, lddy=20, lddt=24, dtable=d.data_ptr(), scale=1.0))
    assert not d.any() and around(raw, d, 1)


def test_gradients_that_are_counted_and_not_written():
    g = [normal(7, 5000), normal(8, 300).to(BF16), normal(9, 40)]
    raw, out = guarded(1, 300, BF16, 0, 3)
    norm, space = torch.full((3,), float(GUARD), device="cuda"), torch.full((1 << 16,), GUARD, device="cuda", dtype=torch.uint8)
    array = (_lib.CGradient * 3)(_lib.CGradient(g[0].data_ptr(), None, 5000, 0), _lib.CGradient(g[1].data_ptr(), out.data_ptr(), 300, 1), _lib.CGradient(g[2].data_ptr(), g[2].data_ptr(), 40, 0))
    op = _lib.CClip(count=3, gradients=ctypes.addressof(array), norm=norm[1:].data_ptr(), workspace=space.data_ptr(), max_norm=1.0)
    need = ctypes.c_int64()
    _lib.check(_lib.load().b200_op_clip_gradients_workspace(ctypes.byref(op), ctypes.byref(need)))
    op.workspace_bytes = need.value
    before = [t.clone() for t in g]
    call("b200_op_clip_gradients", op)
    want, total = ops.clip_gradients(before, 1.0)
    assert torch.equal(g[0], before[0]) and torch.equal(out[0], want[1]) and torch.equal(g[2], want[2]) and around(raw, out, 3)
    assert norm[1] == total and norm[0] == GUARD and norm[2] == GUARD and (space[need.value:] == GUARD).all()


@pytest.mark.parametrize("what", ["ops.dense(x, w)", "ops.dense(x1, w)", "ops.pack4(a).codes", "ops.unpack4(x)", "ops.embed(a, ids)", "ops.embed_backward(a, ids, 12288)", "ops.embed_backward(a, few, 8)",
                                  "ops.clip_gradients([a, a[:3].clone()], 0.5)[0][0]", "ops.gradient_norm([a])"])
def test_the_first_call_of_a_process_may_be_one_that_a_stream_captures(what):
    code = f"""
import torch
from bullet_b200 import ops
g = torch.Generator(device="cuda"); g.manual_seed(1)
a = torch.randn(9000, 256, device="cuda", generator=g)
ids = torch.randint(0, 9000, (9000,), device="cuda", generator=g)
few = ids % 8
code = torch.randint(0, 256, (9000, 128), device="cuda", generator=g, dtype=torch.uint8)
x = ops.Packed4(code, torch.full((71 * 2 * 512,), 127, device="cuda", dtype=torch.uint8), 256)
x1 = ops.Packed4(code[:1], x.scale[:1024], 256)
w = ops.Packed4(code[:64], x.scale[:1024], 256, True)
stream = torch.cuda.Stream()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    out = {what}
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, {what})
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_calls_of_several_threads_and_streams_at_once():
    a, ids = normal(11, 20000, 256).to(BF16), torch.randint(-1, 768, (20000, 4), device="cuda", dtype=torch.int32)
    w = ops.pack4(normal(12, 256, 512), by_column=True)

    def step():
        x = ops.pack4(a)
        return ops.dense(x, w), ops.unpack4(x), ops.embed(a[:768], ids), ops.embed_backward(a, ids, 768), *ops.clip_gradients([a, a[:100]], 3.0)[0]

    want, failed = step(), []
    torch.cuda.synchronize()

    def run():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step()
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(g, v) for g, v in zip(got, want))
        except BaseException as e:  # (of a thread: reported by the test)
            failed.append(e)

    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_two_graphs_of_one_workspace():
    """Two captured gradients that are lent the same memory, replayed one after the other."""
    rows, n, cols = 9000, 12, 64
    dy = normal(13, rows, cols)
    lists = [torch.randint(0, n, (rows,), device="cuda", dtype=torch.int32) for _ in range(2)]
    out = [torch.empty(n, cols, device="cuda") for _ in range(2)]
    space, graphs = torch.empty(1 << 24, device="cuda", dtype=torch.uint8), []
    for ids, d in zip(lists, out):
        op = _lib.CEmbedGrad(rows=rows, slots=1, n=n, cols=cols, dy_type=0, dtable_type=0, ldids=1, lddy=cols, lddt=cols, ids=ids.data_ptr(), dy=dy.data_ptr(), dtable=d.data_ptr(),
                             workspace=space.data_ptr(), scale=1.0, workspace_bytes=space.numel())
        call("b200_op_embed_backward", op)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call("b200_op_embed_backward", op)
        graphs.append(graph)
    for _ in range(3):
        for d in out:
            d.fill_(float("nan"))
        for graph in graphs:
            graph.replay()
        for ids, d in zip(lists, out):
            assert torch.equal(d, ops.embed_backward(dy, ids, n))


def test_a_stretch_of_many_pieces():
    """More than 16 x 16 pieces of one row, and 16 x 16 x 16 + 1 of another: groups of one member among them."""
    rows = 16 * 16 * 16 * 64 + 64 * 300 + 70
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ids[64 * 300:64 * 300 + 70] = 3
    ids[64 * 300 + 70:] = 5
    ids = ids[torch.randperm(rows, device="cuda")]
    dy = torch.randint(-3, 4, (rows, 8), device="cuda").to(BF16)
    want = torch.zeros(7, 8, dtype=torch.float64, device="cuda").index_add_(0, ids.long(), dy.double())
    assert torch.equal(ops.embed_backward(dy, ids, 7).double(), want)


@pytest.mark.parametrize("count", [65, 80, 16 * 16 + 1, 16 * 64 + 1, 16 * 16 * 16 + 1, 16 * 16 * 16 + 17, 70000])
@pytest.mark.parametrize("others", [0, 9000])
def test_stretches_at_the_borders_of_their_groups(count, others):
    ids = torch.cat((torch.full((count,), 2, device="cuda"), torch.arange(others, device="cuda") % 1000 + 3)).to(torch.int32)
    ids = ids[torch.randperm(len(ids), device="cuda")]
    dy = torch.randint(-3, 4, (len(ids), 72), device="cuda").to(BF16)
    want = torch.zeros(1003, 72, dtype=torch.float64, device="cuda").index_add_(0, ids.long(), dy.double())
    assert torch.equal(ops.embed_backward(dy, ids, 1003).double(), want)


@pytest.mark.parametrize("rows", [3, 300])
def test_a_wait_that_gave_up_is_reported_once_by_the_next_call_in_4_bits(rows):
    x, w, word = ops.pack4(normal(21, rows, 64)), ops.pack4(normal(22, 64, 40), by_column=True), ctypes.POINTER(ctypes.c_int32)()
    want = ops.dense(x, w)
    _lib.check(_lib.load().b200_op_dense_gave_up(0, ctypes.byref(word)))
    if not word:
        pytest.skip("the device shares no memory while it is running")
    torch.cuda.synchronize()
    word[0] = 1
    with pytest.raises(_lib.B200Error, match="waited too long") as e:
        ops.dense(x, w)
    assert e.value.code == -2 and word[0] == 0 and torch.equal(ops.dense(x, w), want)


@pytest.mark.parametrize("counts", [(1,), (64, 1, 65), (30, 31, 32, 33, 61, 62, 63, 64, 65, 66), (129, 1, 1, 3000, 2), (4097, 7), (1,) * 9000, (65,) * 130, (20000, 64, 65, 1, 300)])
@pytest.mark.parametrize("pad,at", [(0, 0), (3, 1)])
@pytest.mark.parametrize("places", ["first", "last", "apart"])
def test_gradients_of_tables_with_more_rows_than_ids(counts, pad, at, places):
    """Such tables are set to 0 first: all of their rows, nothing around them; `counts`: how often rows of the table are met."""
    rows, cols = sum(counts), 24
    n = 2 * rows + 100
    named = torch.arange(len(counts)) if places == "first" else n - 1 - torch.arange(len(counts)) if places == "last" else torch.randperm(n)[:len(counts)]
    ids = named.repeat_interleave(torch.tensor(counts))[torch.randperm(rows)].to("cuda", torch.int32)
    dy = torch.randint(-3, 4, (rows, cols), device="cuda").to(BF16)
    raw, d = guarded(n, cols, F32, pad, at)
    op = _lib.CEmbedGrad(rows=rows, slots=1, n=n, cols=cols, dy_type=1, dtable_type=0, wide_ids=0, ldids=1, lddy=cols, lddt=cols + pad, ids=ids.data_ptr(), dy=dy.data_ptr(),
                         dtable=d.data_ptr(), scale=0.5)
    size = ctypes.c_int64()
    _lib.check(_lib.load().b200_op_embed_backward_workspace(ctypes.byref(op), ctypes.byref(size)))
    space = torch.full((size.value,), 255, dtype=torch.uint8, device="cuda")
    op.workspace, op.workspace_bytes = space.data_ptr(), size.value
    want = torch.zeros(n, cols, dtype=torch.float64, device="cuda").index_add_(0, ids.long(), dy.double()) / 2
    for _ in range(2):
        call("b200_op_embed_backward", op)
        assert torch.equal(d.double(), want) and around(raw, d, at)


@pytest.mark.parametrize("rows", [100, 9000])
def test_a_table_with_more_rows_than_ids_in_a_graph(rows):
    ids, dy = torch.randint(-1, 20, (rows, 1), device="cuda", dtype=torch.int32), normal(5, rows, 40)
    ops.embed_backward(dy, ids, 50000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d = ops.embed_backward(dy, ids, 50000)
    for seed in (1, 2):
        ids.copy_((ids * 7 + seed) % 49999)
        dy.copy_(normal(seed, rows, 40))
        graph.replay()
        assert torch.equal(d, ops.embed_backward(dy, ids, 50000))


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 256, 257, 5003, 200000])
@pytest.mark.parametrize("n", [1, 2, 8, 16, 17])
@pytest.mark.parametrize("cols,kind,out,pad,at,wide", [(520, BF16, F32, 0, 0, 0), (24, BF16, BF16, 0, 0, 1), (7, F16, F32, 3, 1, 0), (40, F32, F16, 8, 0, 0), (300, F32, F32, 3, 1, 1),
                                                       (4, BF16, F32, 0, 0, 0), (777, BF16, F32, 5, 3, 0), (32, F32, BF16, 0, 0, 0), (96, BF16, F32, 16, 16, 0)])
def test_gradients_of_tables_of_few_rows(rows, n, cols, kind, out, pad, at, wide):
    """Whole numbers, whose sums are exact: one id a list, some of them none, against 64 bits; the same bits every time; what lies around is left."""
    ids = torch.randint(-1, n + 1, (rows,), device="cuda", dtype=torch.int64 if wide else torch.int32)
    dy = guarded(rows, cols, kind, pad, at)[1]
    dy.copy_(torch.randint(-3, 4, (rows, cols), device="cuda"))
    raw, d = guarded(n, cols, out, pad, at)
    op = _lib.CEmbedGrad(rows=rows, slots=1, n=n, cols=cols, dy_type=TYPE[kind], dtable_type=TYPE[out], wide_ids=wide, ldids=1, lddy=cols + pad, lddt=cols + pad, ids=ids.data_ptr(),
                         dy=dy.data_ptr(), dtable=d.data_ptr(), scale=0.25)
    size = ctypes.c_int64()
    _lib.check(_lib.load().b200_op_embed_backward_workspace(ctypes.byref(op), ctypes.byref(size)))
    space = torch.full((size.value + 64,), 255, dtype=torch.uint8, device="cuda")
    op.workspace, op.workspace_bytes = space.data_ptr(), size.value
    to = torch.where((ids >= 0) & (ids < n), ids, n).long()
    want = (torch.zeros(n + 1, cols, dtype=torch.float64, device="cuda").index_add_(0, to, dy.double()) / 4)[:n].to(out)
    for _ in range(2):
        d.fill_(GUARD)
        call("b200_op_embed_backward", op)
        assert torch.equal(d, want) and around(raw, d, at) and bool((space[size.value:] == 255).all())


def test_what_is_not_finite_stays_in_its_row_and_column_of_a_table_of_few_rows():
    ids, dy = torch.arange(3000, device="cuda", dtype=torch.int32) % 9 - 1, normal(3, 3000, 40)
    clean = ops.embed_backward(dy, ids, 8)
    dy[90, 3], dy[91, 5], dy[92] = float("nan"), float("inf"), float("-inf")  # of ids -1, 0 and 1
    dirty = ops.embed_backward(dy, ids, 8)
    kept = torch.ones(8, 40, dtype=torch.bool, device="cuda")
    kept[0, 5], kept[1] = False, False
    assert torch.equal(clean[kept], dirty[kept]) and torch.isposinf(dirty[0, 5]) and bool(torch.isneginf(dirty[1]).all())


def test_stretches_of_many_pieces_of_larger_tables():
    """As test_a_stretch_of_many_pieces, of a table that is not one of few rows."""
    rows = 16 * 16 * 16 * 64 + 64 * 300 + 70
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ids[64 * 300:64 * 300 + 70] = 33
    ids[64 * 300 + 70:] = 65
    ids = ids[torch.randperm(rows, device="cuda")]
    dy = torch.randint(-3, 4, (rows, 8), device="cuda").to(BF16)
    want = torch.zeros(70, 8, dtype=torch.float64, device="cuda").index_add_(0, ids.long(), dy.double())
    assert torch.equal(ops.embed_backward(dy, ids, 70).double(), want)
