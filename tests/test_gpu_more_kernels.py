"""The kernels of large calls in 4 bits and of embedded rows, on the GPU against 64 bits: each case says which kernel it is about, and that the call launches it is tested as well.

Whole numbers throughout, whose products and sums are exact in fp32 in any order: outputs are those of 64 bits, rounded once to their type, equal bit by bit.  What is not
finite has to stay in its row and column."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from bullet_b200 import _lib, ops
from bullet_b200.configs import ACT_NONE, ACT_RELU
from tests.kernels_launched import through
from tests.test_gpu_four import gen, random_codes, spaced, values
from tests.test_gpu_table import embed64, gradient64, lists

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def whole(seed, kind, *shape, most=8):
    return torch.randint(-most, most + 1, shape, device="cuda", generator=gen(seed)).to(kind)


# ---- layers in 4 bits

# One tile a pair of SMs and several, whose sums share places; all rows and columns there, and ragged ones; whole stages of 256 inputs, and 32 to 224 behind the last one.
PAIRS = [(2304, 2048, 2048), (2300, 2000, 2041), (5003, 1100, 2040), (9001, 1500, 1000), (16384, 1024, 2048), (300, 4096, 9000), (2500, 2079, 1900)]
ONES = [(9, 64, 48), (5003, 1100, 777), (3000, 512, 1024), (20000, 320, 256), (1000, 8200, 130)]
LAYERS = [(shape, (256, True)) for shape in PAIRS] + [(shape, (128, False)) for shape in ONES]


def layer(rows, n_in, n_out):
    """Operands whose products, multiples of 2^-4, have sums of magnitudes below 2^19."""
    return random_codes(41, rows, n_in, -1, 1), random_codes(42, n_out, n_in, -1, 0)._replace(by_column=True)


def check_layer(tile, x, w, out, residual, bias, act):
    got = through(lambda: ops.dense(x, w, bias=bias, act=act, residual=residual, out_dtype=out), "product4_kernel", *tile, residual is not None)
    want = values(x) @ values(w).t()
    if bias is not None:
        want += bias.double()
    if act == ACT_RELU:
        want = want.clamp(min=0)
    if residual is not None:
        # (a row's sum of 32 bits, then the residual: exact, as both are multiples of 2^-4 below 2^20)
        want += residual.double()
    assert torch.equal(got, want.to(out))


@pytest.mark.parametrize("shape,tile", LAYERS, ids=str)
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("adds", [False, True])
def test_tiles_of_layers(shape, tile, out, adds):
    rows, _, n_out = shape
    x, w = layer(*shape)
    check_layer(tile, x, w, out, whole(43, out, rows, n_out) if adds else None, whole(44, F32, n_out), ACT_RELU if adds else ACT_NONE)


@pytest.mark.parametrize("shape,tile", [(PAIRS[1], (256, True)), (PAIRS[2], (256, True)), (ONES[1], (128, False))], ids=str)
@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("pad,at", [(8, 0), (3, 1), (16, 8)])
def test_tiles_of_layers_inside_larger_matrices(shape, tile, out, pad, at):
    rows, _, n_out = shape
    x, w = layer(*shape)
    x, w = x._replace(codes=spaced(x.codes, 32, 16)), w._replace(codes=spaced(w.codes, 16, 32))
    check_layer(tile, x, w, out, spaced(whole(45, out, rows, n_out), pad, at), None, ACT_NONE)


@pytest.mark.parametrize("shape,tile", [(PAIRS[0], (256, True)), (PAIRS[2], (256, True)), (PAIRS[3], (256, True)), (ONES[2], (128, False))], ids=str)
@pytest.mark.parametrize("adds", [False, True])
def test_tiles_keep_groups_that_are_not_finite_in_their_rows_and_columns(shape, tile, adds):
    rows, n_in, n_out = shape
    x, w = layer(*shape)
    clean = through(lambda: ops.dense(x, w, out_dtype=F32), "product4_kernel", *tile, False)

    def place(r, g):
        return (r // 128 * ((n_in + 127) // 128) + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4

    groups = (n_in + 31) // 32
    bad_rows, bad_columns = [0, 129, 255, 256, rows - 1], [1, 127, 128, 300, n_out - 1]
    for k, r in enumerate(bad_rows):
        x.scale[place(r, (groups - 1) * k // 4)] = 255
    for k, c in enumerate(bad_columns):
        w.scale[place(c, (groups - 1) * (4 - k) // 4)] = 255
    residual = torch.zeros(rows, n_out, device="cuda") if adds else None
    got = through(lambda: ops.dense(x, w, residual=residual, out_dtype=F32), "product4_kernel", *tile, adds)
    bad = torch.zeros(rows, n_out, dtype=torch.bool, device="cuda")
    bad[bad_rows], bad[:, bad_columns] = True, True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], clean[~bad])


# ---- rows named by ids

# (lists, ids each, rows of the table, columns, type, bytes of a lane, rows on their way)
LOOKUPS = [(700, 18, 900, 1024, BF16, 32, 4), (3001, 32, 5000, 504, F16, 32, 4), (1300, 5, 300, 1000, F32, 32, 4), (500, 33, 700, 520, BF16, 16, 4), (700, 9, 2000, 600, F32, 16, 4),
           (300, 40, 700, 1024, BF16, 16, 16), (30, 7, 9, 1024, F32, 16, 16)]
SHORT = [(5003, 1, 8, 1024, BF16, 32), (3000, 2, 300, 256, F32, 32), (1300, 3, 40, 504, F16, 32), (2001, 4, 900, 1000, F32, 32), (40000, 1, 8, 512, BF16, 32), (131072, 1, 8, 1000, BF16, 32),
         (2500, 3, 50, 520, BF16, 16), (9000, 2, 77, 144, F32, 16)]
# (...; by places: the table has more rows than there are ids)
GRADIENTS = [(700, 9, 1500, 1024, BF16, 32, 4, False), (4000, 18, 12288, 1024, BF16, 32, 4, False), (2000, 5, 2900, 504, F16, 32, 4, False), (1100, 7, 2400, 1000, F32, 32, 4, False),
             (3000, 1, 2600, 248, F32, 32, 4, False), (700, 4, 2800, 520, BF16, 16, 4, False), (9000, 1, 40, 1024, BF16, 16, 16, False), (600, 9, 8000, 1024, BF16, 32, 4, True),
             (9001, 1, 20000, 504, F16, 32, 4, True), (1300, 5, 6600, 250, F32, 0, 4, True), (2500, 4, 10001, 248, F32, 32, 4, True), (700, 4, 2900, 520, BF16, 16, 4, True)]
WIDE = [torch.int32, torch.int64]


@pytest.mark.parametrize("rows,slots,n,cols,kind,lane,ahead", LOOKUPS)
@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("pad", [0, 32])
def test_lookups_of_long_lists(rows, slots, n, cols, kind, lane, ahead, out, pad):
    table, ids = spaced(whole(11, kind, n, cols), pad, pad), lists(12, rows, slots, n, WIDE[pad > 0])
    got = through(lambda: ops.embed(table, ids, scale=0.5, out_dtype=out), "embed_kernel", lane, ahead)
    assert torch.equal(got, embed64(table, ids, 0.5).to(out))


@pytest.mark.parametrize("rows,slots,n,cols,kind,lane", SHORT)
@pytest.mark.parametrize("out", [F32, F16])
@pytest.mark.parametrize("pad", [0, 32])
def test_lookups_of_short_lists(rows, slots, n, cols, kind, lane, out, pad):
    table, ids = spaced(whole(13, kind, n, cols), pad, pad), lists(14, rows, slots, n, WIDE[pad > 0])
    got = through(lambda: ops.embed(table, spaced(ids, pad, 1 if pad else 0), scale=0.5, out_dtype=out), "embed_short_kernel", lane)
    assert torch.equal(got, embed64(table, ids, 0.5).to(out))


@pytest.mark.parametrize("rows,slots,n,cols,kind,lane,ahead,places", GRADIENTS)
@pytest.mark.parametrize("how", ["even", "skewed"])
@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("pad", [0, 32])
def test_gradients(rows, slots, n, cols, kind, lane, ahead, places, how, out, pad):
    dy, ids = spaced(whole(21, kind, rows, cols, most=3), pad, pad), lists(22, rows, slots, n, WIDE[pad > 0], how=how)
    ids[::3, 0] = n // 2  # (a stretch of many pieces in any case)
    got = through(lambda: ops.embed_backward(dy, ids, n, scale=0.5, dtype=out), "embed_backward_kernel", lane, ahead, places)
    assert torch.equal(got, gradient64(dy, ids, n, 0.5).to(out))


@pytest.mark.parametrize("rows,slots,n,cols,kind,lane,ahead,places", [GRADIENTS[1], GRADIENTS[3], GRADIENTS[7]])
def test_gradients_of_values_that_are_not_finite(rows, slots, n, cols, kind, lane, ahead, places):
    dy, ids = whole(23, kind, rows, cols, most=3), lists(24, rows, slots, n)
    ids[ids == 5] = 6
    ids[7] = torch.tensor([5, -1, n] + [-1] * (slots - 3))
    clean = ops.embed_backward(dy, ids, n)
    dy[7, cols // 2 + 1] = float("nan")
    got = through(lambda: ops.embed_backward(dy, ids, n), "embed_backward_kernel", lane, ahead, places)
    bad = torch.zeros(n, cols, dtype=torch.bool, device="cuda")
    bad[5, cols // 2 + 1] = True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], clean[~bad])


# ---- the gradient's memory: of graphs that share it, and of a first call that a stream captures

SORTED = [(9000, 1, 40, 64), (5000, 1, 40, 64), (9000, 1, 20000, 64), (3000, 2, 9000, 40), (3000, 3, 2500, 1024), (9001, 1, 700, 248)]


@pytest.mark.parametrize("rows,slots,n,cols", SORTED)
def test_graphs_of_sorted_gradients_in_one_workspace(rows, slots, n, cols):
    """Two captured gradients that are lent the same memory for sorted ids, starts, pieces and their counters, replayed one after the other on inputs that change."""
    dy = whole(31, F32, rows, cols, most=3)
    ids = [lists(32 + k, rows, slots, n, how=("skewed", "one")[k]) for k in range(2)]
    out = [torch.empty(n, cols, device="cuda") for _ in range(2)]
    calls, need, space, graphs = [], ctypes.c_int64(), None, []
    for i, d in zip(ids, out):
        op = _lib.CEmbedGrad(rows=rows, slots=slots, n=n, cols=cols, dy_type=0, dtable_type=0, ldids=slots, lddy=cols, lddt=cols, ids=i.data_ptr(), dy=dy.data_ptr(), dtable=d.data_ptr(),
                             scale=1.0)
        _lib.check(_lib.load().b200_op_embed_backward_workspace(ctypes.byref(op), ctypes.byref(need)))
        space = torch.full((need.value,), 255, device="cuda", dtype=torch.uint8) if space is None else space
        op.workspace, op.workspace_bytes = space.data_ptr(), space.numel()
        calls.append(op)

    def run(op):
        _lib.check(_lib.load().b200_op_embed_backward(0, torch.cuda.current_stream().cuda_stream, ctypes.byref(op)))

    for op in calls:
        run(op)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(op)
    for seed in range(3):
        for k, i in enumerate(ids):
            i.copy_(lists(40 + seed + 7 * k, rows, slots, n, how=("one", "even", "skewed")[(seed + k) % 3]))
        for d in out:
            d.fill_(float("nan"))
        for graph in graphs:
            graph.replay()
        for i, d in zip(ids, out):
            assert torch.equal(d.double(), gradient64(dy, i, n, 1.0))


FIRST = """
import torch
from bullet_b200 import ops
from tests.test_gpu_four import random_codes
g = torch.Generator(device="cuda"); g.manual_seed(1)
a = torch.randn(9000, 256, device="cuda", generator=g)
wide = torch.randn(4000, 1024, device="cuda", generator=g)
ids = torch.randint(0, 9000, (9000,), device="cuda", generator=g)
x, w = random_codes(1, 2304, 2048, -1, 1), random_codes(2, 2048, 2048, -1, 0)._replace(by_column=True)
r = torch.ones(2304, 2048, device="cuda", dtype=torch.bfloat16)
stream = torch.cuda.Stream()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    out = WHAT
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, WHAT)
"""


@pytest.mark.parametrize("what", ["ops.embed_backward(a[:5000], ids[:5000] % 40, 40)", "ops.embed_backward(a[:5000], ids[:5000], 9000)", "ops.embed_backward(a, ids % 40, 40)",
                                  "ops.embed_backward(wide, ids[:4000] % 2500, 2500)", "ops.embed(wide, ids[:8000].view(1000, 8) % 4000)", "ops.embed(wide, ids[:8000] % 4000)",
                                  "ops.dense(x, w)", "ops.dense(x, w, residual=r)"])
def test_the_first_call_of_a_process_may_be_one_that_a_stream_captures(what):
    done = subprocess.run([sys.executable, "-c", FIRST.replace("WHAT", what)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
