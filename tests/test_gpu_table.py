"""Sums of a table's rows that lists of ids name, and their gradient, on the GPU against plain forms in 64 bits.

Tolerances.  A sum of k values in 32 bits is off by at most k 2^-23 of the sum of their magnitudes, in any order, and sums of small whole numbers are exact.  A
value rounded to a type with p significand bits is off by at most 2^-p of itself (24, 8 and 11 bits: fp32, bf16, fp16), times a scale by one rounding more."""
import pytest
import torch

from bullet_b200 import _lib, ops

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROUND = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}  # half a step below fp16's smallest normal number


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(seed, *shape):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def spaced(t, pad, at=0):
    """The same matrix with `pad` more elements between rows, `at` elements into a buffer of NaN (ids: of 0)."""
    rows, cols = t.shape
    raw = torch.full((at + rows * (cols + pad),), 0.0 if not t.is_floating_point() else float("nan"), device="cuda").to(t.dtype)
    v = raw[at:].view(rows, cols + pad)[:, :cols]
    v.copy_(t)
    return v


def near(got, want, relative, absolute=0.0):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    off = (got - want).abs() - (relative * want.abs() + absolute)
    assert not torch.isnan(off).any() and off.max() <= 0 if off.numel() else True, float(off.max())


def lists(seed, rows, slots, n, kind=torch.int32, how="skewed"):
    g = gen(seed)
    u = torch.rand(rows, slots, device="cuda", generator=g)
    ids = {"skewed": (u.pow(3) * n).long(), "even": (u * n).long(), "one": torch.full((rows, slots), n // 2, device="cuda"), "none": torch.full((rows, slots), -1, device="cuda"),
           "all": torch.arange(rows * slots, device="cuda").view(rows, slots) % n}[how].clamp(max=n - 1)
    if how != "all":
        empty = torch.rand(rows, slots, device="cuda", generator=g) < 0.2
        other = torch.tensor([-1, n, -(2 ** 31), 2 ** 31 - 1], device="cuda")[torch.randint(0, 4, (rows, slots), device="cuda", generator=g)]
        ids = torch.where(empty, other, ids)
    return ids.to(kind)


def embed64(table, ids, scale):
    there = (ids >= 0) & (ids < table.shape[0])
    t, y = table.double(), torch.zeros(ids.shape[0], table.shape[1], dtype=torch.float64, device="cuda")
    for s in range(ids.shape[1]):
        y += torch.where(there[:, s, None], t[ids[:, s].long().clamp(0, len(t) - 1)], 0.0)
    return y * scale


def gradient64(dy, ids, n, scale):
    out = torch.zeros(n + 1, dy.shape[1], dtype=torch.float64, device="cuda")
    there = (ids >= 0) & (ids < n)
    for s in range(ids.shape[1]):
        out.index_add_(0, torch.where(there[:, s], ids[:, s].long(), n), dy.double())
    return out[:n] * scale


SHAPES = [(1, 1, 1, 1), (1, 32, 768, 1024), (2, 32, 12288, 256), (3, 5, 7, 33), (17, 1, 8, 520), (300, 3, 1000, 40), (64, 1, 1, 8), (65, 1, 1, 16), (129, 31, 100, 7),
          (1000, 32, 12288, 64), (5003, 1, 8, 136), (4097, 2, 255, 24), (4096, 1, 256, 16), (900, 20, 70000, 12), (20000, 7, 300, 48)]


@pytest.mark.parametrize("rows,slots,n,cols", SHAPES)
@pytest.mark.parametrize("kind,out", [(BF16, BF16), (BF16, F32), (F32, F32), (F16, F16), (F32, BF16)])
@pytest.mark.parametrize("ids_kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("pad,at", [(0, 0), (8, 0), (3, 1)])
def test_embed(rows, slots, n, cols, kind, out, ids_kind, pad, at):
    table, ids = spaced(normal(11, n, cols).to(kind), pad, at), lists(12, rows, slots, n, ids_kind)
    got = ops.embed(table, spaced(ids, pad, at), scale=0.7, out_dtype=out)
    size = embed64(table.abs(), ids, 0.7) * slots * 2.0 ** -23
    near(got, embed64(table, ids, float(torch.tensor(0.7, dtype=F32))), ROUND[out] + 2.0 ** -22, size + TINY[out])
    assert torch.equal(got, ops.embed(table, ids, scale=0.7, out_dtype=out))
    if out is kind:
        assert torch.equal(got, ops.embed(table, ids, scale=0.7))
    if slots == 1:
        assert torch.equal(got, ops.embed(table, ids[:, 0], scale=0.7, out_dtype=out))


@pytest.mark.parametrize("rows,slots,n,cols", SHAPES)
@pytest.mark.parametrize("kind,out", [(BF16, F32), (BF16, BF16), (F32, F32), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("how", ["skewed", "even", "one", "all"])
@pytest.mark.parametrize("pad,at", [(0, 0), (3, 1)])
def test_gradient(rows, slots, n, cols, kind, out, how, pad, at):
    dy, ids = spaced(normal(21, rows, cols).to(kind), pad, at), lists(22, rows, slots, n, how=how)
    got = ops.embed_backward(dy, spaced(ids, pad, at), n, scale=0.7, dtype=out)
    want = gradient64(dy, ids, n, float(torch.tensor(0.7, dtype=F32)))
    # of the most that a row is met, in stretches of 64 whose sums are added up
    met = torch.bincount(ids[(ids >= 0) & (ids < n)].long(), minlength=n).max().item() if n < 10 ** 6 else rows * slots
    size = gradient64(dy.abs(), ids, n, 0.7) * (64 + met / 64 + 2) * 2.0 ** -23
    near(got, want, ROUND[out] + 2.0 ** -22, size + TINY[out])
    assert torch.equal(got, ops.embed_backward(dy, ids.long(), n, scale=0.7, dtype=out))
    if slots == 1:
        assert torch.equal(got, ops.embed_backward(dy, ids[:, 0], n, scale=0.7, dtype=out))


@pytest.mark.parametrize("rows,slots,n,cols,how", [(70000, 1, 3, 8, "even"), (70000, 1, 40, 8, "skewed"), (3000, 32, 20000, 16, "skewed"), (300000, 1, 100000, 8, "even"),
                                                   (150000, 3, 300, 8, "skewed"), (131072, 1, 12288, 16, "even"), (9000, 32, 12288, 8, "skewed"), (8192, 1, 12288, 8, "even"),
                                                   (8193, 1, 12288, 8, "one"), (40, 1, 5000000, 8, "even"), (100000, 1, 20000000, 1, "even"), (2000, 3, 2 ** 24, 1, "all")])
def test_gradient_of_whole_numbers_is_exact(rows, slots, n, cols, how):
    dy, ids = torch.randint(-3, 4, (rows, cols), device="cuda", generator=gen(31)).to(BF16), lists(32, rows, slots, n, how=how)
    got = ops.embed_backward(dy, ids, n, scale=0.5)
    assert torch.equal(got.double(), gradient64(dy, ids, n, 0.5))


def test_gradients_sums_are_taken_in_the_order_of_the_lists():
    """Values whose sum in fp32 depends on the order: a row's up to 64 lists one after another, from the first on."""
    rows, n = 3000, 60
    ids, dy = lists(41, rows, 1, n, how="even"), normal(42, rows, 8) * torch.exp(4 * normal(43, rows, 1))
    got = ops.embed_backward(dy, ids, n)
    for t in range(n):
        mine = dy[ids[:, 0] == t]
        if len(mine) <= 64:
            sum_ = torch.zeros(8, device="cuda")
            for row in mine:
                sum_ += row
            assert torch.equal(got[t], sum_), t


@pytest.mark.parametrize("rows,slots", [(50, 4), (20000, 8)])
def test_lists_without_ids(rows, slots):
    table, dy = normal(51, 100, 40), normal(52, rows, 40)
    ids = lists(53, rows, slots, 100, how="none")
    assert not ops.embed(table, ids).any() and not ops.embed_backward(dy, ids, 100).any()
    assert ops.embed(table, ids[:0]).shape == (0, 40) and not ops.embed_backward(dy[:0], ids[:0], 100).any()


def test_what_is_not_finite_stays_where_it_belongs():
    table, dy = normal(54, 50, 24), normal(55, 400, 24)
    table[7], dy[11] = float("nan"), float("inf")
    ids = lists(56, 400, 3, 50)
    ids[11] = torch.tensor([3, -1, 4])
    bad = torch.isnan(ops.embed(table, ids))
    assert torch.equal(bad, (ids == 7).any(1)[:, None].expand_as(bad)) and bad.any()
    grad = ops.embed_backward(dy, ids, 50)
    assert torch.equal(torch.isfinite(grad).all(1).nonzero()[:, 0], torch.tensor([t for t in range(50) if t not in (3, 4)], device="cuda"))
    # a list that names nothing is not touched by the table's first row, nor the first row by its gradient
    table[0], none = float("nan"), torch.full((5, 3), -1, device="cuda")
    assert not ops.embed(table, none).any() and not ops.embed_backward(torch.full((5, 24), float("nan"), device="cuda"), none, 50).any()


def test_gradient_against_differences_and_the_forward():
    """embed is linear: <embed(t), dy> = <t, embed_backward(dy)> for any t, and a difference of the first along t is the second's product with t."""
    rows, slots, n, cols = 700, 9, 90, 40
    ids, dy = lists(61, rows, slots, n), normal(62, rows, cols)
    grad = ops.embed_backward(dy, ids, n, scale=0.3)
    table, along = normal(63, n, cols), normal(64, n, cols)
    h = 0.5  # (no error of a linear function's)
    up, down = ops.embed(table + h * along, ids, scale=0.3), ops.embed(table - h * along, ids, scale=0.3)
    difference = ((up.double() - down.double()) * dy.double()).sum() / (2 * h)
    formula = (grad.double() * along.double()).sum()
    size = (embed64(table.abs() + along.abs(), ids, 0.3) * dy.abs().double()).sum()
    assert abs(float(difference - formula)) < float(size) * slots * 2.0 ** -21


@pytest.mark.parametrize("rows", [5, 6000])
def test_calls_run_on_the_current_stream_and_in_graphs(rows):
    table, dy = normal(71, 768, 64).to(BF16), normal(72, rows, 64).to(BF16)
    ids = lists(73, rows, 4, 768)
    want = ops.embed(table, ids), ops.embed_backward(dy, ids, 768)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(10000000)
        got = ops.embed(table, ids), ops.embed_backward(dy, ids, 768)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph, held = torch.cuda.CUDAGraph(), ids.clone()
    with torch.cuda.graph(graph):
        out = ops.embed(table, held), ops.embed_backward(dy, held, 768)
    for seed in (74, 75):
        held.copy_(lists(seed, rows, 4, 768))
        graph.replay()
        assert torch.equal(out[0], ops.embed(table, held)) and torch.equal(out[1], ops.embed_backward(dy, held, 768))


def test_tables_pass_32_bit_offsets():
    n, cols = 2200000, 1024
    table = torch.zeros(n, cols, dtype=BF16, device="cuda")
    table[-100:] = normal(81, 100, cols).to(BF16)
    ids = torch.randint(n - 100, n, (500, 3), device="cuda", generator=gen(82))
    assert torch.equal(ops.embed(table, ids), ops.embed(table[-100:], ids - (n - 100)))
    dy = normal(83, 500, cols).to(BF16)
    del table
    got = ops.embed_backward(dy, ids, n, dtype=BF16)
    assert torch.equal(got[-100:], ops.embed_backward(dy, ids - (n - 100), 100, dtype=BF16)) and not got[:1000].any() and not got[-300:-100].any()
    del got
    y = ops.embed(normal(84, 5, cols).to(BF16), torch.arange(n, device="cuda") % 5)
    assert torch.equal(y[-10:], y[:10])  # (n is a multiple of 5)
    assert torch.equal(ops.embed_backward(y, torch.arange(n, device="cuda") - (n - 10), 10, dtype=BF16), y[-10:])


def test_refusals():
    table, ids, dy = normal(91, 10, 16), lists(92, 6, 3, 10), normal(93, 6, 16)
    for call in (lambda: ops.embed(table, ids.float()), lambda: ops.embed(table, ids.to(torch.int16)), lambda: ops.embed(table, ids.cpu()), lambda: ops.embed(table.double(), ids),
                 lambda: ops.embed(table, ids.t()), lambda: ops.embed(table, ids[None]), lambda: ops.embed(table, ids, out_dtype=torch.int8), lambda: ops.embed(table[0], ids),
                 lambda: ops.embed_backward(dy[:5], ids, 10), lambda: ops.embed_backward(dy, ids, -1), lambda: ops.embed_backward(dy, ids, 10, dtype=torch.float64),
                 lambda: ops.embed_backward(dy.t(), ids, 10), lambda: ops.embed(table, ids[:1].expand(4, 3)), lambda: ops.embed(table, torch.tensor(3, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.embed(table[:0], ids), lambda: ops.embed(table, ids[:, :0]), lambda: ops.embed_backward(dy, ids, 0), lambda: ops.embed(table[:, :0], ids)):
        with pytest.raises(_lib.B200Error):
            call()
    with pytest.raises(TypeError):
        ops.embed(table, ids, scale="x")
