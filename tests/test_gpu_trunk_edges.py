"""The dense trunk's operators at the edges of their ranges: scales of every size, what an activation's codes have to keep, waits that gave
up.  Expected values are the definitions in 64 bits; where a test asks for equality, every value on the way is exact."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from bullet_b200 import _lib, ops
from bullet_b200.configs import ACT_CRELU, ACT_NONE, ACT_RELU, ACT_SCRELU

pytestmark = pytest.mark.gpu
F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn


def kept(v, scale, act):
    """The values of the codes of an activation's outputs `v` at a scale: the nearest (halves to the even one), but above 0 what was above 0,
    and for outputs that are cut off at 1 below 1 what was below 1.  Scales up to 2^8, past which no code lies between."""
    codes = torch.arange(127, device=v.device, dtype=torch.uint8).view(E4M3).double()
    q = (v / scale).float().to(E4M3).double()  # (in fp32 exactly: a power of two)
    if act != ACT_NONE:
        q = torch.where((v > 0) & (q == 0), codes[1], q)
    if act in (ACT_CRELU, ACT_SCRELU):
        q = torch.where((v > 0) & (v < 1) & (q * scale >= 1), codes[codes * scale < 1].max(), q)
    return q * scale


# Scales 2^e around those at which the codes below 1 and above 0 change places: 2^5 is the last at which 15/16 is a code, 2^-117 the last at
# which half the smallest code is a normal number.
@pytest.mark.parametrize("e", [-120, -118, -117, -116, -20, -9, -8, -7, -1, 0, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("act", [ACT_NONE, ACT_CRELU, ACT_SCRELU, ACT_RELU])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_codes_of_outputs_keep_the_mask_at_every_scale(e, act, kind):
    if kind is F16 and not -8 <= e <= 7:
        pytest.skip("past fp16")
    scale = 2.0 ** e
    one = torch.tensor(1.0, dtype=kind)
    last = torch.nextafter(one, one * 0).item()
    below_one = [1.0, last, 0.999, 0.97, 0.95, 0.94, 0.9375, 0.93, 0.91, 0.9, 0.88, 0.876, 0.875, 0.8, 0.76, 0.75, 0.7, 0.6, 0.51, 0.5, 0.49, 0.3, 0.1]
    of_scale = [scale * f for f in (2.0 ** -12, 2.0 ** -10, 2.0 ** -9, 1.4 * 2.0 ** -9, 1.5 * 2.0 ** -9, 2.0 ** -6, 0.3, 1.0, 17.3, 239.0, 299.0)]
    values = torch.tensor([v for v in below_one + of_scale if v < 300 * scale] + [0.0], dtype=torch.float64, device="cuda").to(kind)
    top = torch.tensor([300 * scale], dtype=torch.float64, device="cuda").to(kind)
    for cols in (96, 77, 1100, 17000):  # vectors or single elements, one warp or several, rows past registers
        x = torch.zeros(5, cols, device="cuda", dtype=kind)
        for r in range(5):
            x[r, r:r + len(values)] = values
            x[r, cols - 1] = top[0]
        want = kept(x.double(), scale, act)
        p = ops.pack8(x, act=act)
        assert (p.scale == scale).all() and torch.equal(ops.unpack8(p, F32).double(), want), cols
        p = ops.pack8(x.t().contiguous(), act=act, by_column=True)
        assert (p.scale == scale).all() and torch.equal(ops.unpack8(p, F32).t().double(), want), cols


def near(got, want, absolute):
    off = (got.double() - want.double()).abs() - absolute
    assert not torch.isnan(off).any() and off.max() <= 0, float(off.max())


def random(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g)


def of_any_scale(rows, n_in):
    x, scale = random(1, rows, n_in), torch.exp(random(4, rows))
    x[4] = 320  # (beside a scale below fp32's normal numbers: the value is a normal one)
    scale[1], scale[2], scale[3], scale[4] = 0.0, -1.5, 1 + 2.0 ** -23, 2.0 ** -130
    return x.to(E4M3), scale


@pytest.mark.parametrize("rows,n_in,n_out", [(70, 64, 32), (300, 200, 700), (2500, 256, 512)])
def test_scales_that_are_no_powers_of_two_mean_the_same_to_unpack_and_the_gradients(rows, n_in, n_out):
    """unpack8 and both gradients take a scale as it is.  The weights' gradient multiplies bf16: each value is rounded by 2^-9 of
    itself there, which is nothing for powers of two.  Sums as in the other tests: 2^-23 of their magnitudes' sum a term."""
    (x, scale), y = of_any_scale(rows, n_in), random(7, rows, n_out).abs().clamp(max=1).to(E4M3)
    w, dy = random(2, n_in, n_out).to(BF16), random(3, rows, n_out).to(BF16)
    packed = ops.Packed8(x, scale)
    xv = x.double() * scale.double()[:, None]
    assert torch.equal(ops.unpack8(packed, F32), (x.float() * scale[:, None]))
    _, dw, _ = ops.dense_backward(dy, packed, None, need_dx=False)
    size = xv.abs().t() @ dy.double().abs()
    near(dw, xv.t() @ dy.double(), size * (2.0 ** -9 + rows * 2.0 ** -23))
    alone = torch.zeros_like(dy)  # a row at a time
    for k, row in enumerate((1, 2, 3, 4, 5)):
        alone[row, k] = 1
    _, dw, _ = ops.dense_backward(alone, packed, None, need_dx=False)
    assert torch.equal(dw, (xv.to(BF16).double().t() @ alone.double()).float())
    # dz is cut off by the value that y stands for
    sy = torch.exp(random(6, rows))
    yv = y.double() * sy.double()[:, None]
    dx, _, db = ops.dense_backward(dy, None, w, y=ops.Packed8(y, sy), act=ACT_CRELU, need_dw=False)
    dz = torch.where((yv > 0) & ((y.float() * sy[:, None]) < 1), dy.double(), torch.zeros_like(yv))
    near(db, dz.sum(0), dz.abs().sum(0) * (rows * 2.0 ** -23))
    near(dx, dz @ w.double().t(), (dz.abs() @ w.double().abs().t()) * (n_out * 2.0 ** -23 + 2.0 ** -8))


@pytest.mark.parametrize("rows,n_in,n_out", [(3, 64, 40), (8, 1024, 64), (17, 2048, 16), (70, 64, 32), (300, 200, 700), (1000, 96, 520), (2500, 256, 512)])
def test_dense_at_scales_whose_product_is_out_of_range(rows, n_in, n_out):
    """Whole numbers in codes, scales of 2^-126 to 2^119: what the scales make of an exact sum, rounded once.  A sum of 0 stays 0."""
    x, w = (3 * random(11, rows, n_in)).round().clamp(-3, 3), (2 * random(12, n_in, n_out)).round().clamp(-2, 2)
    x[0] = 0
    ex, ew = (60 * random(13, rows)).round().clamp(-126, 119), (60 * random(14, n_out)).round().clamp(-126, 119)
    ex[0], ex[1], ew[0], ew[1] = 119, -126, 119, -126
    want = (x.double() @ w.double()) * torch.exp2(ex.double())[:, None] * torch.exp2(ew.double())
    y = ops.dense(ops.Packed8(x.to(E4M3), torch.exp2(ex.double()).float()), ops.Packed8(w.to(E4M3), torch.exp2(ew.double()).float(), True), out_dtype=F32)
    assert torch.equal(y, want.float())


@pytest.mark.parametrize("rows,n_in,n_out", [(70, 64, 32), (300, 200, 700), (2500, 256, 512)])
def test_dense_takes_scales_that_are_no_powers_of_two(rows, n_in, n_out):
    x, scale = of_any_scale(rows, n_in)
    w = random(2, n_in, n_out).to(BF16)
    packed = ops.Packed8(x, scale)
    xv = x.double() * scale.double()[:, None]
    w8 = ops.pack8(w, by_column=True)
    sw = w8.scale * torch.exp(random(5, n_out))
    wv = w8.codes.double() * sw.double()
    near(ops.dense(packed, ops.Packed8(w8.codes, sw, True), out_dtype=F32), xv @ wv, (xv.abs() @ wv.abs()) * (n_in * 2.0 ** -23 + 2.0 ** -20))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("rows,n_in,n_out", [(5003, 2048, 1024), (16384, 512, 256), (2000, 512, 512), (700, 256, 2048), (60, 64, 48)])
def test_all_three_gradients_of_a_call_are_there_for_who_follows(rows, n_in, n_out, packed):
    """The bias's sums are joined while the products run, and those beside each other: copies right behind a call find what calls
    for one gradient each give, eagerly and in a graph, also when dz changes from call to call."""
    act = ACT_CRELU if packed else ACT_SCRELU
    w = random(21, n_in, n_out).to(BF16)
    x, y = random(22, rows, n_in).abs().clamp(max=1).to(BF16), random(23, rows, n_out).abs().clamp(max=1).to(BF16)
    if packed:
        x, y = ops.pack8(x, act=act), ops.pack8(y, act=act)
    dys = [random(24 + k, rows, n_out).to(BF16) for k in range(3)]
    needs = [dict(need_dx=k == 0, need_dw=k == 1, need_dbias=k == 2) for k in range(3)]
    want = [[ops.dense_backward(dy, x, w, y=y, act=act, **needs[k])[k] for k in range(3)] for dy in dys]

    def one(dy):
        got = ops.dense_backward(dy, x, w, y=y, act=act)
        copies = [t.clone() for t in got]
        for t in got:
            t.zero_()
        return copies

    for got in [[one(dy) for dy in dys] for _ in range(4)]:
        assert all(torch.equal(a, b) for g, v in zip(got, want) for a, b in zip(g, v))
    dy = dys[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = one(dy)
    for k in (1, 2, 0, 1):
        dy.copy_(dys[k])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))


def test_a_wait_that_gave_up_is_reported_once_by_the_next_dense_call():
    """The host sets the word that kernels would."""
    word = ctypes.POINTER(ctypes.c_int32)()
    _lib.check(_lib.load().b200_op_dense_gave_up(0, ctypes.byref(word)))
    few, many, w = random(31, 3, 64).to(BF16), random(32, 300, 64).to(BF16), random(33, 64, 48).to(BF16)
    dy = random(34, 300, 48).to(BF16)
    for call in (lambda: ops.dense(few, w), lambda: ops.dense(many, w), lambda: ops.dense_backward(dy, many, w), lambda: ops.dense_backward(dy, many, w, need_dw=False)):
        call()
        torch.cuda.synchronize()
        assert word[0] == 0
        word[0] = 1
        assert ops.dense(few[:0], w).shape == (0, 48)  # (no rows: nothing is asked)
        with pytest.raises(_lib.B200Error) as e:
            call()
        assert e.value.code == -2 and "not valid" in str(e.value) and word[0] == 0
        call()
    assert not ops.gave_up(0)
    word[0] = 1
    assert ops.gave_up(0) and not ops.gave_up(0)
    ops.dense(few, w)
    assert _lib.load().b200_op_dense_gave_up(0, None) == -1


def test_want_of_memory_is_torchs_error():
    """A result of 1 TB, which the allocator refuses at once: callers that catch torch's error go on with less."""
    x, w = torch.zeros(1 << 20, 16, device="cuda", dtype=BF16), torch.zeros(16, 1 << 19, device="cuda", dtype=BF16)
    with pytest.raises(torch.OutOfMemoryError):
        ops.dense(x, w)
    assert (ops.dense(x[:100], w[:, :64]) == 0).all()


@pytest.mark.parametrize("cols", [96, 777, 2048, 8192])
@pytest.mark.parametrize("kind,with_residual", [(F32, False), (F32, True), (BF16, True), (F16, False)])
def test_roundings_of_a_norms_product_move_no_code(cols, kind, with_residual):
    """Whole numbers, whose squares add up exactly, and weights that put every product next to a halfway point between two codes (normal
    ones): the code is that of total * rstd * weight before any rounding of the two products and of rstd."""
    rows, eps = 64, 2.0 ** -10
    g = torch.Generator(device="cuda")
    g.manual_seed(cols)
    sizes = torch.tensor([1.0, 2.0, 4.0, 8.0], device="cuda")[torch.randint(0, 4, (1, cols), device="cuda", generator=g)].expand(rows, cols)
    total = (sizes.gather(1, torch.rand(rows, cols, device="cuda", generator=g).argsort(1)) * (2 * torch.randint(0, 2, (rows, cols), device="cuda", generator=g) - 1)).double()
    rstd = 1 / torch.sqrt(total[0].square().mean() + eps)  # of every row: they are in another order only
    halfway = (8.5 + torch.randint(0, 8, (cols,), device="cuda", generator=g).double()) * torch.exp2(torch.randint(-2, 1, (cols,), device="cuda", generator=g).double())
    w = (halfway / rstd).float()
    r = torch.randint(-4, 5, (rows, cols), device="cuda", generator=g).to(kind) if with_residual else None
    x = (total if r is None else total - r.double()).to(kind)
    y, _, got_rstd = ops.rms_norm(x, w, residual=r, eps=eps, out_dtype=E4M3)
    assert torch.equal(got_rstd, rstd.float().expand(rows))
    want = total * rstd * w.double()
    code = want.abs() / y.scale.double()[:, None]  # at least 2^-6: normal codes
    step = torch.exp2(torch.floor(torch.log2(code)) - 3)
    assert (y.scale.double() >= want.abs().amax(1) / 448).all() and (y.scale.double() < want.abs().amax(1) / 224).all() and code.min() >= 2.0 ** -6
    clear = ((code / step).frac() - 0.5).abs() > 2.0 ** -45  # (where 64 bits tell on which side it lies)
    assert clear.float().mean() > 0.95
    nearest = torch.round(code / step) * step * want.sign()
    assert torch.equal(y.codes.double()[clear], nearest[clear])


FIRST_CALL = """
import sys
import torch
from bullet_b200 import ops
x, w = torch.ones(int(sys.argv[1]), 64, device="cuda").bfloat16(), torch.ones(64, 48, device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.dense(x, w)
graph.replay()
assert (y == 64).all()
"""


@pytest.mark.parametrize("rows", [3, 300])
def test_the_first_dense_call_of_a_process_may_be_captured(rows):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL, str(rows)], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


class Inside:
    """A matrix inside a larger buffer of `fill`: `at` elements behind its start, `pad` more elements a row."""

    def __init__(self, rows, cols, kind, at, pad, fill):
        self.raw = torch.full((at + rows * (cols + pad) + 64,), fill, device="cuda").to(kind)
        self.ld, self.address = cols + pad, self.raw.data_ptr() + at * self.raw.element_size()
        self.view = self.raw[at:at + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]

    @classmethod
    def of(cls, t, at, pad):
        m = cls(*t.shape, t.dtype, at, pad, float("nan"))
        m.view.copy_(t)
        return m

    def taken(self, fill):
        """Its values; everything around it has to be `fill`."""
        v = self.view.clone()
        self.view.fill_(fill)
        assert (self.raw == fill).all()
        return v


# Rows that start on 16 bytes and end inside 16, in and out, of one row and of more
@pytest.mark.parametrize("rows,n_in,n_out", [(1, 23, 7), (1, 2, 549), (9, 7, 1), (40, 23, 331), (300, 517, 23), (2000, 9, 70)])
@pytest.mark.parametrize("dw_kind", [F32, BF16])
def test_what_lies_behind_rows_that_end_inside_16_bytes(rows, n_in, n_out, dw_kind):
    def pad(cols, kind):  # to the next 16 bytes, and 16 more
        each = 8 if kind is BF16 else 4
        return -cols % each + each

    x, w = random(41, rows, n_in).mul(2).round().clamp(-3, 3).to(BF16), random(42, n_in, n_out).round().clamp(-2, 2).to(BF16)
    dy = random(43, rows, n_out).round().clamp(-1, 1).to(BF16)
    mx, mw, mdy = (Inside.of(t, 8, pad(t.shape[1], BF16)) for t in (x, w, dy))
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    code = {F32: 0, BF16: 1}

    def run(op, size, call):
        need = ctypes.c_int64()
        _lib.check(size(ctypes.byref(op), ctypes.byref(need)))
        space = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
        op.workspace, op.workspace_bytes = space.data_ptr(), need.value
        _lib.check(call(0, stream, ctypes.byref(op)))

    for kind in (F32, BF16):
        y = Inside(rows, n_out, kind, 8, pad(n_out, kind), 77.0)
        op = _lib.CDense(rows, n_in, n_out, 1, code[kind], 0, mx.ld, mw.ld, 0, y.ld, mx.address, None, mw.address, None, None, None, y.address)
        run(op, lib.b200_op_dense_workspace, lib.b200_op_dense)
        assert torch.equal(y.taken(77.0), (x.double() @ w.double()).to(kind))
    dx, dw = Inside(rows, n_in, BF16, 8, pad(n_in, BF16), 77.0), Inside(n_in, n_out, dw_kind, 8, pad(n_out, dw_kind), 77.0)
    db = torch.empty(n_out, device="cuda")
    op = _lib.CDenseGrad(rows, n_in, n_out, 1, 1, 1, code[dw_kind], 0, mdy.ld, mx.ld, 0, mw.ld, 0, dx.ld, dw.ld, mdy.address, mx.address, None, None, None, mw.address, None, dx.address,
                         dw.address, db.data_ptr())
    run(op, lib.b200_op_dense_backward_workspace, lib.b200_op_dense_backward)
    assert torch.equal(dx.taken(77.0), (dy.double() @ w.double().t()).to(BF16)) and torch.equal(dw.taken(77.0), (x.double().t() @ dy.double()).to(dw_kind))
    assert torch.equal(db.double(), dy.double().sum(0))
