"""The dense trunk's operators on the GPU against plain forms in 64 bits.

Tolerances.  A value rounded to a type with p significand bits is off by at most 2^-p of itself (24, 8 and 11 bits: fp32, bf16,
fp16).  A sum of k products in 32 bits is off by at most k 2^-23 of the sum of their magnitudes, in any order and whether a step
rounds or cuts off; products of small whole numbers are exact, and have to come out exactly.  A code of 8 bits is off by half a step of its
binade.  2^-18 covers the few roundings of elementwise arithmetic in 32 bits."""
import ctypes
import math

import pytest
import torch

from bullet_b200 import _lib, ops
from bullet_b200.configs import ACT_CRELU, ACT_NONE, ACT_RELU, ACT_SCRELU

pytestmark = pytest.mark.gpu
F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
ROUND = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}  # half a step below fp16's smallest normal number
FEW = 2.0 ** -18


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(seed, *shape):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def whole(seed, low, high, *shape, kind=BF16):
    return torch.randint(low, high + 1, shape, device="cuda", generator=gen(seed)).to(kind)


def spaced(t, pad, at=0):
    """The same matrix with `pad` more elements between rows, `at` elements into a buffer of NaN."""
    rows, cols = t.shape
    raw = t.new_empty(at + rows * (cols + pad), dtype=torch.float32).fill_(float("nan")).to(t.dtype)
    v = raw[at:].view(rows, cols + pad)[:, :cols]
    v.copy_(t)
    return v


def near(got, want, relative, absolute=0.0):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    off = (got - want).abs() - (relative * want.abs() + absolute)
    assert not torch.isnan(off).any() and off.max() <= 0 if off.numel() else True, float(off.max())


def exact_scale(v, dim):
    v = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).double()
    amax = v.amax(dim, keepdim=True)
    m, e = torch.frexp(amax / 448)  # (a logarithm may be off by its last bit where this is a power of two)
    k = torch.where(m == 0.5, e - 1, e).clamp(min=-126).double()
    return torch.where(amax > 0, torch.exp2(k), torch.ones_like(amax))


def half_step(v, scale):
    """Half the distance of the codes around v."""
    return torch.exp2(torch.floor(torch.log2((v.abs() / scale).clamp(min=2.0 ** -6))) - 4) * scale


# ------------------------------------------------------------------------------------------------- norm
NORMS = [(1, 2048, BF16, BF16, True), (3, 1, F32, F32, False), (2, 7, F16, BF16, True), (5, 200, F32, E4M3, False), (33, 520, BF16, E4M3, True),
         (129, 768, F16, F16, False), (17, 1000, BF16, F32, True), (7, 333, BF16, E4M3, True), (4, 4100, F32, BF16, True), (3, 8192, BF16, E4M3, True),
         (2, 20000, BF16, E4M3, True), (2, 40001, F32, F32, True), (300, 64, BF16, BF16, True), (1000, 96, F32, E4M3, True), (5, 16, BF16, E4M3, False)]


@pytest.mark.parametrize("rows,cols,kind,out,with_residual", NORMS)
@pytest.mark.parametrize("pad,at", [(0, 0), (8, 0), (3, 1)])
def test_norm(rows, cols, kind, out, with_residual, pad, at):
    spread = torch.exp(normal(1, cols))
    x = spaced((normal(2, rows, cols) * spread).to(kind), pad, at)
    r = spaced((normal(3, rows, cols) * spread).to(kind), pad, at) if with_residual else None
    w = 1 + 0.3 * normal(4, cols)
    y, total, rstd = ops.rms_norm(x, w, residual=r, eps=1e-5, out_dtype=out)
    t = x.double() + (r.double() if with_residual else 0)
    s = 1 / torch.sqrt(t.square().mean(1) + 1e-5)
    sums = cols * 2.0 ** -23
    near(rstd, s, FEW + sums)
    if with_residual:
        near(total, t, ROUND[kind], TINY[kind])
    else:
        assert total is x
    want = t * s[:, None] * w.double()
    if out is E4M3:
        scale = exact_scale(want, 1)
        assert (y.scale.double() == scale[:, 0]).all()
        near(ops.unpack8(y, F32), want, FEW + sums, (half_step(want, scale) * (1 + FEW)))
    else:
        near(y, want, ROUND[out] + FEW + sums, TINY[out])
    again = ops.rms_norm(x, w, residual=r, eps=1e-5, out_dtype=out)[0]
    assert torch.equal(y.codes.view(torch.uint8), again.codes.view(torch.uint8)) if out is E4M3 else torch.equal(y, again)


def test_norm_without_weight_is_that_of_ones():
    x = normal(5, 9, 260).to(BF16)
    assert torch.equal(ops.rms_norm(x)[0], ops.rms_norm(x, torch.ones(260, device="cuda"))[0])


@pytest.mark.parametrize("cols", [96, 2048, 2049, 20000])
@pytest.mark.parametrize("out", [F32, E4M3])
def test_norm_of_rows_of_zeros_and_of_what_is_not_finite(cols, out):
    x = normal(6, 6, cols)
    x[1] = 0
    x[2, cols // 2] = float("nan")
    x[3, 5] = float("inf")
    x[4] = 1e19  # its square is past fp32
    y, _, rstd = ops.rms_norm(x, out_dtype=out)
    v = ops.unpack8(y, F32) if out is E4M3 else y
    clean = ops.rms_norm(x[[0, 5]].contiguous(), out_dtype=out)[0]
    assert torch.equal(v[[0, 5]], ops.unpack8(clean, F32) if out is E4M3 else clean)
    assert (v[1] == 0).all() and torch.isnan(v[2]).all() and rstd[4] == 0 and (v[4] == 0).all()
    assert rstd[3] == 0 and torch.isnan(v[3, 5]) and (v[3, :5] == 0).all() and (v[3, 6:] == 0).all()
    if out is E4M3:
        assert (y.scale[1:5] == 1).all()


NORM_GRADS = [(1, 2048, BF16, BF16, True), (3, 1, F32, F32, False), (5003, 40, BF16, BF16, True), (40, 520, F32, BF16, False), (65, 333, F16, F32, True),
              (257, 768, BF16, BF16, False), (3, 8192, BF16, BF16, True), (2, 20001, F32, F32, True), (700, 1024, F32, BF16, True)]


def norm_of(x, w, eps=1e-5):
    return x / torch.sqrt(x.square().mean(1, keepdim=True) + eps) * w


@pytest.mark.parametrize("rows,cols,kind,dkind,through", NORM_GRADS)
@pytest.mark.parametrize("pad,at", [(0, 0), (3, 1)])
def test_norm_gradient(rows, cols, kind, dkind, through, pad, at):
    total = spaced(normal(11, rows, cols).to(kind), pad, at)
    dy = spaced(normal(12, rows, cols).to(dkind), pad, at)
    ds = spaced(normal(13, rows, cols).to(kind), pad, at) if through else None
    w = 1 + 0.3 * normal(14, cols)
    t = total.double().requires_grad_()
    v = w.double().requires_grad_()
    dx_want, dw_want = torch.autograd.grad((norm_of(t, v) * dy.double()).sum(), (t, v))
    rstd = (1 / torch.sqrt(total.double().square().mean(1) + 1e-5)).float()
    dx, dw = ops.rms_norm_backward(dy, total, rstd, w, dtotal=ds)
    # the two terms of dx and the mean's sum bound its roundings
    size = rstd.double()[:, None] * ((dy.double() * w.double()).abs() + (total.double() * rstd.double()[:, None]).abs()
                                     * (dy.double() * w.double() * total.double() * rstd.double()[:, None]).abs().mean(1, keepdim=True))
    if through:
        dx_want = dx_want + ds.double()
        size = size + ds.double().abs()
    near(dx, dx_want, ROUND[kind], TINY[kind] + size * (FEW + cols * 2.0 ** -23))
    near(dw, dw_want, 0, (dy.double() * total.double() * rstd.double()[:, None]).abs().sum(0) * (rows * 2.0 ** -23 + FEW))
    only_dx, none = ops.rms_norm_backward(dy, total, rstd, None, dtotal=ds)
    assert none is None and only_dx.shape == dx.shape
    again = ops.rms_norm_backward(dy, total, rstd, w, dtotal=ds)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def test_norm_gradient_against_differences():
    x, dy, w = normal(21, 7, 96), normal(22, 7, 96), 1 + 0.3 * normal(23, 96)
    vx, vw, h = normal(24, 7, 96).double(), normal(25, 96).double(), 1e-5

    def loss(t):
        return (norm_of(x.double() + t * vx, w.double() + t * vw) * dy.double()).sum()

    _, total, rstd = ops.rms_norm(x, w)
    dx, dw = ops.rms_norm_backward(dy, total, rstd, w)
    slope = float(loss(h) - loss(-h)) / (2 * h)
    mine = float((dx.double() * vx).sum() + (dw.double() * vw).sum())
    # the differences' own error is of the order of h^2 and 2^-52 / h, the gradient's the roundings of some thousand terms
    size = float((dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum())
    assert abs(mine - slope) <= size * (FEW + 1e-8)


# --------------------------------------------------------------------------------------------- 8 bits
PACKS = [(1, 1, F32), (1, 2048, BF16), (7, 200, F32), (33, 333, BF16), (129, 768, F16), (4, 8192, F32), (2, 20001, BF16), (1000, 48, BF16), (513, 64, F32)]


@pytest.mark.parametrize("rows,cols,kind", PACKS)
@pytest.mark.parametrize("act", [ACT_NONE, ACT_CRELU, ACT_SCRELU, ACT_RELU])
@pytest.mark.parametrize("by_column", [False, True])
@pytest.mark.parametrize("pad,at", [(0, 0), (3, 1)])
def test_pack(rows, cols, kind, act, by_column, pad, at):
    x = normal(31, rows, cols) * torch.exp(2 * normal(32, 1, cols))
    if act in (ACT_CRELU, ACT_SCRELU):
        x = (0.5 + 0.5 * x).clamp(0, 1)
        x[0, 0] = 0.999
        x[rows - 1, cols - 1] = 1e-6
    elif act == ACT_RELU:
        x = x.clamp(min=0)
    x = spaced(x.to(kind), pad, at)
    p = ops.pack8(x, act=act, by_column=by_column)
    v = x.double()
    scale = exact_scale(v, 0 if by_column else 1)
    assert (p.scale.double() == scale.flatten()).all()
    got = ops.unpack8(p, F32)
    off = half_step(v, scale)
    if act != ACT_NONE:  # one more step where a code was kept from 0 or 1
        off = off * torch.where((v > 0) & ((v < 2 ** -9 * scale) | (v > 0.9)), 2.0, 1.0)
        inside = (v > 0) if act == ACT_RELU else (v > 0) & (v < 1)
        g = got.double()
        assert (inside == ((g > 0) if act == ACT_RELU else (g > 0) & (g < 1))).all()
    near(got, v, 0, off)
    for kind_out in (BF16, F16):
        if kind_out is BF16:
            assert (ops.unpack8(p, BF16).double() == got.double()).all()
        else:
            near(ops.unpack8(p, F16), got, ROUND[F16], TINY[F16])


def test_pack_agrees_with_the_nearest_code_on_every_halfway_point():
    codes = torch.arange(127, device="cuda", dtype=torch.uint8).view(E4M3).float()
    x = torch.cat([codes, (codes[:-1] + codes[1:]) / 2])
    x = torch.cat([x, -x])[None].contiguous()
    p = ops.pack8(x)
    assert p.scale.item() == 1 and torch.equal(p.codes.float(), x.to(E4M3).float())
    assert torch.equal(ops.unpack8(p, F32), p.codes.float())


@pytest.mark.parametrize("cols", [96, 333, 20000])
@pytest.mark.parametrize("by_column", [False, True])
def test_pack_of_extremes(cols, by_column):
    x = normal(33, 7, cols)
    x[1] = 0
    x[2, 3] = float("nan")
    x[3, 4] = float("-inf")
    x[4] = 3e38
    x[5] = 1e-40
    x[6] = float("nan")
    if by_column:
        x = x.t().contiguous()
    p = ops.pack8(x, by_column=by_column)
    got, scale = ops.unpack8(p, F32), p.scale
    if by_column:
        got, x = got.t(), x.t()
    assert (scale.double() == exact_scale(x.double(), 1)[:, 0]).all()
    assert (torch.isnan(got) == ~torch.isfinite(x)).all()
    assert (got[1] == 0).all() and scale[1] == 1 and scale[6] == 1 and torch.isfinite(got[4]).all() and scale[5] == 2.0 ** -126
    fine = torch.isfinite(x)
    v = torch.where(fine, x, torch.zeros_like(x)).double()
    near(torch.where(fine, got, torch.zeros_like(got)), v, 0, half_step(v, exact_scale(x.double(), 1)))


# ---------------------------------------------------------------------------------------------- dense
def act_of(z, act):
    z = z if act == ACT_NONE else z.clamp(min=0) if act == ACT_RELU else z.clamp(0, 1)
    return z * z if act == ACT_SCRELU else z


SHAPES = [(1, 64, 64), (1, 2048, 1024), (3, 40, 24), (8, 1024, 512), (9, 96, 200), (17, 2048, 16), (64, 72, 2048), (127, 128, 128), (128, 64, 256), (129, 200, 136),
          (200, 1000, 264), (513, 512, 768), (1000, 336, 1032), (77, 33, 65), (130, 7, 3), (5, 777, 1), (260, 1, 9), (300, 130, 1858), (2, 4096, 4096), (4096, 16, 16)]


@pytest.mark.parametrize("rows,n_in,n_out", SHAPES)
@pytest.mark.parametrize("kind", [BF16, F16, E4M3])
def test_dense_of_whole_numbers_is_exact(rows, n_in, n_out, kind):
    x, w = whole(41, -3, 3, rows, n_in, kind=kind), whole(42, -2, 2, n_in, n_out, kind=kind)
    b, r = whole(43, -9, 9, n_out, kind=F32), whole(44, -9, 9, rows, n_out, kind=F32)
    want = x.double() @ w.double()
    if kind is E4M3:
        sx, sw = torch.exp2(whole(45, -4, 3, rows, kind=F32)), torch.exp2(whole(46, -3, 4, n_out, kind=F32))
        want = want * sx.double()[:, None] * sw.double()
        x, w = ops.Packed8(x, sx), ops.Packed8(w, sw, True)
    y = ops.dense(x, w, bias=b, residual=r, out_dtype=F32)
    assert torch.equal(y.double(), want + b.double() + r.double())
    assert torch.equal(ops.dense(x, w, out_dtype=F32).double(), want)


@pytest.mark.parametrize("rows,n_in,n_out", [(1, 512, 256), (6, 96, 40), (130, 1024, 264), (700, 2048, 512), (65, 77, 33)])
@pytest.mark.parametrize("kind,out", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, BF16), (E4M3, BF16), (E4M3, F32), (E4M3, F16)])
@pytest.mark.parametrize("act", [ACT_NONE, ACT_CRELU, ACT_SCRELU, ACT_RELU])
def test_dense(rows, n_in, n_out, kind, out, act):
    x, w = normal(51, rows, n_in), normal(52, n_in, n_out) * n_in ** -0.5
    if kind is E4M3:
        x, w = ops.pack8(x), ops.pack8(w, by_column=True)
        xv, wv = ops.unpack8(x, F32).double(), ops.unpack8(w, F32).double()
    else:
        x, w = x.to(kind), w.to(kind)
        xv, wv = x.double(), w.double()
    b, r = normal(53, n_out), normal(54, rows, n_out).to(out)
    z = xv @ wv + b.double()
    sums = (xv.abs() @ wv.abs() + b.double().abs()) * (n_in * 2.0 ** -23 + FEW)
    for residual in (None, r):
        want = act_of(z, act) + (0 if residual is None else residual.double())
        near(ops.dense(x, w, bias=b, act=act, residual=residual, out_dtype=out), want, ROUND[out], 2 * sums + TINY[out])


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("pads", [(8, 16, 8, 0), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 5, 0), (3, 5, 7, 1), (16, 16, 16, 3), (0, 0, 0, 1)])
@pytest.mark.parametrize("rows,n_in,n_out", [(1, 128, 64), (7, 64, 48), (150, 96, 272)])
def test_dense_of_matrices_inside_larger_ones(rows, n_in, n_out, kind, pads):
    """Any distance of rows and any first element, in and out; nothing around the output is touched."""
    x, w = whole(61, -3, 3, rows, n_in, kind=kind), whole(62, -2, 2, n_in, n_out, kind=kind)
    r = whole(63, -9, 9, rows, n_out, kind=BF16)
    want = x.double() @ w.double() + r.double()
    px, pw, pr, at = pads
    holder = torch.full((at + rows * (n_out + pr) + 64,), 77.0, device="cuda", dtype=BF16)
    y = holder[at:at + rows * (n_out + pr)].view(rows, n_out + pr)
    x, w, r = spaced(x, px, at), spaced(w, pw, at), spaced(r, pr, at)
    one = torch.ones(max(rows, n_out), device="cuda")
    codes = kind is E4M3
    op = _lib.CDense(rows, n_in, n_out, 3 if codes else 1, 1, 0, n_in + px, n_out + pw, n_out + pr, n_out + pr, x.data_ptr(), one.data_ptr() if codes else None,
                     w.data_ptr(), one.data_ptr() if codes else None, None, r.data_ptr(), y.data_ptr())
    lib, need = _lib.load(), ctypes.c_int64()
    _lib.check(lib.b200_op_dense_workspace(ctypes.byref(op), ctypes.byref(need)))
    space = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")[at % 2 * 16:]  # (aligned to 16 bytes and no more)
    op.workspace, op.workspace_bytes = space.data_ptr(), need.value
    _lib.check(lib.b200_op_dense(0, torch.cuda.current_stream().cuda_stream, ctypes.byref(op)))
    assert torch.equal(y[:, :n_out].double(), want.to(BF16).double())
    assert (y[:, n_out:] == 77).all() and (holder[:at] == 77).all() and (holder[at + rows * (n_out + pr):] == 77).all()


@pytest.mark.parametrize("rows", [3, 200])
def test_dense_keeps_what_is_not_finite_where_it_belongs(rows):
    x, w = whole(64, -3, 3, rows, 128), whole(65, -2, 2, 128, 72)
    b = torch.zeros(72, device="cuda")
    x[1, 7], b[5] = float("nan"), float("inf")
    for act in (ACT_NONE, ACT_RELU, ACT_CRELU):
        y = ops.dense(x, w, bias=b, act=act, out_dtype=F32)
        assert torch.isnan(y[1]).all() and torch.isfinite(y[torch.arange(rows) != 1][:, torch.arange(72) != 5]).all()
        assert (y[torch.arange(rows) != 1][:, 5] == (1.0 if act == ACT_CRELU else float("inf"))).all()


GRADS = [(1, 64, 64), (3, 40, 24), (9, 96, 200), (64, 128, 256), (129, 200, 136), (513, 512, 768), (1000, 336, 64), (77, 33, 65), (130, 7, 3), (5003, 128, 128), (70000, 32, 48),
         (6000, 16, 2048)]


@pytest.mark.parametrize("rows,n_in,n_out", GRADS)
@pytest.mark.parametrize("kind,codes,dw_kind", [(BF16, False, F32), (F16, False, F32), (BF16, True, F32), (BF16, False, BF16)])
def test_dense_gradient_of_whole_numbers_is_exact(rows, n_in, n_out, kind, codes, dw_kind):
    dy, w = whole(71, -1, 1, rows, n_out, kind=kind), whole(72, -2, 2, n_in, n_out, kind=kind)
    x, y = whole(73, -3, 3, rows, n_in, kind=F32), whole(74, 0, 4, rows, n_out, kind=F32) / 4
    skip = whole(75, -9, 9, rows, n_in, kind=kind)
    dz = torch.where((y > 0) & (y < 1), dy.float(), torch.zeros_like(y)).double()
    xs = x.double()
    if codes:
        sx, sy = torch.exp2(whole(76, -2, 1, rows, kind=F32)), torch.exp2(whole(77, -2, 4, rows, kind=F32))
        xs = xs * sx.double()[:, None]
        x, y = ops.Packed8(x.to(E4M3), sx), ops.Packed8((y / sy[:, None]).to(E4M3), sy)
    else:
        x, y = x.to(kind), y.to(kind)
    dx, dw, db = ops.dense_backward(dy, x, w, y=y, act=ACT_CRELU, dskip=skip, dw_dtype=dw_kind)
    assert torch.equal(dx.double(), (dz @ w.double().t() + skip.double()).to(kind).double())
    assert torch.equal(dw.double(), (xs.t() @ dz).to(dw_kind).double())
    assert torch.equal(db.double(), dz.sum(0))
    dx, dw, db = ops.dense_backward(dy, x, w, need_dw=False)
    assert dw is None and torch.equal(dx.double(), (dy.double() @ w.double().t()).to(kind).double()) and torch.equal(db.double(), dy.double().sum(0))
    dx, dw, db = ops.dense_backward(dy, x, w, need_dx=False, need_dbias=False)
    assert dx is None and db is None and torch.equal(dw.double(), xs.t() @ dy.double())


@pytest.mark.parametrize("rows,n_in,n_out", [(6, 96, 40), (300, 264, 136), (1500, 512, 256), (65, 77, 33)])
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("act", [ACT_NONE, ACT_CRELU, ACT_SCRELU, ACT_RELU])
def test_dense_gradient(rows, n_in, n_out, codes, act):
    x, y = normal(81, rows, n_in), act_of(0.4 + 0.5 * normal(82, rows, n_out), act)
    w, dy = (normal(83, n_in, n_out) * n_in ** -0.5).to(BF16), normal(84, rows, n_out).to(BF16)
    if codes:
        x, y = ops.pack8(x), ops.pack8(y, act=act)
        xv, yv = ops.unpack8(x, F32).double(), ops.unpack8(y, F32).double()
    else:
        x, y = x.to(BF16), y.to(BF16)
        xv, yv = x.double(), y.double()
    dz = dy.double() * (2 * yv.clamp(min=0).sqrt() if act == ACT_SCRELU else 1)
    inside = torch.ones_like(yv, dtype=torch.bool) if act == ACT_NONE else yv > 0 if act == ACT_RELU else (yv > 0) & (yv < 1)
    dz = torch.where(inside, dz, torch.zeros_like(dz))
    dx, dw, db = ops.dense_backward(dy, x, w, y=y, act=act)
    rounded = ROUND[BF16] if act == ACT_SCRELU else 0.0
    near(dx, dz @ w.double().t(), ROUND[BF16], (dz.abs() @ w.double().abs().t()) * (n_out * 2.0 ** -23 + FEW + 2 * rounded))
    near(dw, xv.t() @ dz, 0, (xv.abs().t() @ dz.abs()) * (rows * 2.0 ** -23 + FEW + rounded))
    near(db, dz.sum(0), 0, dz.abs().sum(0) * (rows * 2.0 ** -23 + FEW))


@pytest.mark.parametrize("codes", [False, True])
def test_long_sums_keep_their_bits(codes):
    """Sums over many rows, of one sign and of both: the pipe that multiplies cuts off what it adds, so they are taken out on the way.
    Bound: the 4 x 128 additions between two takings-out cut off less than 2^-23 of the magnitudes' sum each, and adding up what
    was taken out rounds at most 64 times.  (Without, 32768 additions: 2^-8.)"""
    rows, n_in, n_out = 131072, 256, 64
    x = torch.rand(rows, n_in, device="cuda", generator=gen(87))
    dy = torch.cat([torch.rand(rows, 32, device="cuda", generator=gen(88)), normal(89, rows, 32)], 1).to(BF16)
    x = ops.pack8(x) if codes else x.to(BF16)
    xv = (ops.unpack8(x, F32) if codes else x).double()
    _, dw, _ = ops.dense_backward(dy, x, None, need_dx=False, need_dbias=False)
    near(dw, xv.t() @ dy.double(), 0, (4 * 128 + 64) * 2.0 ** -23 * (xv.abs().t() @ dy.double().abs()))


@pytest.mark.parametrize("rows,n_in,n_out", [(30, 20000, 72), (700, 16392, 520)])
def test_dense_of_many_inputs(rows, n_in, n_out):
    x, w = whole(85, -2, 2, rows, n_in), whole(86, -2, 2, n_in, n_out)
    r = whole(87, -9, 9, rows, n_out, kind=F32)
    assert torch.equal(ops.dense(x, w, residual=r, out_dtype=F32).double(), x.double() @ w.double() + r.double())


def test_dense_gradient_against_differences():
    rows, n_in, n_out, h = 40, 64, 48, 1e-6
    x, w = normal(91, rows, n_in).to(BF16), (normal(92, n_in, n_out) * n_in ** -0.5).to(BF16)
    b, dy = 0.5 + 0.1 * normal(93, n_out), normal(94, rows, n_out).to(BF16)
    vx, vw, vb = normal(95, rows, n_in).double(), normal(96, n_in, n_out).double(), normal(97, n_out).double()
    for act in (ACT_NONE, ACT_CRELU, ACT_RELU):
        def loss(t):
            return (act_of((x.double() + t * vx) @ (w.double() + t * vw) + b.double() + t * vb, act) * dy.double()).sum()

        y = ops.dense(x, w, bias=b, act=act)
        dx, dw, db = ops.dense_backward(dy, x, w, y=y, act=act)
        slope = float(loss(h) - loss(-h)) / (2 * h)
        parts = [(dx.double() * vx), (dw.double() * vw), (db.double() * vb)]
        mine = float(sum(p.sum() for p in parts))
        # dx is rounded to 8 bits, the rest to 24.  An output within 2^-9 of 1 rounds to 1, where the gradient is cut off: such
        # outputs are taken out of the loss by their dy
        near_one = (act_of(x.double() @ w.double() + b.double(), act) - 1).abs() < 2.0 ** -8
        if act == ACT_CRELU and bool(near_one.any()):
            dy = torch.where(near_one, torch.zeros_like(dy), dy)
            dx, dw, db = ops.dense_backward(dy, x, w, y=y, act=act)
            slope = float(loss(h) - loss(-h)) / (2 * h)
            parts = [(dx.double() * vx), (dw.double() * vw), (db.double() * vb)]
            mine = float(sum(p.sum() for p in parts))
        size = float(sum(p.abs().sum() for p in parts))
        assert abs(mine - slope) <= float(parts[0].abs().sum()) * ROUND[BF16] + size * (FEW + n_in * 2.0 ** -23) + 1e-6 * size


@pytest.mark.parametrize("rows,n_in,n_out", [(70, 64, 32), (300, 200, 700), (2500, 256, 512), (700, 130, 64)])
def test_checkpoints_of_any_scale_and_with_nan(rows, n_in, n_out):
    """Scales from 2^-126 to 2^119, and codes that are NaN: each reaches the gradient rows that it belongs to."""
    x, dy = whole(121, -3, 3, rows, n_in, kind=E4M3), torch.zeros(rows, n_out, device="cuda", dtype=BF16)
    e = torch.zeros(rows, device="cuda")
    e[3], e[5], e[rows - 1], e[7], e[9] = 8, 30, 119, -126, 7
    scale = torch.exp2(e)
    for k, row in enumerate((3, 5, rows - 1, 7, 9)):  # a row of dy each, in columns of their own
        dy[row, k] = 1
    _, dw, _ = ops.dense_backward(dy, ops.Packed8(x, scale), None, need_dx=False)
    assert torch.equal(dw.double(), (x.double() * scale.double()[:, None]).t() @ dy.double())
    codes = x.view(torch.uint8).clone()
    codes[5, 11], codes[rows - 1, n_in - 1] = 0x7F, 0xFF
    _, dw, _ = ops.dense_backward(dy, ops.Packed8(codes.view(E4M3), scale), None, need_dx=False)
    nan = torch.zeros(n_in, dtype=torch.bool, device="cuda")
    nan[11] = nan[n_in - 1] = True
    assert torch.isnan(dw[nan]).all() and torch.isfinite(dw[~nan]).all()
    want = (x.double() * scale.double()[:, None]).t() @ dy.double()
    assert torch.equal(dw[~nan].double(), want[~nan])


def test_pack_of_what_would_round_out_of_range():
    top = torch.tensor([[3.38e38, -3.38e38, 1.0], [2.0 ** 127, -(2.0 ** 127), 0.0]], device="cuda")
    for kind in (F32, BF16):
        for by_column in (False, True):
            p = ops.pack8(top.to(kind), by_column=by_column)
            v = ops.unpack8(p, F32)
            assert torch.isfinite(v).all() and (v[0, :2].abs() >= 2.0 ** 127 * 1.8).all() and torch.equal(v[1, :2], top[1, :2])


def test_gradient_is_cut_off_whatever_comes_in():
    dy = torch.full((4, 16), float("inf"), device="cuda", dtype=BF16)
    y = torch.zeros(4, 16, device="cuda", dtype=BF16)
    y[:, 8:] = 1
    dx, dw, db = ops.dense_backward(dy, torch.ones(4, 8, device="cuda", dtype=BF16), torch.ones(8, 16, device="cuda", dtype=BF16), y=y, act=ACT_CRELU)
    assert (dx == 0).all() and (dw == 0).all() and (db == 0).all()


# -------------------------------------------------------------------------------------------- any call
def test_no_rows():
    e = torch.empty(0, 32, device="cuda", dtype=BF16)
    w = torch.ones(32, 16, device="cuda", dtype=BF16)
    assert ops.rms_norm(e, residual=e, out_dtype=E4M3)[0].codes.shape == (0, 32)
    assert ops.dense(e, w).shape == (0, 16)
    assert (ops.pack8(e, by_column=True).scale == 1).all() and ops.unpack8(ops.pack8(e)).shape == (0, 32)
    dx, dw, db = ops.dense_backward(torch.empty(0, 16, device="cuda", dtype=BF16), e, w)
    assert dx.shape == (0, 32) and (dw == 0).all() and (db == 0).all()
    dx, dw = ops.rms_norm_backward(e, e, torch.empty(0, device="cuda"), torch.ones(32, device="cuda"))
    assert dx.shape == (0, 32) and (dw == 0).all()


def block(x, r, w1, w2, norm_w, b1):
    y, total, rstd = ops.rms_norm(x, norm_w, residual=r, out_dtype=E4M3)
    h = ops.dense(ops.unpack8(y), w1, bias=b1, act=ACT_SCRELU)
    h8 = ops.pack8(h, act=ACT_SCRELU)
    z = ops.dense(h, w2, residual=total)
    dh, dw2, _ = ops.dense_backward(z, h8, w2)
    dn, dw1, db1 = ops.dense_backward(dh, y, w1, y=h8, act=ACT_SCRELU)
    dx, dweight = ops.rms_norm_backward(dn, total, rstd, norm_w, dtotal=z)
    return z, dw2, dw1, db1, dx, dweight


@pytest.mark.parametrize("rows", [5, 700])
def test_calls_run_on_the_current_stream_and_in_graphs(rows):
    args = (normal(101, rows, 128).to(BF16), normal(102, rows, 128).to(BF16), normal(103, 128, 256).to(BF16), normal(104, 256, 128).to(BF16),
            1 + 0.1 * normal(105, 128), normal(106, 256))
    want = block(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = block(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block(*args)
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("rows,cols,out", [(5003, 2048, 1024), (16384, 512, 256), (700, 256, 2048)])
def test_gradients_of_one_call_are_those_of_two_and_all_there_for_who_follows(rows, cols, out, packed):
    """The two products of a call may run beside each other: a copy right behind the call has to find both results."""
    dy, w = normal(401, rows, out).to(BF16), normal(402, cols, out).to(BF16)
    x, y = torch.rand(rows, cols, device="cuda", generator=gen(403)).to(BF16), torch.rand(rows, out, device="cuda", generator=gen(404)).to(BF16)
    act = ACT_CRELU if packed else ACT_SCRELU
    if packed:
        x, y = ops.pack8(x, act=act), ops.pack8(y, act=act)
    dx = ops.dense_backward(dy, x, w, y=y, act=act, need_dw=False)[0]
    dw = ops.dense_backward(dy, x, w, y=y, act=act, need_dx=False)[1]

    def both():
        got = ops.dense_backward(dy, x, w, y=y, act=act)[:2]
        copies = [t.clone() for t in got]
        for t in got:
            t.zero_()
        return copies

    for got in [both() for _ in range(5)]:
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    for _ in range(3):
        graph.replay()
        assert torch.equal(captured[0], dx) and torch.equal(captured[1], dw)


def test_long_matrices_pass_32_bit_offsets():
    """More than 2^31 elements: the last rows are those of the plain forms, by the bounds of the tests above."""
    rows, cols, n = (1 << 20) + 37, 2056, 40
    sums = cols * 2.0 ** -23 + FEW
    x = torch.zeros(rows, cols, device="cuda", dtype=BF16)
    x[-n:] = normal(111, n, cols).to(BF16)
    tail = x[-n:].double()
    w = normal(112, cols, 16).to(BF16)
    near(ops.dense(x, w)[-n:], tail @ w.double(), ROUND[BF16], 2 * sums * (tail.abs() @ w.double().abs()))
    y, _, rstd = ops.rms_norm(x, out_dtype=E4M3)
    s = 1 / torch.sqrt(tail.square().mean(1) + 1e-5)
    near(rstd[-n:], s, sums)
    want, last = tail * s[:, None], ops.Packed8(y.codes[-n:], y.scale[-n:])
    near(ops.unpack8(y, F32)[-n:], want, sums, half_step(want, exact_scale(want, 1)) * (1 + FEW))
    assert (last.scale.double() == exact_scale(want, 1)[:, 0]).all()
    del y, last
    p = ops.pack8(x)
    near(ops.unpack8(p)[-n:], tail, 0, half_step(tail, exact_scale(tail, 1)))
    dy = torch.zeros(rows, 16, device="cuda", dtype=BF16)
    dy[-n:] = whole(113, -1, 1, n, 16)
    g, xv = dy[-n:].double(), ops.unpack8(p)[-n:].double()
    dx, dw, db = ops.dense_backward(dy, p, w)
    near(dx[-n:], g @ w.double().t(), ROUND[BF16], (g.abs() @ w.double().abs().t()) * (16 * 2.0 ** -23 + FEW))
    near(dw, xv.t() @ g, 0, (xv.abs().t() @ g.abs()) * (n * 2.0 ** -23 + FEW))
    assert torch.equal(db.double(), g.sum(0))
    del dx, p, dy
    dn = torch.zeros_like(x)
    dn[-n:] = normal(114, n, cols).to(BF16)
    g = dn[-n:].double()
    dx, dweight = ops.rms_norm_backward(dn, x, torch.ones(rows, device="cuda"), torch.ones(cols, device="cuda"))
    mean = (g * tail).mean(1, keepdim=True)
    near(dx[-n:], g - tail * mean, ROUND[BF16], (g.abs() + tail.abs() * (g * tail).abs().mean(1, keepdim=True)) * sums)
    near(dweight, (g * tail).sum(0), 0, (g * tail).abs().sum(0) * (n * 2.0 ** -23 + FEW))


def test_the_threads_device_stays(monkeypatch):
    before = torch.cuda.current_device()
    ops.rms_norm(normal(121, 3, 32))
    assert torch.cuda.current_device() == before


def test_refusals_of_tensors():
    x, w = normal(131, 4, 32).to(BF16), normal(132, 32, 16).to(BF16)
    for call in (lambda: ops.rms_norm(x.t()), lambda: ops.rms_norm(x, weight=torch.ones(31, device="cuda")), lambda: ops.rms_norm(x, residual=x[:3]),
                 lambda: ops.rms_norm(x, residual=x.float()), lambda: ops.dense(x, w.to(F16)), lambda: ops.dense(x, w.t()), lambda: ops.dense(x, w[:31]),
                 lambda: ops.dense(ops.pack8(x), ops.pack8(w)), lambda: ops.dense(x, w, act=7), lambda: ops.dense(x, w, residual=x),
                 lambda: ops.dense_backward(x, x, w), lambda: ops.dense_backward(normal(1, 4, 16).to(BF16), x, w, act=ACT_RELU),
                 lambda: ops.dense_backward(normal(1, 4, 16), x.float(), w.float()), lambda: ops.unpack8(ops.pack8(x), torch.int8),
                 lambda: ops.dense_backward(normal(1, 4, 16).to(BF16), x, w, dw_dtype=F16), lambda: ops.rms_norm_backward(x, x, torch.ones(5, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.B200Error):
        ops.dense_backward(normal(1, 4, 16).to(F16), ops.pack8(x), w.to(F16))
    assert math.isfinite(float(ops.dense(x, w).float().sum()))


def test_the_example_trains():
    """The trunk of examples/residual_trunk.py behind the feature transformer: its output is that of the same network in 64 bits but for
    the roundings to 8 bits, its gradients are those of the same formulas in 64 bits from the activations that it kept, but for the
    roundings of passed-on gradients to bf16, and the loss falls."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "residual_trunk.py")
    spec = importlib.util.spec_from_file_location("residual_trunk", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    trunk = example.Trunk(128, 64, 96, 2)
    x, dout = normal(141, 300, 128).clamp(min=0), normal(142, 300, 1).to(BF16)
    out, kept = trunk.forward(x)
    dx = trunk.backward(dout, kept)
    w = {k: v.double() for k, v in trunk.w.value.items()}
    stream = norm_of(x.double(), w["norm_in"]) @ w["in"]
    for k in range(2):
        h = (norm_of(stream, w[f"norm{k}"]) @ w[f"up{k}"] + w[f"bias_up{k}"]).clamp(0, 1)
        stream = stream + h @ w[f"down{k}"] + w[f"bias_down{k}"]
    want = norm_of(stream, w["norm_out"]) @ w["out"] + w["bias_out"]

    def off(a, b):
        return float((a.double() - b).norm() / b.norm())

    # nearest codes of four bits are off by 2^-5.8 in the mean square at most: of a norm's output and a weight, twice, behind which
    # the stream's own part dilutes them
    assert off(out, want) < 0.1

    def norm_back(dn, stream, rstd, weight):
        t, g = stream.double().requires_grad_(), weight.clone().requires_grad_()
        return torch.autograd.grad((norm_of(t, g) * dn).sum(), (t, g))

    b = {k: v.double() for k, v in trunk.w.bf16.items()}
    values = [[ops.unpack8(t, F32).double() if isinstance(t, ops.Packed8) else t.double() for t in step] for step in kept]
    grads, d = {}, dout.double()
    n, stream, rstd = values[-1]
    grads["out"], grads["bias_out"] = n.t() @ d, d.sum(0)
    d, grads["norm_out"] = norm_back(d @ b["out"].t(), stream, rstd, w["norm_out"])
    for k in (1, 0):
        n, stream, rstd, h = values[1 + k]
        grads[f"down{k}"], grads[f"bias_down{k}"] = h.t() @ d, d.sum(0)
        dz = (d @ b[f"down{k}"].t()) * ((h > 0) & (h < 1))
        grads[f"up{k}"], grads[f"bias_up{k}"] = n.t() @ dz, dz.sum(0)
        through, grads[f"norm{k}"] = norm_back(dz @ b[f"up{k}"].t(), stream, rstd, w[f"norm{k}"])
        d = d + through
    n, stream, rstd = values[0]
    grads["in"] = n.t() @ d
    dx_want, grads["norm_in"] = norm_back(d @ b["in"].t(), stream, rstd, w["norm_in"])
    # at most ten roundings to bf16 one behind the other, of 2^-9 each, and a stream whose sum is kept in bf16 while rstd is that of the sum
    assert off(dx, dx_want) < 12 * 2.0 ** -8 and grads.keys() == trunk.w.gradient.keys()
    for k, g in trunk.w.gradient.items():
        assert off(g, grads[k]) < 12 * 2.0 ** -8, k
    losses = example.train(steps=40, batch=2048, width=128, hidden=256, blocks=2, ft_out=128, report=None)
    assert sum(losses[-4:]) < 0.9 * sum(losses[:4])
