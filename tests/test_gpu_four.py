"""Matrices in 4 bits and the dense layers on them, on the GPU against plain forms in 64 bits.

Tolerances.  Codes and scales are the rule's, exactly.  Products of codes are exact; a sum of k of them in 32 bits is off by at most k 2^-23 of the
sum of their magnitudes, in any order and whether a step rounds or cuts off, and sums of few bits are exact.  A value rounded to a type with p
significand bits is off by at most 2^-p of itself (24, 8 and 11 bits: fp32, bf16, fp16)."""
import pytest
import torch

from bullet_b200 import _lib, ops
from bullet_b200.configs import ACT_CRELU, ACT_NONE, ACT_RELU, ACT_SCRELU

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROUND = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}  # half a step below fp16's smallest normal number
SIZES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(seed, *shape):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def spaced(t, pad, at=0):
    """The same matrix with `pad` more elements between rows, `at` elements into a buffer of NaN (codes: of 0xff)."""
    rows, cols = t.shape
    raw = torch.full((at + rows * (cols + pad),), 255 if t.dtype is torch.uint8 else float("nan"), device="cuda").to(t.dtype)
    v = raw[at:].view(rows, cols + pad)[:, :cols]
    v.copy_(t)
    return v


def near(got, want, relative, absolute=0.0):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    off = (got - want).abs() - (relative * want.abs() + absolute)
    assert not torch.isnan(off).any() and off.max() <= 0 if off.numel() else True, float(off.max())


def scale_bytes(scale, rows, length):
    """The scales' bytes [rows][groups], each from where the header says that it lies."""
    r, g = torch.arange(rows, device="cuda")[:, None], torch.arange((length + 31) // 32, device="cuda")[None, :]
    across = (length + 127) // 128
    return scale[(r // 128 * across + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4]


def elements(codes, length):
    """The codes [rows][length], one by one."""
    return torch.stack((codes & 15, codes >> 4), 2).reshape(codes.shape[0], -1)[:, :length]


def values(packed):
    """What a Packed4 stands for in 64 bits, in rows along the packed axis."""
    code = elements(packed.codes, packed.length).long()
    e = scale_bytes(packed.scale, packed.codes.shape[0], packed.length).double()
    f = torch.where(e == 255, float("nan"), torch.exp2(e - 127)).repeat_interleave(32, 1)[:, :packed.length]
    return SIZES.cuda()[code % 8] * torch.where(code >= 8, -1.0, 1.0) * f


def exact_pack(x):
    """(values, bytes of scales) by the rule, of rows in 64 bits."""
    rows, length = x.shape
    whole = torch.zeros(rows, (length + 31) // 32 * 32, dtype=torch.float64, device="cuda")
    whole[:, :length] = x
    whole = whole.view(rows, -1, 32)
    bad = ~torch.isfinite(whole).all(2, keepdim=True)
    amax = torch.where(bad, 0.0, whole.abs().nan_to_num().amax(2, keepdim=True))
    m, e = torch.frexp(amax / 6)  # (a logarithm may be off by its last bit where this is a power of two)
    e = torch.where(amax > 0, torch.where(m == 0.5, e - 1, e).clamp(min=-126), 0)
    v = whole / torch.exp2(e.double())
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=1))) - 1)
    v = torch.round(v / step) * step
    v = torch.where((e == 126) & (v.abs() > 3), v.sign() * 3, v) * torch.exp2(e.double())
    v = torch.where(bad, float("nan"), v)
    return v.view(rows, -1)[:, :length], torch.where(bad, 255, e + 127).view(rows, -1)


def check_pack(x, packed, by_column):
    want, scale = exact_pack(x.double().t() if by_column else x.double())
    rows, length = want.shape
    assert packed.length == length and packed.by_column == by_column and packed.codes.shape == (rows, (length + 31) // 32 * 16)
    assert torch.equal(scale_bytes(packed.scale, rows, length).long(), scale.long())
    assert torch.equal(values(packed).nan_to_num(12345.0), want.nan_to_num(12345.0))
    assert (elements(packed.codes, packed.codes.shape[1] * 2)[:, length:] == 0).all()
    # (bytes of no group of the matrix)
    up, across = (rows + 127) // 128, (length + 127) // 128
    all_of = packed.scale.view(up, across, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(up * 128, across * 4)
    assert (all_of[rows:] == 127).all() and (all_of[:, (length + 31) // 32:] == 127).all()


PACKS = [(1, 2048, BF16), (3, 1, F32), (2, 7, F16), (5, 200, F32), (33, 520, BF16), (129, 768, F16), (128, 128, BF16), (17, 1000, BF16), (7, 333, BF16), (300, 64, BF16),
         (1000, 96, F32), (1, 1, BF16), (31, 31, F32), (2, 20001, F32), (260, 4100, BF16)]


@pytest.mark.parametrize("rows,cols,kind", PACKS)
@pytest.mark.parametrize("by_column", [False, True])
@pytest.mark.parametrize("pad,at", [(0, 0), (8, 0), (3, 1)])
def test_pack(rows, cols, kind, by_column, pad, at):
    x = spaced((normal(21, rows, cols) * torch.exp(2 * normal(22, cols))).to(kind), pad, at)
    packed = ops.pack4(x, by_column=by_column)
    check_pack(x, packed, by_column)
    for out in (F32, BF16, F16):
        got = ops.unpack4(packed, out)
        want = values(packed).t() if by_column else values(packed)
        assert got.shape == x.shape and torch.equal(got, want.to(out))
    # a matrix of codes inside a larger one
    wider = packed._replace(codes=spaced(packed.codes, 32, 16))
    assert torch.equal(ops.unpack4(wider, F32), ops.unpack4(packed, F32))


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("by_column", [False, True])
def test_pack_of_every_halfway_point_and_its_neighbours(kind, by_column):
    points = torch.tensor([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5], dtype=F32)
    points = torch.cat((points, points * (1 + 2.0 ** -7), points * (1 - 2.0 ** -7)))
    points = torch.cat((points, -points))
    x = torch.zeros(points.numel(), 32)
    x[:, 0], x[:, 1] = 6, points
    x = (torch.cat([x * 2.0 ** e for e in (-3, 0, 5)])).to(kind).cuda()
    x = x.t().contiguous() if by_column else x
    check_pack(x, ops.pack4(x, by_column=by_column), by_column)


@pytest.mark.parametrize("cols", [96, 333, 2048])
@pytest.mark.parametrize("by_column", [False, True])
def test_pack_of_extremes(cols, by_column):
    x = normal(23, 12, cols)
    x[0] = 0
    x[1, 40] = float("nan")
    x[2, 70] = float("inf")
    x[3, 5] = float("-inf")
    x[4] *= 2.0 ** 124
    x[5, 3] = torch.finfo(F32).max
    x[6] *= 2.0 ** -130
    x[7] = 2.0 ** -149
    x[8, 64:] = 0
    x[9] = -0.0
    x[10, 33], x[10, 34] = 1.4 * 2.0 ** 127, 2.0 ** 127
    x[11] = torch.where(x[11] > 0, 2.0 ** 125 * 6, 2.0 ** 100)
    x = x.t().contiguous() if by_column else x
    packed = ops.pack4(x, by_column=by_column)
    check_pack(x, packed, by_column)
    got = ops.unpack4(packed, F32)
    want = values(packed).t() if by_column else values(packed)
    assert torch.equal(got.nan_to_num(7), want.float().nan_to_num(7)) and not torch.isinf(got).any()


def random_codes(seed, rows, length, low, high):
    """A Packed4 of every code and of scales 2^low to 2^high."""
    g = gen(seed)
    groups, up, across = (length + 31) // 32, (rows + 127) // 128, (length + 127) // 128
    code = torch.randint(0, 16, (rows, groups * 32), device="cuda", generator=g, dtype=torch.uint8)
    code[:, length:] = 0
    code = code.view(rows, groups * 16, 2)
    scale = torch.randint(127 + low, 128 + high, (up * across * 512,), device="cuda", generator=g, dtype=torch.uint8)
    return ops.Packed4(code[:, :, 0] | code[:, :, 1] << 4, scale, length)


def test_values_of_scales_from_elsewhere():
    p = random_codes(31, 70, 200, -5, 5)
    p.scale[:] = torch.arange(p.scale.numel(), device="cuda") % 255
    assert torch.equal(ops.unpack4(p, F32), values(p).float())


SHAPES = [(1, 32, 8), (1, 2048, 1024), (2, 100, 33), (3, 4096, 16), (4, 64, 1), (5, 1000, 200), (8, 512, 520), (8, 9000, 40), (9, 64, 48), (17, 33, 7), (65, 77, 33),
          (128, 128, 128), (129, 256, 136), (130, 1024, 264), (200, 260, 250), (257, 64, 512), (300, 8, 16), (700, 2048, 512), (1000, 96, 520), (3000, 192, 40), (20000, 320, 256),
          (5003, 1100, 777), (40, 20000, 72)]


@pytest.mark.parametrize("rows,n_in,n_out", SHAPES)
def test_dense_of_few_bits_is_exact(rows, n_in, n_out):
    x, w = random_codes(41, rows, n_in, -1, 1), random_codes(42, n_out, n_in, -1, 0)._replace(by_column=True)
    want = values(x) @ values(w).t()
    assert (values(x).abs() @ values(w).abs().t()).max() < 2.0 ** 20  # (the smallest product is 2^-4)
    assert torch.equal(ops.dense(x, w, out_dtype=F32).double(), want)
    r = torch.randint(-8, 9, (rows, n_out), device="cuda", generator=gen(43)).float()
    b = torch.randint(-8, 9, (n_out,), device="cuda", generator=gen(44)).float()
    assert torch.equal(ops.dense(x, w, bias=b, act=ACT_RELU, residual=r, out_dtype=F32).double(), (want + b).clamp(min=0) + r)


def activated(z, act):
    if act == ACT_NONE:
        return z
    z = z.clamp(min=0) if act == ACT_RELU else z.clamp(0, 1)
    return z * z if act == ACT_SCRELU else z


@pytest.mark.parametrize("rows,n_in,n_out", [(1, 512, 256), (6, 96, 40), (130, 1024, 264), (700, 2048, 512), (65, 77, 33), (3000, 512, 1024)])
@pytest.mark.parametrize("out", [BF16, F32, F16])
@pytest.mark.parametrize("act", [ACT_NONE, ACT_CRELU, ACT_SCRELU, ACT_RELU])
@pytest.mark.parametrize("with_residual", [False, True])
def test_dense(rows, n_in, n_out, out, act, with_residual):
    x = ops.pack4((normal(51, rows, n_in) * 0.6 + 0.3).clamp(0, 1))
    w = ops.pack4(normal(52, n_in, n_out) * n_in ** -0.5, by_column=True)
    b = 0.1 * normal(53, n_out)
    r = spaced(normal(54, rows, n_out).to(out), 8) if with_residual else None
    z, size = values(x) @ values(w).t() + b.double(), values(x).abs() @ values(w).abs().t() + b.double().abs()
    want = activated(z, act) + (r.double() if with_residual else 0)
    off = size * (n_in + 4) * 2.0 ** -23 * (2 if act == ACT_SCRELU else 1) + 2.0 ** -22
    got = ops.dense(x, w, bias=b, act=act, residual=r, out_dtype=out)
    near(got, want, ROUND[out] + 2.0 ** -22, off * (1 + ROUND[out]) + TINY[out])
    assert torch.equal(got, ops.dense(x, w, bias=b, act=act, residual=r, out_dtype=out))
    if out is BF16:
        assert torch.equal(got, ops.dense(x, w, bias=b, act=act, residual=r))


@pytest.mark.parametrize("rows,n_in,n_out", [(1, 128, 64), (7, 64, 48), (150, 96, 272), (400, 600, 264)])
@pytest.mark.parametrize("pads", [(16, 0, 0, 0), (0, 48, 0, 0), (0, 0, 5, 0), (32, 16, 7, 1), (0, 0, 0, 1), (16, 16, 8, 8)])
def test_dense_of_matrices_inside_larger_ones(rows, n_in, n_out, pads):
    x, w = random_codes(61, rows, n_in, -1, 1), random_codes(62, n_out, n_in, -1, 0)._replace(by_column=True)
    inside = x._replace(codes=spaced(x.codes, pads[0], 16)), w._replace(codes=spaced(w.codes, pads[1], 16))
    r = spaced(torch.randint(-8, 9, (rows, n_out), device="cuda", generator=gen(63)).to(BF16), pads[2], pads[3])
    want = values(x) @ values(w).t() + r.double()
    assert torch.equal(ops.dense(*inside, residual=r, out_dtype=BF16), want.to(BF16))


@pytest.mark.parametrize("rows", [3, 200])
def test_dense_keeps_what_is_not_finite_where_it_belongs(rows):
    x = normal(71, rows, 320)
    x[1, 200] = float("nan")
    w = normal(72, 320, 96)
    w[7, 40] = float("inf")
    got = ops.dense(ops.pack4(x), ops.pack4(w, by_column=True), out_dtype=F32)
    bad = torch.isnan(got)
    assert bad[1].all() and bad[:, 40].all()
    bad[1] = False
    bad[:, 40] = False
    assert not bad.any()


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("high", [100, -100])
def test_dense_at_extreme_scales(rows, high):
    """Scales whose product is moderate, each of them far out."""
    x, w = random_codes(73, rows, 256, 0, 2), random_codes(74, 40, 256, 0, 1)._replace(by_column=True)
    want = ops.dense(x, w, out_dtype=F32)
    moved = ops.dense(x._replace(scale=x.scale + high % 256), w._replace(scale=w.scale + -high % 256), out_dtype=F32)
    assert torch.equal(moved, want) and want.abs().max() > 1


def test_gradient_of_a_layer_in_4_bits_is_that_of_its_values():
    """dense_backward at the values that codes stand for: the gradient of the layer as computed, against differences of its output in 64 bits."""
    x, w = ops.pack4(normal(81, 70, 96)), ops.pack4(normal(82, 96, 40) * 0.1, by_column=True)
    y = ops.dense(x, w, act=ACT_CRELU)
    dy = normal(83, 70, 40).to(BF16)
    dx, dw, db = ops.dense_backward(dy, ops.unpack4(x), ops.unpack4(w), y=y, act=ACT_CRELU)
    xv, wv = values(x), values(w).t().contiguous()
    z = xv @ wv
    # (what rounding y to bf16 may put on the other side of a border is left out)
    clear = ((z.abs() > 1e-5) & ((z - 1).abs() > 5e-3)).double()
    dz = dy.double() * ((z > 0) & (z < 1))
    assert ((dy.double() * ((y > 0) & (y < 1)) - dz).abs() * clear).max() == 0
    dz = dy.double() * ((y > 0) & (y < 1))
    size = 40 * 2.0 ** -23
    near(dx, dz @ wv.t(), ROUND[BF16] + size, size * (dz.abs() @ wv.abs().t()))
    near(dw, xv.t() @ dz, 2.0 ** -24, 70 * 2.0 ** -23 * (xv.abs().t() @ dz.abs()))
    g, h = gen(84), 1e-6
    along = torch.randn(96, 40, device="cuda", generator=g, dtype=torch.float64)
    inner = ((z > 1e-3) & (z < 1 - 1e-2)).double() * dy.double()
    difference = (((xv @ (wv + h * along)).clamp(0, 1) - (xv @ (wv - h * along)).clamp(0, 1)) * inner).sum() / (2 * h)
    formula = ((xv.t() @ inner) * along).sum()
    assert abs(float(difference - formula)) < 1e-6 * float((xv.abs().t() @ inner.abs() * along.abs()).sum())


def test_no_rows():
    w = ops.pack4(normal(91, 64, 32), by_column=True)
    x = ops.pack4(torch.empty(0, 64, device="cuda"))
    assert ops.dense(x, w).shape == (0, 32) and ops.unpack4(x).shape == (0, 64)
    assert ops.unpack4(ops.pack4(torch.empty(0, 5, device="cuda"), by_column=True)).shape == (0, 5)


@pytest.mark.parametrize("rows", [5, 700])
def test_calls_run_on_the_current_stream_and_in_graphs(rows):
    x, w = normal(92, rows, 512), ops.pack4(normal(93, 512, 256), by_column=True)
    want = ops.dense(ops.pack4(x), w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(10000000)
        got = ops.dense(ops.pack4(x), w)
    stream.synchronize()
    assert torch.equal(got, want)
    graph, held = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = ops.dense(ops.pack4(held), w)
    for seed in (94, 95):
        held.copy_(normal(seed, rows, 512))
        graph.replay()
        assert torch.equal(out, ops.dense(ops.pack4(held), w))


def test_long_matrices_pass_32_bit_offsets():
    """More than 2^32 bytes of values and 2^31 of codes: the last rows are those of a short matrix."""
    rows, cols = 2200000, 2048
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    x[-300:] = normal(96, 300, cols).to(BF16)
    packed = ops.pack4(x)
    short = ops.pack4(x[-300:].contiguous())
    assert torch.equal(packed.codes[-300:], short.codes)
    w = ops.pack4(normal(97, cols, 16), by_column=True)
    del x
    got = ops.dense(packed, w)
    assert torch.equal(got[-300:], ops.dense(short, w)) and not got[:-300].any()
    del got
    y = ops.unpack4(packed)
    assert torch.equal(y[-300:], ops.unpack4(short)) and not y[:1000].any()


def test_refusals_of_tensors():
    x, w = ops.pack4(normal(98, 4, 64)), ops.pack4(normal(99, 64, 16), by_column=True)
    for call in (lambda: ops.dense(x, normal(1, 64, 16).to(BF16)), lambda: ops.dense(normal(1, 4, 64).to(BF16), w), lambda: ops.dense(x, x), lambda: ops.dense(w, w),
                 lambda: ops.dense(x, ops.pack4(normal(1, 96, 16), by_column=True)), lambda: ops.dense(x._replace(length=96), w), lambda: ops.dense(x._replace(scale=x.scale[:256]), w),
                 lambda: ops.dense(x._replace(codes=x.codes.int()), w), lambda: ops.dense(x, w, act=7), lambda: ops.dense(x, w, residual=normal(1, 4, 16)),
                 lambda: ops.dense(x, w, bias=normal(1, 15)), lambda: ops.dense(x, w, out_dtype=torch.int8), lambda: ops.unpack4(x, torch.int8), lambda: ops.pack4(normal(1, 64)),
                 lambda: ops.pack4(normal(1, 4, 64).double()), lambda: ops.dense(x._replace(codes=spaced(x.codes, 8)), w), lambda: ops.dense(x._replace(codes=spaced(x.codes, 0, 8)), w),
                 lambda: ops.dense(x._replace(codes=x.codes.cpu()), w), lambda: ops.dense(x._replace(scale=x.scale.cpu()), w), lambda: ops.pack4(normal(1, 4, 64).t()),
                 lambda: ops.unpack4(x._replace(length=-1)), lambda: ops.dense(x, ops.pack8(normal(1, 64, 16), by_column=True))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.B200Error):
        ops.pack4(torch.empty(4, 0, device="cuda"))
