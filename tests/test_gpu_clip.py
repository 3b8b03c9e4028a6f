"""The norm of many tensors and its limit on the GPU against plain forms in 64 bits.

Tolerances.  A thread sums 32 squares in 32 bits, each step off by at most 2^-24 of the sum: 33 x 2^-24 of the squares' sum, half of that of its root, and one rounding of
the result.  An output is its gradient times a share that was rounded once, rounded again to its type."""
import math

import pytest
import torch

from bullet_b200 import _lib, ops

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROUND = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}  # half a step below the smallest normal number
NORM = 18 * 2.0 ** -24


def normal(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g)


def norm64(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


def check(gradients, max_norm, got, norm):
    want = norm64(gradients)
    assert norm.shape == () and norm.dtype is F32
    assert abs(float(norm) - want) <= NORM * want
    share = max_norm / want if want > max_norm else 1.0
    for g, o in zip(gradients, got):
        assert o.dtype is g.dtype and o.shape == g.shape
        off = (o.double() - g.double() * share).abs() - (g.double() * share).abs() * (ROUND[g.dtype] + NORM + 2.0 ** -23) - TINY[g.dtype]
        assert off.numel() == 0 or off.max() <= 0


SETS = [[(1,)], [(7,)], [(3, 5), (1,), (0,), (8192,), (8193,)], [(512, 256), (256,), (256, 512), (512,)], [(1000, 777), (31,), (0, 4), (2, 3, 5)], [(4097, 2049)], [(12288, 256), (256,)],
        [(n,) for n in range(1, 130)], [(33,)] * 300, [()]]


@pytest.mark.parametrize("shapes", SETS, ids=range(len(SETS)))
@pytest.mark.parametrize("kinds", [(F32,), (BF16,), (F16,), (BF16, F32, F16)])
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_clip(shapes, kinds, share):
    gradients = [normal(k, *shape).to(kinds[k % len(kinds)]) for k, shape in enumerate(shapes)]
    norm = ops.gradient_norm(gradients)
    max_norm = share * float(norm)
    got, again = ops.clip_gradients(gradients, max_norm)
    check(gradients, max_norm, got, again)
    assert torch.equal(norm, again)
    before = [g.clone() for g in gradients]
    assert all(torch.equal(a, b) for a, b in zip(gradients, before))
    # in place, and into tensors at hand: the same bits
    at_hand = [torch.full_like(g, 9) for g in gradients]
    out, _ = ops.clip_gradients(gradients, max_norm, out=at_hand)
    assert all(a is b or a.data_ptr() == b.data_ptr() for a, b in zip(out, at_hand)) and all(torch.equal(a, b) for a, b in zip(at_hand, got))
    out, norm = ops.clip_gradients(gradients, max_norm, out=gradients)
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(gradients, got))
    if share > 1:
        assert all(torch.equal(a, b) for a, b in zip(gradients, before))


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("at", [1, 3, 8])
def test_tensors_that_start_anywhere(kind, at):
    raw = normal(11, 30000).to(kind)
    gradients = [raw[at:at + 20000], raw[20008:20009], raw[20011:29998]]
    to = torch.full((30010,), 9.0, device="cuda", dtype=kind)
    out = [to[5:20005], to[20005:20006], to[20008:29995]]
    got, norm = ops.clip_gradients(gradients, 1.5, out=out)
    check(gradients, 1.5, out, norm)
    assert (to[:5] == 9).all() and (to[20006:20008] == 9).all() and (to[29995:] == 9).all()


def test_matrices_in_another_order_of_memory():
    g = normal(12, 300, 200).t()
    got, norm = ops.clip_gradients([g, normal(13, 5)], 0.5)
    assert got[0].stride() == g.stride()
    check([g, normal(13, 5)], 0.5, got, norm)


@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -100, 2.0 ** -70, 2.0 ** 62, 2.0 ** 66, 2.0 ** 120])
def test_squares_that_leave_the_range(size):
    gradients = [normal(14, 10000) * size, torch.zeros(5000, device="cuda"), normal(15, 77) * min(size * 2.0 ** 3, 2.0 ** 120)]
    max_norm = 2.0 ** -20 if size > 1 else 0.5 * norm64(gradients)
    got, norm = ops.clip_gradients(gradients, max_norm)
    want = norm64(gradients)
    assert abs(float(norm) - want) <= NORM * want + 2.0 ** -150
    share = float(torch.tensor(max_norm, dtype=F32)) / want
    for g, o in zip(gradients, got):
        assert ((o.double() - g.double() * share).abs() <= (g.double() * share).abs() * 2.0 ** -21 + 2.0 ** -149).all()


def test_a_norm_past_fp32():
    gradients = [torch.full((1000,), 2.0 ** 127, device="cuda")]
    got, norm = ops.clip_gradients(gradients, 1.0)
    assert torch.isinf(norm) and abs(float(got[0].double().norm()) - 1) < 2.0 ** -20


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), float("-inf")])
def test_a_norm_that_is_not_finite_changes_nothing(bad):
    gradients = [normal(16, 9000), normal(17, 40).to(BF16)]
    gradients[0][4321] = bad
    got, norm = ops.clip_gradients(gradients, 0.5)
    assert not torch.isfinite(norm) and torch.isnan(norm) == math.isnan(bad)
    assert all(torch.equal(a.nan_to_num(5, 6, 7), b.nan_to_num(5, 6, 7)) for a, b in zip(got, gradients))


def test_limits_of_zero_and_without_end():
    g = [normal(18, 100)]
    assert not ops.clip_gradients(g, 0.0)[0][0].any()
    assert torch.equal(ops.clip_gradients(g, float("inf"))[0][0], g[0])
    zeros = [torch.zeros(50, device="cuda")]
    got, norm = ops.clip_gradients(zeros, 0.0)
    assert norm == 0 and not got[0].any()
    assert ops.gradient_norm([torch.empty(0, device="cuda")]) == 0


def test_whole_numbers_are_exact():
    g = [torch.full((3 * 8192 + 5,), 3.0, device="cuda"), torch.full((70000,), 4.0, device="cuda", dtype=BF16)]
    assert float(ops.gradient_norm(g)) == float(torch.tensor(math.sqrt(9 * (3 * 8192 + 5) + 16 * 70000), dtype=F32))


def test_calls_run_on_the_current_stream_and_in_graphs():
    g = [normal(19, 200, 300), normal(20, 300).to(BF16)]
    want, norm = ops.clip_gradients(g, 1.0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(10000000)
        got, _ = ops.clip_gradients(g, 1.0)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = [t.clone() for t in g]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, out_norm = ops.clip_gradients(held, 1.0)
    with torch.cuda.graph(second := torch.cuda.CUDAGraph()):
        ops.clip_gradients(held, 0.25, out=held)
    for seed in (21, 22):
        for k, t in enumerate(held):
            t.copy_(normal(seed + 10 * k, *t.shape))
        want, norm = ops.clip_gradients(held, 1.0)
        less, _ = ops.clip_gradients(held, 0.25)
        graph.replay()
        assert torch.equal(norm, out_norm) and all(torch.equal(a, b) for a, b in zip(out, want))
        second.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, less))


def test_long_tensors():
    g = torch.zeros(2 ** 31 + 5003, dtype=BF16, device="cuda")
    g[-5000:] = normal(23, 5000).to(BF16)
    short = g[-5000:].clone()
    norm = float(ops.gradient_norm([g]))
    assert abs(norm - norm64([short])) <= NORM * norm
    ops.clip_gradients([g], 0.5 * norm, out=[g])
    assert torch.equal(g[-5000:], ops.clip_gradients([short], 0.5 * norm)[0][0]) and not g[:5000].any()


def test_refusals():
    g = normal(24, 64)
    for call in (lambda: ops.gradient_norm([]), lambda: ops.gradient_norm([g, None]), lambda: ops.gradient_norm([g.cpu()]), lambda: ops.gradient_norm([g.double()]),
                 lambda: ops.gradient_norm([g.view(8, 8)[:, :4]]), lambda: ops.gradient_norm([g[:1].expand(4)]), lambda: ops.clip_gradients([g], -1.0),
                 lambda: ops.clip_gradients([g], float("nan")), lambda: ops.clip_gradients([g], 1.0, out=[]), lambda: ops.clip_gradients([g], 1.0, out=[g.to(BF16)]),
                 lambda: ops.clip_gradients([g], 1.0, out=[g[:32]]), lambda: ops.clip_gradients([g.clone().requires_grad_()], 1.0)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.gradient_norm(3), lambda: ops.clip_gradients([g], "x"), lambda: ops.clip_gradients([g], 1.0, out=5)):
        with pytest.raises(TypeError):
            call()
    # one tensor twice in place, outputs that overlap gradients or one another
    for gradients, out in (([g, g], [g, g]), ([g[:40]], [g[20:60]]), ([g[:20], g[20:40]], [g[20:40], g[:20]]), ([g[:8], g[8:16]], [torch.empty(8, device="cuda"), g[:8]]),
                           ([g[:8], g[8:16]], [(t := torch.empty(12, device="cuda"))[:8], t[4:]])):
        with pytest.raises(_lib.B200Error):
            ops.clip_gradients(gradients, 1.0, out=out)
    # one tensor twice, counted or written elsewhere
    assert abs(float(ops.gradient_norm([g, g])) - norm64([g, g])) <= NORM * norm64([g, g])
    ops.clip_gradients([g, g], 1.0)
