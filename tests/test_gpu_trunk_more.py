"""The operators of 4 bits, of embedded rows and of the gradients' norm together, as a training step and a server use them: the residual trunk of
examples/residual_trunk.py with a table by output bucket, its gradients limited, its blocks served in 4 bits."""
import importlib.util
import math
import os

import pytest
import torch

from bullet_b200 import ops

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "residual_trunk.py")
    spec = importlib.util.spec_from_file_location("residual_trunk", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def normal(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g)


def off(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def buckets_of(seed, rows, n):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(0, n, (rows,), device="cuda", generator=g, dtype=torch.int32)


@pytest.mark.parametrize("rows", [300, 5003])
def test_a_table_by_bucket_in_the_stream_and_its_gradient(example, rows):
    trunk = example.Trunk(128, 64, 96, 2, buckets=8)
    x, dout, bucket = normal(1, rows, 128).clamp(min=0), normal(2, rows, 1).to(BF16), buckets_of(3, rows, 8)
    out, kept = trunk.forward(x, bucket)
    trunk.backward(dout, kept, bucket)
    # the stream that the first block's norm was taken of is the projection's row and the bucket's
    n, _, rstd = kept[0]
    want = ops.dense(n, trunk.w.bf16["in"]).double() + trunk.w.bf16["bucket"].double()[bucket.long()]
    assert (kept[1][1].double() - want).abs().max() <= want.abs().max() * 2.0 ** -8
    # the table's gradient is, bucket by bucket, the sum of what reaches the projection's output: that is its bias's gradient
    grad = trunk.w.gradient["bucket"]
    assert grad.shape == (8, 64) and grad.dtype is F32
    for k in range(8):
        only = torch.where((bucket == k)[:, None], dout, torch.zeros_like(dout))
        trunk.backward(only, kept, bucket)
        mine = trunk.w.gradient["bucket"]
        assert off(mine[k], grad[k]) < 1e-5 and not mine[[j for j in range(8) if j != k]].any()
    # a bucket that no position has stays without a gradient
    trunk.backward(dout, kept, bucket.clamp(max=5))
    assert not trunk.w.gradient["bucket"][6:].any() and trunk.w.gradient["bucket"][:6].any(1).all()


def test_a_step_whose_gradients_are_limited(example):
    trunk = example.Trunk(128, 64, 96, 2, buckets=8)
    x, dout, bucket = normal(4, 700, 128).clamp(min=0), normal(5, 700, 1).to(BF16), buckets_of(6, 700, 8)
    out, kept = trunk.forward(x, bucket)
    trunk.backward(dout, kept, bucket)
    before = {k: g.clone() for k, g in trunk.w.gradient.items()}
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in before.values()))
    assert abs(float(trunk.w.step(0.1, max_norm=0.25 * norm)) - norm) < 1e-5 * norm
    for k, g in trunk.w.gradient.items():
        assert (g.double() - 0.25 * before[k].double()).abs().max() <= 1e-5 * before[k].abs().max()
        assert torch.equal(trunk.w.moved[k], g)
    # above the norm nothing changes
    trunk.backward(dout, kept, bucket)
    before = {k: g.clone() for k, g in trunk.w.gradient.items()}
    trunk.w.step(0.1, max_norm=2 * math.sqrt(sum(float(g.double().square().sum()) for g in before.values())))  # (of the moved weights' gradients)
    assert all(torch.equal(g, before[k]) for k, g in trunk.w.gradient.items())


@pytest.mark.parametrize("rows", [1, 300])
def test_the_trunk_served_in_4_bits_is_its_formulas_on_the_values_of_the_codes(example, rows):
    trunk = example.Trunk(128, 64, 96, 2, buckets=8)
    x, bucket = normal(7, rows, 128).clamp(min=0), buckets_of(8, rows, 8)
    packed = trunk.pack_weights()
    got = trunk.serve(x, bucket, packed)
    assert torch.equal(got, trunk.serve(x, bucket))
    w = {k: v.double() for k, v in trunk.w.value.items()}
    stream = ops.dense(ops.rms_norm(x, trunk.w.value["norm_in"], out_dtype=BF16)[0], trunk.w.bf16["in"])
    delta = ops.embed(trunk.w.bf16["bucket"], bucket)
    for k in range(2):
        n, stream, _ = ops.rms_norm(stream, trunk.w.value[f"norm{k}"], residual=delta)
        up, down = (ops.unpack4(packed[f"{name}{k}"], F32).double() for name in ("up", "down"))
        h = (ops.unpack4(ops.pack4(n), F32).double() @ up + w[f"bias_up{k}"]).clamp(0, 1).to(BF16)
        delta = (ops.unpack4(ops.pack4(h), F32).double() @ down + w[f"bias_down{k}"]).to(BF16)
    n, _, _ = ops.rms_norm(stream, trunk.w.value["norm_out"], residual=delta)
    want = ops.dense(n, trunk.w.bf16["out"], bias=trunk.w.value["bias_out"], out_dtype=F32)
    # sums of 64 and 96 products in 32 bits may round to the other neighbour in bf16, which moves a code of 4 bits now and then
    assert off(got, want) < 0.02
    # and codes of 4 bits are what it costs: of norms' outputs, activations and weights, of 2^-3.5 each in the mean square at most, twice, beside the stream's own part
    assert off(got, trunk.forward(x, bucket)[0]) < 0.5


def test_training_with_buckets_and_a_limit_runs(example):
    losses = example.train(steps=6, batch=512, width=64, hidden=96, blocks=1, ft_out=64, report=None, buckets=8, clip=0.01)
    assert len(losses) == 6 and all(math.isfinite(v) for v in losses)


def test_the_operators_together_in_one_graph(example):
    """Packing, a layer, a lookup with its gradient and the limit of two gradients, captured once and replayed on other inputs, beside an eager call in between."""
    table, w = normal(11, 8, 256).to(BF16), ops.pack4(normal(12, 256, 128) * 0.1, by_column=True)
    x, bucket, dy = normal(13, 500, 256).to(BF16), buckets_of(14, 500, 8), normal(15, 500, 256).to(BF16)

    def step():
        y = ops.dense(ops.pack4(ops.rms_norm(x, residual=ops.embed(table, bucket))[0]), w)
        g = [ops.embed_backward(dy, bucket, 8), dy]
        return (y, *ops.clip_gradients(g, 1.0)[0], ops.gradient_norm(g))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (16, 17):
        x.copy_(normal(seed, 500, 256))
        dy.copy_(normal(seed + 10, 500, 256))
        bucket.copy_(buckets_of(seed, 500, 8))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
