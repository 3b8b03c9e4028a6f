"""The residual trunk served in 4 bits, call by call against 64 bits: each operand's codes are the rule's, each layer is its formula at the values of the codes, and
the trunk's output is that of the calls one after another, bit by bit.

Tolerances: those of tests/test_gpu_four.py for a layer in 4 bits, at the values that the very codes stand for; a code that rounding moved moves both sides."""
import pytest
import torch

from bullet_b200 import ops
from bullet_b200.configs import ACT_CRELU
from tests.test_gpu_four import ROUND, check_pack, near, values
from tests.test_gpu_trunk_more import buckets_of, example, normal  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def layer(x, w, bias, act):
    got = ops.dense(x, w, bias=bias, act=act)
    z, size = values(x) @ values(w).t() + bias.double(), values(x).abs() @ values(w).abs().t() + bias.double().abs()
    near(got, z.clamp(0, 1) if act == ACT_CRELU else z, ROUND[BF16] + 2.0 ** -22, (size * (x.length + 4) * 2.0 ** -23 + 2.0 ** -22) * (1 + ROUND[BF16]))
    return got


@pytest.mark.parametrize("rows,width,hidden", [(1, 64, 96), (300, 64, 96), (5003, 256, 512), (16384, 512, 1024)])
def test_the_served_trunk_is_its_calls_and_each_call_its_formula(example, rows, width, hidden):  # noqa: F811
    trunk = example.Trunk(128, width, hidden, 2, buckets=8)
    x, bucket, w, packed = normal(7, rows, 128).clamp(min=0), buckets_of(8, rows, 8), trunk.w, trunk.pack_weights()
    for name, p in packed.items():
        check_pack(w.value[name], p, True)
    stream = ops.dense(ops.rms_norm(x, w.value["norm_in"], out_dtype=BF16)[0], w.bf16["in"])
    delta = ops.embed(w.bf16["bucket"], bucket)
    assert torch.equal(delta, w.bf16["bucket"][bucket.long()])
    for k in range(2):
        n, stream, _ = ops.rms_norm(stream, w.value[f"norm{k}"], residual=delta)
        n4 = ops.pack4(n)
        check_pack(n, n4, False)
        h = layer(n4, packed[f"up{k}"], w.value[f"bias_up{k}"], ACT_CRELU)
        h4 = ops.pack4(h)
        check_pack(h, h4, False)
        delta = layer(h4, packed[f"down{k}"], w.value[f"bias_down{k}"], 0)
    n, _, _ = ops.rms_norm(stream, w.value["norm_out"], residual=delta)
    want = ops.dense(n, w.bf16["out"], bias=w.value["bias_out"], out_dtype=F32)
    assert torch.equal(trunk.serve(x, bucket, packed), want)
