"""Pairs of SMs that multiply together in 4 bits, beside other work."""
import pytest
import torch

from bullet_b200 import ops
from tests.test_gpu_four import values
from tests.test_gpu_more_kernels import PAIRS, layer, whole

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("shape", [PAIRS[0], PAIRS[2]], ids=str)
def test_pairs_of_tiles_give_the_same_bits_beside_other_work(shape):
    """Again and again, in two streams at once: scales and sums of one CTA of a pair that the other's products met too early or too late would show."""
    rows, _, n_out = shape
    x, w = layer(*shape)
    r = whole(46, BF16, rows, n_out)
    want = ((values(x) @ values(w).t()) + r.double()).to(BF16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(ops.dense(x, w, residual=r))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
