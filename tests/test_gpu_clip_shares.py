"""Shares that fp32 holds in few bits or not at all: the limit of gradients on the GPU against 64 bits.

Tolerances.  A norm is that of one element, or of as many equal ones as a power of four, and its share is right to 2^-52; an output is off by at most half a step of its
type, and what lies below its type's normal numbers by half a step of the smallest."""
import pytest
import torch

from bullet_b200 import ops

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("limit", [-60, -100, -110, -120, -126, -130, -140, -149])
@pytest.mark.parametrize("size", [100, 120, 127])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_one_large_element(limit, size, kind):
    g = torch.zeros(5000, device="cuda", dtype=kind)
    g[77] = 2.0 ** size
    (got,), norm = ops.clip_gradients([g], 2.0 ** limit)
    assert float(norm) == 2.0 ** size
    # (bf16: halves of its smallest number go to the even one)
    assert float(got[77]) == (2.0 ** limit if kind is F32 or limit >= -133 else 0.0) and int(got.count_nonzero()) == int(got[77] != 0)


@pytest.mark.parametrize("limit", [1.3 * 2.0 ** -80, 1.7 * 2.0 ** -100, 1.1 * 2.0 ** -120, 1.9 * 2.0 ** -126])
@pytest.mark.parametrize("count", [1, 4, 4096, 65536])
def test_elements_of_all_sizes_beside_large_ones(limit, count):
    """The large ones are the norm to the last bit of 64: the squares of the others are below 2^-60 of theirs."""
    large = torch.full((count,), 2.0 ** 126, device="cuda")
    small = torch.randn(3000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 2.0 ** 90
    limit = float(torch.tensor(limit, dtype=F32))
    got, _ = ops.clip_gradients([large, small], limit)
    share = limit / (2.0 ** 126 * count ** 0.5)
    for g, o in zip((large, small), got):
        want = g.double() * share
        assert ((o.double() - want).abs() <= want.abs() * 2.0 ** -24 * (1 + 2.0 ** -20) + 2.0 ** -150).all()


def test_a_share_that_no_output_survives():
    g = torch.full((100,), 2.0 ** 20, device="cuda")
    assert not ops.clip_gradients([g], 2.0 ** -149)[0][0].any()
