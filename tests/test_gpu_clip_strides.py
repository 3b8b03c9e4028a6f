"""Outputs whose dimensions of one element have strides of their own lie as their gradients do."""
import pytest
import torch

from bullet_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,strides", [((1, 6), (77, 1)), ((6, 1), (1, 99)), ((3, 1, 4), (4, 1000, 1)), ((1, 1), (5, 3)), ((0, 4), (9, 2))])
def test_dimensions_of_one_element(shape, strides):
    g = torch.randn(*shape, device="cuda")
    out = torch.empty_strided(shape, strides, device="cuda")
    got, norm = ops.clip_gradients([g], 0.5, out=[out])
    want, other = ops.clip_gradients([g], 0.5)
    assert torch.equal(out, want[0]) and torch.equal(norm, other) and got[0].data_ptr() == out.data_ptr()


def test_other_orders_of_memory_are_refused_still():
    g = torch.randn(4, 6, device="cuda")
    for out in (torch.empty(6, 4, device="cuda").t(), torch.empty(4, 12, device="cuda")[:, :6], torch.empty(4, 6, 1, device="cuda"), torch.empty(4, 1, 6, device="cuda")):
        with pytest.raises(ValueError):
            ops.clip_gradients([g], 0.5, out=[out])
