"""What torch is told of tensors that the limit of gradients writes."""
import pytest
import torch

from bullet_b200 import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def normal(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g)


@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_autograd_hears_of_tensors_that_were_written(max_norm):
    """As behind torch's own operations in place, changed or not: a backward that has kept the tensor refuses to go on with other values."""
    x, w = normal(1, 40).requires_grad_(), normal(2, 40)
    y = (x * w).sum()
    ops.clip_gradients([w], max_norm, out=[w])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_versions_of_what_is_written_and_read():
    g, out, whole = [normal(3, 7), normal(4, 5, 3).to(BF16)], [torch.empty(7, device="cuda"), torch.empty(5, 3, device="cuda", dtype=BF16)], normal(5, 9)
    before = [t._version for t in g + out]
    ops.clip_gradients(g, 0.5, out=out)
    assert [t._version for t in g] == before[:2] and [t._version for t in out] == [v + 1 for v in before[2:]]
    ops.gradient_norm(g)
    ops.clip_gradients(g, 0.5)
    assert [t._version for t in g] == before[:2]
    # what another tensor has a view of
    was = whole._version
    ops.clip_gradients([whole[:4]], 0.5, out=[whole[:4]])
    assert whole._version == was + 1
    # a call that is refused has written nothing
    with pytest.raises(ValueError):
        ops.clip_gradients(g, -1.0, out=out)
    assert [t._version for t in out] == [v + 1 for v in before[2:]]


def test_tensors_of_inference_mode_have_no_versions():
    with torch.inference_mode():
        t = normal(6, 100)
    want = ops.clip_gradients([t.clone()], 0.5)[0][0]
    ops.clip_gradients([t], 0.5, out=[t])
    assert torch.equal(t, want)
