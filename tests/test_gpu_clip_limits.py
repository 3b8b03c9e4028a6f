"""Limits of 64 bits, as Python's numbers are: the share is the limit by the norm in 64 bits, rounded once to fp32, and an output is rounded once more."""
import ctypes

import numpy as np
import pytest
import torch

from bullet_b200 import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [0, -30, 40])
def test_shares_are_of_the_limit_as_it_is(power):
    """Of 3 and 4 the norm is 5 in all bits."""
    g = torch.tensor([3.0, 4.0], device="cuda") * 2.0 ** power
    limits = np.random.default_rng(7).uniform(0.01, 4.99, 300) * 2.0 ** power
    cut = 0
    for limit in limits.tolist():
        (got,), norm = ops.clip_gradients([g], limit)
        share = np.float32(limit / (5 * 2.0 ** power))
        assert float(norm) == 5 * 2.0 ** power and got.tolist() == (g.cpu().numpy() * share).tolist()
        cut += share != np.float32(float(np.float32(limit)) / (5 * 2.0 ** power))
    assert cut > 20  # (those that a limit of 32 bits would move by a step)


def test_limits_past_32_bits():
    g = [torch.full((16,), 2.0 ** 127, device="cuda")]
    assert torch.equal(ops.clip_gradients(g, 1e39)[0][0], g[0])
    assert not ops.clip_gradients(g, 1e-60)[0][0].any()
    for bad in (-1e-60, -1e39, float("-inf"), float("nan")):
        with pytest.raises(ValueError):
            ops.clip_gradients(g, bad)


def test_the_two_parts_of_a_limit_over_the_c_abi():
    g, space = torch.tensor([3.0, 4.0], device="cuda"), torch.empty(1 << 16, device="cuda", dtype=torch.uint8)
    out, norm = torch.empty(2, device="cuda"), torch.empty(1, device="cuda")
    array = (_lib.CGradient * 1)(_lib.CGradient(g.data_ptr(), out.data_ptr(), 2, 0))

    def call(limit, low):
        op = _lib.CClip(count=1, gradients=ctypes.addressof(array), norm=norm.data_ptr(), workspace=space.data_ptr(), max_norm=limit, max_norm_low=low, workspace_bytes=space.numel())
        return _lib.load().b200_op_clip_gradients(0, torch.cuda.current_stream().cuda_stream, ctypes.byref(op))

    for limit, low in ((1.0, 0.0), (1.0, 2.0 ** -26), (1.0, -(2.0 ** -26)), (0.7, 3e-9)):
        assert call(limit, low) == 0
        share = np.float32((float(np.float32(limit)) + float(np.float32(low))) / 5)
        assert out.tolist() == (np.array([3, 4], np.float32) * share).tolist()
    assert call(1.0, -1.5) == -1 and call(1.0, float("nan")) == -1 and call(float("inf"), float("-inf")) == -1
