"""A residual trunk behind the feature transformer, trained on synthetic positions with activations kept in 8 bits.

    python examples/residual_trunk.py [--steps 60] [--batch 4096] [--width 256] [--hidden 512] [--blocks 2]

The feature transformer (king-bucketed chess inputs, CReLU, both perspectives) runs as the library's operator and stays as it is;
behind it stand a projection, blocks of  stream += W2 crelu(W1 norm(stream) + b1) + b2  and a norm with the value head, which all
train.  Of a block the backward keeps the sum that the norm was taken of, and in 8 bits the norm's output, which is the first layer's
operand as well, and the hidden layer's; the weights that meet 8-bit activations are packed once per step.
"""
from __future__ import annotations

import argparse
import ctypes
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402
import torch  # noqa: E402

from bullet_b200 import _lib, ops, synth  # noqa: E402
from bullet_b200.configs import ACT_CRELU, NetDesc  # noqa: E402
from bullet_b200.net import featurise, pack_indices  # noqa: E402

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


class FeatureTransformer:
    """b200_op_ft_forward: packed index lists to both perspectives' activations, fp32 [n][2 * out]."""

    def __init__(self, out: int, seed: int):
        self.desc = NetDesc(n_inputs=12288, nnz=32, ft_out=out, ft_act=ACT_CRELU, ft_block_rows=768)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.table = 0.15 * torch.randn(12288, out, device="cuda", generator=g)
        self.bias = torch.full((out,), 0.3, device="cuda")

    def __call__(self, stm, nstm):
        d, n = self.desc, stm.shape[0]
        x = torch.empty(n, 2 * d.ft_out, device="cuda")
        op = _lib.CFtOp(d.n_inputs, d.nnz, d.ft_out, d.ft_act, 0, d.ft_block_rows, n, self.table.data_ptr(), self.bias.data_ptr(), stm.data_ptr(),
                        nstm.data_ptr(), x.data_ptr(), None)
        _lib.check(_lib.load().b200_op_ft_forward(x.device.index, torch.cuda.current_stream().cuda_stream, ctypes.byref(op)))
        return x


class Weights:
    """fp32 weights by name, their gradients, momentum, and the bf16 copies that products take."""

    def __init__(self, shapes: dict, seed: int):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.value = {}
        for name, shape in shapes.items():
            if name.startswith("norm"):
                self.value[name] = torch.ones(shape, device="cuda")
            elif len(shape) == 1:
                self.value[name] = torch.zeros(shape, device="cuda")
            else:
                self.value[name] = torch.randn(shape, device="cuda", generator=g) * shape[0] ** -0.5
        self.moved = {k: torch.zeros_like(v) for k, v in self.value.items()}
        self.gradient = {}
        self.copies()

    def copies(self):
        self.bf16 = {k: v.to(BF16) for k, v in self.value.items() if v.dim() == 2}
        self.codes = {k: ops.pack8(v, by_column=True) for k, v in self.value.items() if k.startswith("up")}

    def step(self, lr: float):
        for k, g in self.gradient.items():
            self.moved[k].mul_(0.9).add_(g)
            self.value[k].add_(self.moved[k], alpha=-lr)
        self.copies()


class Trunk:
    def __init__(self, inputs: int, width: int, hidden: int, blocks: int, seed: int = 1):
        shapes = {"norm_in": (inputs,), "in": (inputs, width), "norm_out": (width,), "out": (width, 1), "bias_out": (1,)}
        for k in range(blocks):
            shapes |= {f"norm{k}": (width,), f"up{k}": (width, hidden), f"bias_up{k}": (hidden,), f"down{k}": (hidden, width), f"bias_down{k}": (width,)}
        self.blocks, self.w = blocks, Weights(shapes, seed)

    def forward(self, x):
        w, kept = self.w, []
        n, _, rstd = ops.rms_norm(x, w.value["norm_in"], out_dtype=BF16)
        kept.append((n, x, rstd))
        stream, delta = ops.dense(n, w.bf16["in"]), None
        for k in range(self.blocks):
            n, stream, rstd = ops.rms_norm(stream, w.value[f"norm{k}"], residual=delta, out_dtype=E4M3)
            h = ops.dense(n, w.codes[f"up{k}"], bias=w.value[f"bias_up{k}"], act=ACT_CRELU)
            kept.append((n, stream, rstd, ops.pack8(h, act=ACT_CRELU)))
            delta = ops.dense(h, w.bf16[f"down{k}"], bias=w.value[f"bias_down{k}"])
        n, stream, rstd = ops.rms_norm(stream, w.value["norm_out"], residual=delta)
        kept.append((n, stream, rstd))
        return ops.dense(n, w.bf16["out"], bias=w.value["bias_out"], out_dtype=torch.float32), kept

    def backward(self, dout, kept):
        """Gradients of all weights into self.w.gradient; returns the gradient at the feature transformer's output."""
        w, g = self.w, self.w.gradient
        n, stream, rstd = kept[-1]
        dn, g["out"], g["bias_out"] = ops.dense_backward(dout, n, w.bf16["out"])
        dstream, g["norm_out"] = ops.rms_norm_backward(dn, stream, rstd, w.value["norm_out"])
        for k in reversed(range(self.blocks)):
            n, stream, rstd, h = kept[1 + k]
            dh, g[f"down{k}"], g[f"bias_down{k}"] = ops.dense_backward(dstream, h, w.bf16[f"down{k}"])
            dn, g[f"up{k}"], g[f"bias_up{k}"] = ops.dense_backward(dh, n, w.bf16[f"up{k}"], y=h, act=ACT_CRELU)
            dstream, g[f"norm{k}"] = ops.rms_norm_backward(dn, stream, rstd, w.value[f"norm{k}"], dtotal=dstream)
        n, x, rstd = kept[0]
        dn, g["in"], _ = ops.dense_backward(dstream, n, w.bf16["in"], need_dbias=False)
        dx, g["norm_in"] = ops.rms_norm_backward(dn, x, rstd, w.value["norm_in"])
        return dx


def train(steps: int = 60, batch: int = 4096, width: int = 256, hidden: int = 512, blocks: int = 2, ft_out: int = 256, lr: float = 0.05, report=print):
    """The mean loss of every step."""
    ft = FeatureTransformer(ft_out, seed=5)
    trunk = Trunk(2 * ft_out, width, hidden, blocks)
    batches = []
    for seed in range(4):
        stm, nstm, _, targets = featurise("chess_buckets", synth.records("chess_buckets", batch, seed=40 + seed), ft.desc)
        lists = [torch.from_numpy(pack_indices(a).view(np.int16)).cuda() for a in (stm, nstm)]
        batches.append((*lists, torch.from_numpy(targets).cuda()))
    losses = []
    for step in range(steps):
        stm, nstm, target = batches[step % len(batches)]
        out, kept = trunk.forward(ft(stm, nstm))
        p = torch.sigmoid(out[:, 0])
        losses.append((p - target).square().mean())
        dout = (2 / batch * (p - target) * p * (1 - p)).to(BF16)[:, None]
        trunk.backward(dout, kept)
        trunk.w.step(lr)
        if report and step % 10 == 0:
            report(f"step {step}: loss {float(losses[-1]):.5f}")
    return [float(v) for v in losses]


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    for name, value in (("steps", 60), ("batch", 4096), ("width", 256), ("hidden", 512), ("blocks", 2)):
        parser.add_argument(f"--{name}", type=int, default=value)
    losses = train(**vars(parser.parse_args()))
    print(f"loss {losses[0]:.5f} -> {losses[-1]:.5f}")
