"""Cases of the operators of a wide dense trunk behind the feature transformer: root-mean-square norm with the residual's
addition, activation checkpoints in 8 bits, dense layers with bias, activation and residual, and the gradients of all.

`run` computes a case in plain torch operations in 32 bits, or, where `own` is true, with the package's operators.  Weights
are what the package's networks have: [in][out] in memory, the column-major out x in matrix.  Codes of 8 bits are e4m3 with a
power of two as scale, per row for activations and per column of the memory for weights.

Sizes: the networks' batches (1 position, 5003, 16384, 131072) and widths (200 to 2048), and what lies between.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
ACTS = {"none": 0, "crelu": 1, "screlu": 2, "relu": 3}
EPS = 1e-5
LARGEST = 131072 * 2048 * 512  # rows x in x out of the largest listed dense case


def listed():
    return [
        # one position through a residual block of a served network: latency
        {"name": "norm-one", "op": "norm", "rows": 1, "cols": 2048, "x": "bf16", "y": "bf16", "residual": True},
        # the feature transformer's output (2 x 1024, fp32) on its way into an 8-bit layer
        {"name": "norm-ft-8bit", "op": "norm", "rows": 16384, "cols": 2048, "x": "f32", "y": "e4m3", "residual": False},
        # a whole training batch's residual stream, the normed copy kept in 8 bits
        {"name": "norm-large-8bit", "op": "norm", "rows": 131072, "cols": 2048, "x": "bf16", "y": "e4m3", "residual": True},
        # gradient for a batch that fills no power of two, a narrow stream
        {"name": "norm-back-ragged", "op": "norm_back", "rows": 5003, "cols": 520, "x": "bf16", "dy": "bf16", "through": True},
        # gradient of a whole training batch, back into an fp32 feature transformer
        {"name": "norm-back-large", "op": "norm_back", "rows": 131072, "cols": 1024, "x": "f32", "dy": "bf16", "through": False},
        # a checkpoint of a narrow layer's outputs written and read back
        {"name": "checkpoint-ragged", "op": "pack", "rows": 5003, "cols": 200, "x": "f32", "act": "screlu", "by_column": False},
        # a checkpoint of a whole batch of wide activations written and read back
        {"name": "checkpoint-large", "op": "pack", "rows": 131072, "cols": 2048, "x": "bf16", "act": "crelu", "by_column": False},
        # one position through a layer of a served network: latency
        {"name": "dense-one", "op": "dense", "rows": 1, "in": 2048, "out": 1024, "x": "bf16", "y": "bf16", "act": "crelu", "residual": False},
        # the second half of a residual block, an ordinary batch
        {"name": "dense-residual", "op": "dense", "rows": 16384, "in": 1024, "out": 2048, "x": "bf16", "y": "bf16", "act": "none", "residual": True},
        # the narrowing layer of a large batch on 8-bit activations and weights
        {"name": "dense-8bit", "op": "dense", "rows": 131072, "in": 2048, "out": 512, "x": "e4m3", "y": "bf16", "act": "screlu", "residual": False},
        # gradient of a layer for a ragged batch, all in 16 bits
        {"name": "dense-back-ragged", "op": "dense_back", "rows": 5003, "in": 2048, "out": 1024, "x": "bf16", "dy": "bf16", "saved": "bf16", "dw": "bf16",
         "act": "screlu", "skip": True},
        # gradient of the large batch's layer from 8-bit checkpoints of its input and its output
        {"name": "dense-back-8bit", "op": "dense_back", "rows": 131072, "in": 2048, "out": 512, "x": "e4m3", "dy": "bf16", "saved": "e4m3", "dw": "f32",
         "act": "crelu", "skip": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high, odd):
    """A width: a multiple of 16 as a rule, now and then any number."""
    w = _log(rng, low, high)
    return w if rng.random() < odd else max(16, w // 16 * 16)


def draw(rng):
    op = rng.choice(["norm", "norm_back", "pack", "dense", "dense", "dense_back"])
    rows = _log(rng, 1, 131072)
    if op == "norm":
        return {"op": op, "rows": rows, "cols": _width(rng, 64, 2048, 0.25), "x": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "y": rng.choice(["bf16", "f32", "e4m3", "e4m3"]), "residual": rng.random() < 0.6}
    if op == "norm_back":
        return {"op": op, "rows": rows, "cols": _width(rng, 64, 1024, 0.25), "x": rng.choice(["bf16", "bf16", "f32"]), "dy": "bf16",
                "through": rng.random() < 0.6}
    if op == "pack":
        return {"op": op, "rows": rows, "cols": _width(rng, 64, 2048, 0.25), "x": rng.choice(["bf16", "bf16", "f32"]),
                "act": rng.choice(["none", "crelu", "screlu", "relu"]), "by_column": rng.random() < 0.25}
    n_in, n_out = _width(rng, 64, 2048, 0.1), _width(rng, 16, 2048, 0.1)
    rows = max(1, min(rows, LARGEST // (n_in * n_out)))
    if op == "dense":
        x = rng.choice(["bf16", "bf16", "f16", "e4m3"])
        return {"op": op, "rows": rows, "in": n_in, "out": n_out, "x": x, "y": rng.choice(["f16" if x == "f16" else "bf16", "f32"]) if x != "e4m3" else "bf16",
                "act": rng.choice(["none", "crelu", "screlu", "relu"]), "residual": rng.random() < 0.4}
    act = rng.choice(["none", "crelu", "screlu", "relu"])
    checkpoint = rng.random() < 0.5
    return {"op": op, "rows": rows, "in": n_in, "out": n_out, "x": "e4m3" if checkpoint else "bf16", "dy": "bf16", "saved": "e4m3" if checkpoint else "bf16",
            "dw": "bf16" if act == "screlu" else rng.choice(["bf16", "f32"]), "act": act, "skip": rng.random() < 0.4}


def work(case):
    c, b = case, BYTES
    op, rows = c["op"], c["rows"]
    if op in ("norm", "norm_back", "pack"):
        n = rows * c["cols"]
    else:
        n_in, n_out = c["in"], c["out"]
    if op == "norm":
        moved = n * (b[c["x"]] * (3 if c["residual"] else 1) + b[c["y"]]) + 4 * rows + 4 * c["cols"] + (4 * rows if c["y"] == "e4m3" else 0)
        if c["y"] == "e4m3":
            moved += 2 * n  # the values that the codes stand for, which the pass returns
        return {"bytes": moved, "flops": 6 * n}
    if op == "norm_back":
        return {"bytes": n * (b[c["x"]] * (3 if c["through"] else 2) + b[c["dy"]]) + 4 * rows + 8 * c["cols"], "flops": 10 * n}
    if op == "pack":
        return {"bytes": n * (b[c["x"]] + 1 + 2) + 4 * (c["cols"] if c["by_column"] else rows), "flops": 4 * n}
    if op == "dense":
        moved = b[c["x"]] * (rows * n_in + n_in * n_out) + b[c["y"]] * rows * n_out * (2 if c["residual"] else 1) + 4 * n_out
        if c["x"] == "e4m3":
            moved += 4 * (rows + n_out)
        return {"bytes": moved, "flops": 2 * rows * n_in * n_out}
    moved = 2 * rows * n_out + b[c["x"]] * rows * n_in + 2 * n_in * n_out + b[c["dw"]] * n_in * n_out + 2 * rows * n_in * (2 if c["skip"] else 1) + 4 * n_out
    if c["act"] != "none":
        moved += b[c["saved"]] * rows * n_out
    return {"bytes": moved, "flops": 4 * rows * n_in * n_out}


# ---- inputs


def _activated(v, act):
    """Outputs of an activation: what a layer leaves behind."""
    if act == "crelu":
        return v.clamp_(0, 1)
    if act == "screlu":
        return v.clamp_(0, 1).square_()
    return v.clamp_(min=0) if act == "relu" else v


def _power_of_two(e):
    """2^e in 32 bits, put together from its exponent."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _codes(v, by_column):
    """Codes of 8 bits and their scales, as a program has them from the step before."""
    _, e = torch.frexp(v.abs().amax(0 if by_column else 1))
    scale = _power_of_two(e - 8)
    return (v / (scale if by_column else scale[:, None])).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    c, rows = case, case["rows"]
    s = {"case": dict(case)}
    if c["op"] in ("norm", "norm_back"):
        cols, kind = c["cols"], TYPES[c["x"]]
        spread = torch.exp(0.5 * normal(cols))  # channels of a residual stream differ in size
        s["weight"] = 1 + 0.2 * normal(cols)
        if c["op"] == "norm":
            s["x"] = (normal(rows, cols) * spread).to(kind)
            s["residual"] = normal(rows, cols).mul_(spread).to(kind) if c["residual"] else None
        else:
            total = normal(rows, cols).mul_(spread)
            s["rstd"] = (total.square().mean(1) + EPS).rsqrt()
            s["total"] = total.to(kind)
            s["dy"] = normal(rows, cols).mul_(1e-2).to(TYPES[c["dy"]])
            s["dtotal"] = normal(rows, cols).mul_(1e-2).to(kind) if c["through"] else None
        return s
    if c["op"] == "pack":
        v = normal(rows, c["cols"]).mul_(0.6)
        s["x"] = _activated(v.add_(0.3) if c["act"] in ("crelu", "screlu") else v, c["act"]).to(TYPES[c["x"]])
        return s
    n_in, n_out = c["in"], c["out"]
    w = normal(n_in, n_out).mul_(n_in ** -0.5)
    x = _activated(normal(rows, n_in).mul_(0.6).add_(0.3), "crelu")
    if c["x"] == "e4m3":
        s["x"], s["x_scale"] = _codes(x, False)
    else:
        s["x"] = x.to(TYPES[c["x"]])
    if c["op"] == "dense":
        if c["x"] == "e4m3":
            s["w"], s["w_scale"] = _codes(w, True)
        else:
            s["w"] = w.to(TYPES[c["x"]])
        s["bias"] = 0.1 * normal(n_out)
        s["residual"] = normal(rows, n_out).to(TYPES[c["y"]]) if c["residual"] else None
        return s
    s["w"] = w.to(TYPES[c["dy"]])
    s["dy"] = normal(rows, n_out).mul_(1e-2).to(TYPES[c["dy"]])
    if c["act"] != "none":
        y = _activated(normal(rows, n_out).mul_(0.6).add_(0.3), c["act"])
        if c["saved"] == "e4m3":
            s["y"], s["y_scale"] = _codes(y, False)
        else:
            s["y"] = y.to(TYPES[c["saved"]])
    s["dskip"] = normal(rows, n_in).mul_(1e-2).to(TYPES[c["dy"]]) if c["skip"] else None
    return s


# ---- the plain form


def _plain_act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp(min=0)
    z = z.clamp(0, 1)
    return z * z if act == "screlu" else z


def _plain_scale(v, dim):
    """The smallest power of two that brings the largest magnitude to 448 or below."""
    amax = v.abs().amax(dim, keepdim=True)
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(amax > 0, _power_of_two(e), torch.ones_like(amax))


def _plain_values(v, scale):
    return (v / scale).to(torch.float8_e4m3fn).float() * scale


def _plain_norm(s):
    c = s["case"]
    total = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
    rstd = torch.rsqrt((total * total).mean(1, keepdim=True) + EPS)
    y = total * rstd * s["weight"]
    out = {"rstd": rstd[:, 0]}
    if s["residual"] is not None:
        out["total"] = total.to(s["x"].dtype)
    if c["y"] == "e4m3":
        out["y"] = _plain_values(y, _plain_scale(y, 1)).bfloat16()
    else:
        out["y"] = y.to(TYPES[c["y"]])
    return out


def _plain_norm_back(s):
    n = s["total"].float() * s["rstd"][:, None]
    dy = s["dy"].float()
    g = dy * s["weight"]
    dx = s["rstd"][:, None] * (g - n * (g * n).mean(1, keepdim=True))
    if s["dtotal"] is not None:
        dx = dx + s["dtotal"].float()
    return {"dx": dx.to(s["total"].dtype), "dweight": (dy * n).sum(0)}


def _plain_pack(s):
    c, x = s["case"], s["x"].float()
    scale = _plain_scale(x, 0 if c["by_column"] else 1)
    v = _plain_values(x, scale)
    if c["act"] != "none":
        v = torch.where((x > 0) & (v == 0), scale * 2.0 ** -9, v)
    if c["act"] in ("crelu", "screlu"):
        v = torch.where((x < 1) & (v >= 1), torch.full_like(v, 0.9375), v)
    return {"values": v.bfloat16(), "scale": scale.reshape(-1)}


def _plain_dense(s):
    c = s["case"]
    x, w = s["x"].float(), s["w"].float()
    if c["x"] == "e4m3":
        x, w = x * s["x_scale"][:, None], w * s["w_scale"]
    y = _plain_act(x @ w + s["bias"], c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[c["y"]])


def _plain_dense_back(s):
    c = s["case"]
    x, dz = s["x"].float(), s["dy"].float()
    if c["x"] == "e4m3":
        x = x * s["x_scale"][:, None]
    if c["act"] != "none":
        y = s["y"].float()
        if c["saved"] == "e4m3":
            y = y * s["y_scale"][:, None]
        inside = (y > 0) if c["act"] == "relu" else (y > 0) & (y < 1)
        if c["act"] == "screlu":
            dz = dz * 2 * torch.sqrt(y)
        dz = torch.where(inside, dz, torch.zeros_like(dz))
    dx = dz @ s["w"].float().t()
    if s["dskip"] is not None:
        dx = dx + s["dskip"].float()
    return {"dx": dx.to(s["dy"].dtype), "dw": (x.t() @ dz).to(TYPES[c["dw"]]), "dbias": dz.sum(0)}


PLAIN = {"norm": _plain_norm, "norm_back": _plain_norm_back, "pack": _plain_pack, "dense": _plain_dense, "dense_back": _plain_dense_back}


# ---- the package's operators


def _own(s):
    from bullet_b200 import ops

    c = s["case"]
    if c["op"] == "norm":
        y, total, rstd = ops.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, out_dtype=torch.float8_e4m3fn if c["y"] == "e4m3" else TYPES[c["y"]])
        out = {"rstd": rstd}
        if s["residual"] is not None:
            out["total"] = total
        out["y"] = ops.unpack8(y) if c["y"] == "e4m3" else y
        return out
    if c["op"] == "norm_back":
        dx, dweight = ops.rms_norm_backward(s["dy"], s["total"], s["rstd"], s["weight"], dtotal=s["dtotal"])
        return {"dx": dx, "dweight": dweight}
    if c["op"] == "pack":
        packed = ops.pack8(s["x"], act=ACTS[c["act"]], by_column=c["by_column"])
        return {"values": ops.unpack8(packed), "scale": packed.scale}
    x = ops.Packed8(s["x"], s["x_scale"]) if c["x"] == "e4m3" else s["x"]
    if c["op"] == "dense":
        w = ops.Packed8(s["w"], s["w_scale"], True) if c["x"] == "e4m3" else s["w"]
        return ops.dense(x, w, bias=s["bias"], act=ACTS[c["act"]], residual=s["residual"], out_dtype=TYPES[c["y"]])
    y = None
    if c["act"] != "none":
        y = ops.Packed8(s["y"], s["y_scale"]) if c["saved"] == "e4m3" else s["y"]
    dx, dw, dbias = ops.dense_backward(s["dy"], x, s["w"], y=y, act=ACTS[c["act"]], dskip=s["dskip"], dw_dtype=TYPES[c["dw"]])
    return {"dx": dx, "dw": dw, "dbias": dbias}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---- the definition in 64 bits


def _nearest_e4m3(v):
    """The nearest value of four significand bits, 2^-9 the smallest step, halves to the even one."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _exact_scale(v, dim):
    amax = v.abs().amax(dim, keepdim=True)
    m, e = torch.frexp(amax / 448)  # (a logarithm may be off by its last bit where this is a power of two)
    k = torch.where(m == 0.5, e - 1, e).clamp(min=-126).double()
    return torch.where(amax > 0, torch.exp2(k), torch.ones_like(amax))


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "norm":
        v = s["x"].double()
        out = {}
        if s["residual"] is not None:
            v = v + s["residual"].double()
            out["total"] = v
        r = 1 / torch.sqrt(torch.einsum("ij,ij->i", v, v) / c["cols"] + EPS)
        out["rstd"] = r
        y = torch.einsum("ij,i,j->ij", v, r, s["weight"].double())
        if c["y"] == "e4m3":
            k = _exact_scale(y, 1)
            y = _nearest_e4m3(y / k) * k
        out["y"] = y
        return out
    if c["op"] == "norm_back":
        r, dy = s["rstd"].double(), s["dy"].double()
        n = s["total"].double() * r.unsqueeze(1)
        dot = torch.einsum("ij,j,ij->i", dy, s["weight"].double(), n) / c["cols"]
        dx = (dy * s["weight"].double() - n * dot.unsqueeze(1)) * r.unsqueeze(1)
        if s["dtotal"] is not None:
            dx = dx + s["dtotal"].double()
        return {"dx": dx, "dweight": torch.einsum("ij,ij->j", dy, n)}
    if c["op"] == "pack":
        x = s["x"].double()
        k = _exact_scale(x, 0 if c["by_column"] else 1)
        q = _nearest_e4m3(x / k)
        if c["act"] != "none":
            q[(x > 0) & (q == 0)] = 2.0 ** -9
        if c["act"] in ("crelu", "screlu"):
            v = q * k
            v[(x < 1) & (v >= 1)] = 1 - 2.0 ** -4
            return {"values": v, "scale": k.flatten()}
        return {"values": q * k, "scale": k.flatten()}
    x = s["x"].double()
    if c["x"] == "e4m3":
        x = torch.einsum("ij,i->ij", x, s["x_scale"].double())
    w = s["w"].double()
    if c["op"] == "dense":
        if c["x"] == "e4m3":
            w = torch.einsum("ij,j->ij", w, s["w_scale"].double())
        z = torch.addmm(s["bias"].double(), x, w)
        if c["act"] == "relu":
            z[z < 0] = 0
        elif c["act"] != "none":
            z[z < 0] = 0
            z[z > 1] = 1
            if c["act"] == "screlu":
                z = z.pow(2)
        return z if s["residual"] is None else z + s["residual"].double()
    dz = s["dy"].double()
    if c["act"] != "none":
        y = s["y"].double()
        if c["saved"] == "e4m3":
            y = torch.einsum("ij,i->ij", y, s["y_scale"].double())
        if c["act"] == "screlu":
            dz = dz * y.pow(0.5) * 2
        dz[y <= 0] = 0
        if c["act"] != "relu":
            dz[y >= 1] = 0
    dx = torch.einsum("ij,kj->ik", dz, w)
    if s["dskip"] is not None:
        dx = dx + s["dskip"].double()
    return {"dx": dx, "dw": torch.einsum("ij,ik->jk", x, dz), "dbias": dz.sum(0)}
