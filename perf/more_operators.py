"""What training a graph network from node ids takes beside the graph layer's first operators, as measurable cases.

A stack is ``y = embedding(ids, W, scale)``; then in each layer ``C = A . y``; ``n, h = layer_norm(C, w, b, residual=h)``;
``y = linear(gated_linear(n, W2, b2), W1, b1)``; a step ends with ``clip_gradients`` over the gradients of all parameters.
``listed()`` names twelve cases over the range of these operators and ``draw(rng)`` gives further ones.  Where ``own`` is false,
``run`` computes them from elementary torch operations; where it is true, through this package.

Operations (``case["op"]``):
  layer_norm       h = x + residual; y = (h - mean) / sqrt(var + eps) w + b
  layer_norm_grad  gradients of x (and the residual), w and b, with the gradient that comes down the residual stream
  gated            z = x W^T + b for W of 2 n rows; y = act(z[:, :n]) z[:, n:]; with ``keep`` z too, as a training step needs it
  gated8           the same of 8-bit rows with scales (e4m3 or int8)
  gated_grad       gradients of x, W and b
  embedding        rows of W by id, times a scale; an id outside of W (padding is -1) gives a row of zeros
  embedding_grad   its gradient of W: sums of the rows of dy by id
  clip             norm of all gradients, and each of them times min(1, most / (norm + eps))
Feature sizes and row counts of graphs are those of the package's benchmark workloads; the others are generic.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
CLIP_EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}
TOP8 = {"e4m3": 448.0, "int8": 127.0}


def listed():
    return [
        # one row of features being served, the smallest call: what a launch costs
        {"name": "layer_norm_1_4096", "op": "layer_norm", "rows": 1, "dim": 4096, "x": "bf16", "res": "bf16", "pad": 0},
        # the aggregated features of a citation graph (an f32 product) added to its residual stream
        {"name": "layer_norm_170k_128", "op": "layer_norm", "rows": 170_000, "dim": 128, "x": "f32", "res": "f32", "pad": 0},
        # a training step of a wide model, two weight gradients to reduce
        {"name": "layer_norm_grad_32k_2048", "op": "layer_norm_grad", "rows": 32_768, "dim": 2048, "x": "bf16", "pad": 0},
        # one row being served: both projections are read once
        {"name": "gated_1_4096_8192", "op": "gated", "rows": 1, "k": 4096, "n": 8192, "x": "bf16", "act": "silu", "keep": False, "pad": 0},
        # the forward half of a wide block's training step
        {"name": "gated_8k_4k_8k", "op": "gated", "rows": 8192, "k": 4096, "n": 8192, "x": "bf16", "act": "silu", "keep": True, "pad": 0},
        # a batch of rows served in 8 bits, with sizes that fit no tile
        {"name": "gated8_4001_4000_1001", "op": "gated8", "rows": 4001, "k": 4000, "n": 1001, "x": "e4m3", "act": "gelu", "keep": False, "pad": 0},
        # a narrow float32 block over the nodes of a small graph, being trained
        {"name": "gated_grad_57k_100_200", "op": "gated_grad", "rows": 57_001, "k": 100, "n": 200, "x": "f32", "act": "gelu", "pad": 0},
        # a wide block being trained
        {"name": "gated_grad_8k_4k_4k", "op": "gated_grad", "rows": 8192, "k": 4096, "n": 4096, "x": "bf16", "act": "silu", "pad": 0},
        # the features of the nodes of a sampled batch, some of it padding, out of the table of a large graph
        {"name": "embedding_57k_of_2450k_128", "op": "embedding", "ids": 57_001, "rows": 2_450_000, "dim": 128, "x": "f16", "spread": "even", "padding": 0.1, "pad": 0},
        # the table of a vocabulary being trained: few ids are most of the batch
        {"name": "embedding_grad_16k_of_32k_4096", "op": "embedding_grad", "ids": 16_384, "rows": 32_000, "dim": 4096, "x": "bf16", "spread": "zipf", "padding": 0.0, "pad": 0},
        # the gradients of a small stack of graph layers: latency
        {"name": "clip_3_layers_128", "op": "clip", "layers": 3, "dim": 128, "x": "f32", "size": 0.5},
        # ... and of a large one
        {"name": "clip_8_layers_4096", "op": "clip", "layers": 8, "dim": 4096, "x": "bf16", "size": 20.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of lo .. hi, two in three of them multiples of 16."""
    v = _log(rng, lo, hi)
    return max(16, v // 16 * 16) if v >= 16 and rng.random() < 0.67 else v


def draw(rng):
    op = rng.choice(("layer_norm", "layer_norm_grad", "gated", "gated", "gated8", "gated_grad", "gated_grad", "embedding", "embedding_grad", "embedding_grad", "clip"))
    x = rng.choice(("f32", "bf16", "bf16", "f16"))
    pad = rng.choice((0, 0, 0, 8, 24, 5))
    if op.startswith("layer_norm"):
        dim = _size(rng, 16, 16_384)
        rows = _log(rng, 1, min(170_000, (1 << 24) // dim))
        case = {"op": op, "rows": rows, "dim": dim, "x": x, "pad": pad}
        if op == "layer_norm":
            case["res"] = rng.choice(("none", "f32", "bf16")) if x == "f32" else rng.choice(("none", "f32", x))
        return case
    if op.startswith("embedding"):
        dim = _size(rng, 16, 4096)
        rows = _log(rng, 47, min(2_450_000, (1 << 27) // dim))
        ids = _log(rng, 1, min(1_000_000, (1 << 26) // dim))
        return {"op": op, "ids": ids, "rows": rows, "dim": dim, "x": x, "spread": rng.choice(("even", "zipf")), "padding": rng.choice((0.0, 0.0, 0.2)), "pad": pad}
    if op == "clip":
        dim = _size(rng, 47, 4096)
        layers = _log(rng, 1, min(64, max(1, (1 << 27) // (3 * dim * dim))))
        return {"op": op, "layers": layers, "dim": dim, "x": x, "size": rng.choice((0.1, 0.5, 20.0))}
    k, n = _size(rng, 16, 8192), _size(rng, 16, 8192)
    if op == "gated8":
        x = rng.choice(("e4m3", "e4m3", "int8"))
    most = {"gated": 6e10 if x == "f32" else 1e12, "gated8": 5e11, "gated_grad": 5e10 if x == "f32" else 4e11}[op]
    rows = _log(rng, 1, max(1, min(170_000, int(most / (4 * k * n)), int(6e7 / max(k, 2 * n)))))
    case = {"op": op, "rows": rows, "k": k, "n": n, "x": x, "act": rng.choice(("none", "relu", "gelu", "silu")), "pad": pad}
    if op != "gated_grad":
        case["keep"] = op == "gated" and rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------- inputs


def _normal(shape, dtype, gen, scale=1.0, pad=0):
    """Normal values; with `pad`, the first columns of a buffer that is so much wider."""
    t = torch.randn((*shape[:-1], shape[-1] + pad), device="cuda", generator=gen).mul_(scale).to(dtype)
    return t[..., :shape[-1]] if pad else t


def _rows8(shape, name, gen, scale, pad=0):
    """Normal rows in 8 bits with a scale each."""
    t = torch.randn(shape, device="cuda", generator=gen).mul_(scale)
    s = t.abs().amax(dim=1) / TOP8[name]
    t = t / s[:, None]
    q = t.round().to(torch.int8) if name == "int8" else t.to(DTYPES[name])
    if pad:
        wide = torch.zeros((shape[0], shape[1] + pad), device="cuda", dtype=q.dtype)
        wide[:, :shape[1]] = q
        q = wide[:, :shape[1]]
    return q, s


def _ids(case, gen):
    """Node ids of a batch: evenly out of the table, or the v-th with a probability of about 1 / v; some of them -1, which is padding."""
    u = torch.rand(case["ids"], device="cuda", generator=gen, dtype=torch.float64)
    v = u * case["rows"] if case["spread"] == "even" else torch.pow(float(case["rows"]), u) - 1.0
    v = v.long().clamp_(0, case["rows"] - 1)
    if case["padding"]:
        v[torch.rand(case["ids"], device="cuda", generator=gen) < case["padding"]] = -1
    return v


def _clip_shapes(case):
    """The parameters of a layer: a norm's weight and bias, a gated block's projections and biases, all of `dim` features."""
    d = case["dim"]
    return [(d,), (d,), (2 * d, d), (2 * d,), (d, d), (d,)] * case["layers"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], DTYPES[case["x"]]
    s = {"case": case}
    if op == "clip":
        shapes = _clip_shapes(case)
        total = math.sqrt(sum(math.prod(t) for t in shapes))
        # gradients of a norm of about `size`, which is to be 1 at most
        s["grads"] = [_normal(t, dt, gen, case["size"] / total) for t in shapes]
        return s
    pad, rows = case["pad"], case["rows"]
    if op.startswith("embedding"):
        s["ids"] = _ids(case, gen)
        if op == "embedding":
            s["w"] = _normal((rows, case["dim"]), dt, gen, 0.05, pad)
        else:
            s["dy"] = _normal((case["ids"], case["dim"]), dt, gen, 0.1, pad)
        s["scale"] = math.sqrt(case["dim"])
        return s
    if op.startswith("layer_norm"):
        dim = case["dim"]
        # aggregated features, which need not be centred
        s["x"] = _normal((rows, dim), dt, gen, 2.0, pad).add_(0.5)
        s["w"] = (1.0 + 0.2 * torch.randn(dim, device="cuda", generator=gen)).to(dt)
        if op == "layer_norm_grad":
            s["dy"], s["dh"] = _normal((rows, dim), dt, gen, 0.1), _normal((rows, dim), dt, gen, 0.1)
        else:
            s["b"] = _normal((dim,), dt, gen, 0.1)
            s["res"] = None if case["res"] == "none" else _normal((rows, dim), DTYPES[case["res"]], gen, 3.0)
        return s
    k, n = case["k"], case["n"]
    y = torch.bfloat16 if op == "gated8" else dt
    if op == "gated8":
        s["x"], s["sx"] = _rows8((rows, k), case["x"], gen, 1.0, pad)
        s["w"], s["sw"] = _rows8((2 * n, k), case["x"], gen, k ** -0.5)
    else:
        s["x"] = _normal((rows, k), dt, gen, 1.0, pad)
        s["w"] = _normal((2 * n, k), dt, gen, k ** -0.5)
    if op == "gated_grad":
        s["dy"], s["z"] = _normal((rows, n), dt, gen, 0.1), _normal((rows, 2 * n), dt, gen, 1.0)
    else:
        s["b"] = _normal((2 * n,), y, gen, 0.1)
    return s


# ---------------------------------------------------------------------------- one pass


def run(s):
    case = s["case"]
    return (_own if own else _plain)(s, case, case["op"], DTYPES[case["x"]])


def _y_type(case):
    """The norm's output is what the next product reads: the narrower of the two types that it adds."""
    return case["res"] if SIZE.get(case["res"], 8) < SIZE[case["x"]] else case["x"]


def _own(s, case, op, dt):
    from liteform_ae_amd import layer_ops as lo
    act = None if case.get("act", "none") == "none" else case["act"]
    if op == "layer_norm":
        out = lo.layer_norm(s["x"], s["w"], s["b"], residual=s["res"], eps=EPS, out_dtype=DTYPES[_y_type(case)])
        return {"y": out} if s["res"] is None else {"y": out[0], "h": out[1]}
    if op == "layer_norm_grad":
        return dict(zip(("dx", "dw", "db"), lo.layer_norm_grad(s["dy"], s["x"], s["w"], eps=EPS, dh=s["dh"], bias_dtype=dt)))
    if op == "gated":
        out = lo.gated_linear(s["x"], s["w"], s["b"], activation=act, return_preactivation=case["keep"])
        return {"y": out[0], "z": out[1]} if case["keep"] else {"y": out}
    if op == "gated8":
        return {"y": lo.gated_linear_8bit(s["x"], s["sx"], s["w"], s["sw"], s["b"], activation=act, out_dtype=torch.bfloat16)}
    if op == "gated_grad":
        return dict(zip(("dx", "dw", "db"), lo.gated_linear_grad(s["dy"], s["x"], s["w"], s["z"], activation=act, bias_dtype=dt)))
    if op == "embedding":
        return {"y": lo.embedding(s["ids"], s["w"], scale=s["scale"])}
    if op == "embedding_grad":
        return {"dw": lo.embedding_grad(s["dy"], s["ids"], case["rows"], scale=s["scale"])}
    clipped, norm = lo.clip_gradients(s["grads"], 1.0, eps=CLIP_EPS)
    return {"grads": clipped, "norm": norm}


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    return z * torch.sigmoid(z) if act == "silu" else z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "silu":
        return torch.sigmoid(z) * (1.0 + z * torch.sigmoid(-z))
    return torch.ones_like(z)


def _plain(s, case, op, dt):
    f = torch.float32
    if op == "layer_norm":
        h = s["x"].to(f) if s["res"] is None else s["x"].to(f) + s["res"].to(f)
        c = h - h.mean(dim=1, keepdim=True)
        y = c * torch.rsqrt(c.square().mean(dim=1, keepdim=True) + EPS) * s["w"].to(f) + s["b"].to(f)
        y = y.to(DTYPES[_y_type(case)])
        return {"y": y} if s["res"] is None else {"y": y, "h": h.to(s["res"].dtype)}
    if op == "layer_norm_grad":
        h, dy = s["x"].to(f), s["dy"].to(f)
        c = h - h.mean(dim=1, keepdim=True)
        r = torch.rsqrt(c.square().mean(dim=1, keepdim=True) + EPS)
        t, g = c * r, dy * s["w"].to(f)
        dx = r * (g - g.mean(dim=1, keepdim=True) - t * (g * t).mean(dim=1, keepdim=True)) + s["dh"].to(f)
        return {"dx": dx.to(dt), "dw": (dy * t).sum(dim=0).to(dt), "db": dy.sum(dim=0).to(dt)}
    if op in ("gated", "gated8"):
        n = case["n"]
        z = s["x"].to(f) @ s["w"].to(f).t()
        if op == "gated8":
            z = z * s["sx"][:, None] * s["sw"]
        z = z + s["b"].to(f)
        y = (_act(z[:, :n], case["act"]) * z[:, n:]).to(s["b"].dtype)
        return {"y": y, "z": z.to(dt)} if case["keep"] else {"y": y}
    if op == "gated_grad":
        n, dy, z = case["n"], s["dy"].to(f), s["z"].to(f)
        dz = torch.cat([dy * z[:, n:] * _act_grad(z[:, :n], case["act"]), dy * _act(z[:, :n], case["act"])], dim=1)
        return {"dx": (dz @ s["w"].to(f)).to(dt), "dw": (dz.t() @ s["x"].to(f)).to(dt), "db": dz.sum(dim=0).to(dt)}
    if op == "embedding":
        ids = s["ids"]
        y = s["w"][ids.clamp_min(0)].to(f) * s["scale"]
        return {"y": torch.where((ids >= 0)[:, None], y, 0.0).to(dt)}
    if op == "embedding_grad":
        # (in 64 bits: one id may have most of the rows)
        ids = s["ids"]
        dw = torch.zeros((case["rows"] + 1, case["dim"]), device="cuda", dtype=torch.float64)
        dw.index_add_(0, torch.where(ids >= 0, ids, case["rows"]), s["dy"].double() * s["scale"])
        return {"dw": dw[:case["rows"]].to(dt)}
    norm = torch.stack([g.to(f).square().sum() for g in s["grads"]]).sum().sqrt()
    factor = (1.0 / (norm + CLIP_EPS)).clamp_max(1.0)
    return {"grads": [(g.to(f) * factor).to(dt) for g in s["grads"]], "norm": norm}


# ---------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    op, e = case["op"], SIZE[case["x"]]
    if op == "clip":
        size = sum(math.prod(t) for t in _clip_shapes(case))
        return {"bytes": 2 * size * e + 4, "flops": 3.0 * size}
    m = case["rows"]
    if op == "embedding":
        # a row that is asked for twice is read once
        return {"bytes": case["ids"] * (8 + case["dim"] * e) + min(case["ids"], m) * case["dim"] * e, "flops": 1.0 * case["ids"] * case["dim"]}
    if op == "embedding_grad":
        return {"bytes": case["ids"] * (8 + case["dim"] * e) + m * case["dim"] * e, "flops": 1.0 * case["ids"] * case["dim"]}
    if op.startswith("layer_norm"):
        d = case["dim"]
        if op == "layer_norm_grad":
            return {"bytes": 4 * m * d * e + 3 * d * e, "flops": 16.0 * m * d}
        r = SIZE.get(case["res"], 0)
        return {"bytes": m * d * (e + 2 * r + SIZE[_y_type(case)]) + 2 * d * e, "flops": 9.0 * m * d}
    k, n = case["k"], case["n"]
    if op == "gated_grad":
        return {"bytes": e * (2 * m * k + 4 * n * k + 3 * m * n + 2 * n), "flops": 8.0 * m * n * k}
    y = 2 if op == "gated8" else e
    scales = 4 * (m + 2 * n) if op == "gated8" else 0
    return {"bytes": e * (m * k + 2 * n * k) + y * (m * n * (3 if case["keep"] else 1) + 2 * n) + scales, "flops": 4.0 * m * n * k}


# ---------------------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        d = [g.double() for g in s["grads"]]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g) for g in d]))
        return {"grads": [g * min(1.0, 1.0 / (float(norm) + CLIP_EPS)) for g in d], "norm": norm}
    if op == "embedding":
        table = torch.cat([s["w"], torch.zeros_like(s["w"][:1])])               # id -1 takes the last row
        return {"y": torch.index_select(table, 0, s["ids"] % len(table)).double() * s["scale"]}
    if op == "embedding_grad":
        order = torch.argsort(s["ids"], stable=True)
        order = order[s["ids"][order] >= 0]
        dw = torch.zeros((case["rows"], case["dim"]), device="cuda", dtype=torch.float64)
        dw.index_put_((s["ids"][order],), s["dy"][order].double(), accumulate=True)
        return {"dw": dw.mul_(s["scale"])}
    d = {key: v.double() for key, v in s.items() if isinstance(v, torch.Tensor)}
    if op.startswith("layer_norm"):
        h = d["x"] + d["res"] if "res" in d else d["x"]
        var, mean = torch.var_mean(h, dim=1, correction=0)
        inv = 1.0 / torch.sqrt(var + EPS)
        t = torch.addcmul(-(mean * inv)[:, None], h, inv[:, None])
        if op == "layer_norm":
            out = {"y": torch.addcmul(d["b"], t, d["w"])}
            return {**out, "h": h} if "res" in d else out
        # y_j = w_j t_j + b_j:  dt_j / dh_i = inv (delta_ij - 1 / size - t_i t_j / size)
        size = h.shape[1]
        one = torch.mv(d["dy"], d["w"]) / size
        along = torch.linalg.vecdot(d["dy"] * d["w"], t) / size
        dx = d["dh"] + inv[:, None] * (d["dy"] * d["w"] - one[:, None] - t * along[:, None])
        return {"dx": dx, "dw": torch.einsum("mj,mj->j", d["dy"], t), "db": torch.mv(d["dy"].t(), torch.ones_like(one))}
    n, act = case["n"], case["act"]

    def phi(g):
        return torch.special.ndtr(g)

    if op == "gated_grad":
        g, u = d["z"][:, :n], d["z"][:, n:]
        if act == "relu":
            a, da = torch.where(g > 0, g, 0.0), torch.where(g > 0, 1.0, 0.0)
        elif act == "gelu":
            a, da = g * phi(g), phi(g) + g * torch.exp(-g * g / 2) * (2 * math.pi) ** -0.5
        elif act == "silu":
            e = torch.exp(-g)
            a, da = g / (1 + e), (1 + e + g * e) / (1 + e).square()
        else:
            a, da = g, torch.ones_like(g)
        dg, du = d["dy"] * u * da, d["dy"] * a
        ones = torch.ones_like(dg[:, 0])
        return {"dx": torch.addmm(torch.mm(dg, d["w"][:n]), du, d["w"][n:]), "dw": torch.cat([torch.mm(dg.t(), d["x"]), torch.mm(du.t(), d["x"])]),
                "db": torch.cat([torch.mv(dg.t(), ones), torch.mv(du.t(), ones)])}
    x, w = d["x"], d["w"]
    if op == "gated8":
        x, w = x * d["sx"][:, None], w * d["sw"][:, None]
    g, u = torch.addmm(d["b"][:n], x, w[:n].t()), torch.addmm(d["b"][n:], x, w[n:].t())
    out = {"z": torch.cat([g, u], dim=1)} if case["keep"] else {}
    if act == "relu":
        g = torch.where(g > 0, g, 0.0)
    elif act == "gelu":
        g = g * phi(g)
    elif act == "silu":
        g = g / (1 + torch.exp(-g))
    return {**out, "y": g * u}
