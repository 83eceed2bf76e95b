"""The operators of a graph layer beside the sparse product, as measurable cases.

A pre-norm residual layer is ``C = A . y``; ``y, h = rms_norm(C, w, residual=h)``; ``y = linear(y, W, b, act, residual)``.
``listed()`` names twelve cases over the range of these operators and ``draw(rng)`` gives further ones.  Where ``own`` is
false, ``run`` computes them from elementary torch operations in 32 bits; where it is true, through this package.

Operations (``case["op"]``):
  norm         y = rms_norm(x, w, residual), and h = x + residual
  norm8        the same with y in 8 bits (e4m3) and one scale a row, what the 8-bit product reads
  norm_grad    gradients of x (and the residual) and of w, with the gradient that comes down the residual stream
  linear       y = act(x W^T + b) + residual
  linear8      the same of 8-bit rows with scales (e4m3 or int8)
  linear_grad  gradients of x, W and b
Feature sizes of graph layers and row counts are those of the package's benchmark workloads; the others are generic.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}
TOP8 = {"e4m3": 448.0, "int8": 127.0}


def listed():
    return [
        # one row of features being served, the smallest call: what a launch costs
        {"name": "norm8_1_4096", "op": "norm8", "rows": 1, "dim": 4096, "x": "bf16", "res": "bf16", "pad": 0},
        # the aggregated features of a citation graph (an f32 product) added to its residual stream
        {"name": "norm_170k_128", "op": "norm", "rows": 170_000, "dim": 128, "x": "f32", "res": "f32", "pad": 0},
        # the input of a large 8-bit product
        {"name": "norm8_16k_4096", "op": "norm8", "rows": 16_384, "dim": 4096, "x": "bf16", "res": "bf16", "pad": 0},
        # a training step of a graph layer with an odd number of features, in the rows of a wider buffer
        {"name": "norm_grad_5003_1001", "op": "norm_grad", "rows": 5003, "dim": 1001, "x": "f16", "pad": 24},
        # ... and of a wide model
        {"name": "norm_grad_32k_2048", "op": "norm_grad", "rows": 32_768, "dim": 2048, "x": "bf16", "pad": 0},
        # one row being served: the weight is read once
        {"name": "linear_1_4096", "op": "linear", "rows": 1, "k": 4096, "n": 4096, "x": "bf16", "act": "gelu", "res": True, "pad": 0},
        # the transform of a citation graph's features
        {"name": "linear_170k_128_256", "op": "linear", "rows": 170_000, "k": 128, "n": 256, "x": "f32", "act": "relu", "res": True, "pad": 0},
        # a large dense product
        {"name": "linear_8k_8k_8k", "op": "linear", "rows": 8192, "k": 8192, "n": 8192, "x": "bf16", "act": "silu", "res": True, "pad": 0},
        # a few rows being served in 8 bits, with sizes that fit no tile
        {"name": "linear8_13_4000_1001", "op": "linear8", "rows": 13, "k": 4000, "n": 1001, "x": "int8", "act": "none", "res": False, "pad": 0},
        # the product that reads the norm's 8-bit output
        {"name": "linear8_16k_4k_4k", "op": "linear8", "rows": 16_384, "k": 4096, "n": 4096, "x": "e4m3", "act": "gelu", "res": True, "pad": 0},
        # the last layer of a graph network, 47 classes, being trained
        {"name": "linear_grad_57k_100_47", "op": "linear_grad", "rows": 57_001, "k": 100, "n": 47, "x": "f32", "act": "none", "pad": 0},
        # a wide layer being trained
        {"name": "linear_grad_8k_4k_4k", "op": "linear_grad", "rows": 8192, "k": 4096, "n": 4096, "x": "bf16", "act": "gelu", "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of lo .. hi, two in three of them multiples of 16."""
    v = _log(rng, lo, hi)
    return max(16, v // 16 * 16) if v >= 16 and rng.random() < 0.67 else v


def draw(rng):
    op = rng.choice(("norm", "norm8", "norm_grad", "linear", "linear", "linear8", "linear_grad", "linear_grad"))
    x = rng.choice(("f32", "bf16", "bf16", "f16"))
    pad = rng.choice((0, 0, 0, 8, 24, 5))
    if op.startswith("norm"):
        dim = _size(rng, 16, 16_384)
        rows = _log(rng, 1, min(170_000, (1 << 24) // dim))
        case = {"op": op, "rows": rows, "dim": dim, "x": x, "pad": pad}
        if op != "norm_grad":
            case["res"] = rng.choice(("none", "f32", "bf16")) if x == "f32" else rng.choice(("none", "f32", x))
        return case
    k, n = _size(rng, 16, 8192), _size(rng, 16, 8192)
    if op == "linear8":
        x = rng.choice(("e4m3", "e4m3", "int8"))
    most = {"linear": 1.2e11 if x == "f32" else 1e12, "linear8": 5e11, "linear_grad": 5e10 if x == "f32" else 4e11}[op]
    rows = _log(rng, 1, max(1, min(170_000, int(most / (2 * k * n)), int(6e7 / max(k, n)))))
    case = {"op": op, "rows": rows, "k": k, "n": n, "x": x, "act": rng.choice(("none", "relu", "gelu", "silu")), "pad": pad}
    if op != "linear_grad":
        case["res"] = rng.random() < 0.5
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


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, pad, dt = case["op"], case["rows"], case["pad"], DTYPES[case["x"]]
    s = {"case": case}
    if op.startswith("norm"):
        dim = case["dim"]
        s["x"] = _normal((rows, dim), dt, gen, 2.0, pad)
        # a learned weight: around one
        s["w"] = (1.0 + 0.2 * torch.randn(dim, device="cuda", generator=gen)).to(dt)
        if op == "norm_grad":
            s["dy"], s["dh"] = _normal((rows, dim), dt, gen, 0.1), _normal((rows, dim), dt, gen, 0.1)
        else:
            s["res"] = None if case["res"] == "none" else _normal((rows, dim), DTYPES[case["res"]], gen, 3.0)
        return s
    k, n = case["k"], case["n"]
    y = torch.bfloat16 if op == "linear8" else dt
    if op == "linear8":
        s["x"], s["sx"] = _rows8((rows, k), case["x"], gen, 1.0, pad)
        s["w"], s["sw"] = _rows8((n, k), case["x"], gen, k ** -0.5)
    else:
        s["x"] = _normal((rows, k), dt, gen, 1.0, pad)
        s["w"] = _normal((n, k), dt, gen, k ** -0.5)
    s["b"] = _normal((n,), y, gen, 0.1)
    if op == "linear_grad":
        s["dy"] = _normal((rows, n), dt, gen, 0.1)
        s["z"] = None if case["act"] == "none" else _normal((rows, n), dt, gen, 1.0)
    else:
        s["res"] = _normal((rows, n), y, gen) if case["res"] else None
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
    if op == "norm":
        out = lo.rms_norm(s["x"], s["w"], residual=s["res"], eps=EPS, out_dtype=DTYPES[_y_type(case)])
        return {"y": out} if s["res"] is None else {"y": out[0], "h": out[1]}
    if op == "norm8":
        out = lo.rms_norm_8bit(s["x"], s["w"], residual=s["res"], eps=EPS, dtype=torch.float8_e4m3fn)
        return dict(zip(("q", "scale", "h"), out))
    if op == "norm_grad":
        return dict(zip(("dx", "dw"), lo.rms_norm_grad(s["dy"], s["x"], s["w"], eps=EPS, dh=s["dh"])))
    if op == "linear":
        return lo.linear(s["x"], s["w"], s["b"], activation=act, residual=s["res"])
    if op == "linear8":
        return lo.linear_8bit(s["x"], s["sx"], s["w"], s["sw"], s["b"], activation=act, residual=s["res"], out_dtype=torch.bfloat16)
    return dict(zip(("dx", "dw", "db"), lo.linear_grad(s["dy"], s["x"], s["w"], z=s["z"], activation=act, bias_dtype=s["b"].dtype)))


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * torch.sigmoid(z) if act == "silu" else z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    sig = torch.sigmoid(z)
    return sig * (1.0 + z * (1.0 - sig))


def _plain(s, case, op, dt):
    f = torch.float32
    if op in ("norm", "norm8"):
        h = s["x"].to(f) if s["res"] is None else s["x"].to(f) + s["res"].to(f)
        y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["w"].to(f)
        out = {} if s["res"] is None else {"h": h.to(s["res"].dtype)}
        if op == "norm":
            out["y"] = y.to(DTYPES[_y_type(case)])
        else:
            out["scale"] = y.abs().amax(dim=1) / TOP8["e4m3"]
            out["q"] = (y / out["scale"][:, None]).to(torch.float8_e4m3fn)
        return out
    if op == "norm_grad":
        h, dy, w = s["x"].to(f), s["dy"].to(f), s["w"].to(f)
        r = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS)
        g = dy * w
        dx = r * (g - h * (g * h).mean(dim=1, keepdim=True) * r * r) + s["dh"].to(f)
        return {"dx": dx.to(dt), "dw": (dy * h * r).sum(dim=0).to(dt)}
    if op in ("linear", "linear8"):
        z = s["x"].to(f) @ s["w"].to(f).t()
        if op == "linear8":
            z = z * s["sx"][:, None] * s["sw"]
        y = _act(z + s["b"].to(f), case["act"])
        return (y if s["res"] is None else y + s["res"].to(f)).to(s["b"].dtype)
    dz = s["dy"].to(f)
    if s["z"] is not None:
        dz = dz * _act_grad(s["z"].to(f), case["act"])
    return {"dx": (dz @ s["w"].to(f)).to(dt), "dw": (dz.t() @ s["x"].to(f)).to(dt), "db": dz.sum(dim=0).to(s["b"].dtype)}


# ---------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    op, m, e = case["op"], case["rows"], SIZE[case["x"]]
    if op.startswith("norm"):
        d = case["dim"]
        if op == "norm_grad":
            return {"bytes": 4 * m * d * e + 2 * d * e, "flops": 12.0 * m * d}
        r = SIZE.get(case["res"], 0)
        y = 1 if op == "norm8" else SIZE[_y_type(case)]
        return {"bytes": m * d * (e + 2 * r + y) + d * e + (4 * m if op == "norm8" else 0), "flops": 6.0 * m * d}
    k, n = case["k"], case["n"]
    if op == "linear_grad":
        z = 0 if case["act"] == "none" else m * n * e
        return {"bytes": e * (2 * m * k + 2 * n * k + m * n + n) + z, "flops": 4.0 * m * n * k}
    y = 2 if op == "linear8" else e
    scales = 4 * (m + n) if op == "linear8" else 0
    return {"bytes": e * (m * k + n * k) + y * (m * n * (2 if case["res"] else 1) + n) + scales, "flops": 2.0 * m * n * k}


# ---------------------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    d = {key: v.double() for key, v in s.items() if isinstance(v, torch.Tensor)}
    op = case["op"]
    if op.startswith("norm"):
        h = d["x"] + d["res"] if "res" in d else d["x"]
        size = h.shape[1]
        inv = 1.0 / torch.sqrt(torch.linalg.vecdot(h, h) / size + EPS)
        if op == "norm_grad":
            # y_j = w_j h_j inv:  dy_j / dh_i = w_j (delta_ij inv - h_j h_i inv^3 / size)
            along = torch.linalg.vecdot(d["dy"] * d["w"], h) * inv.pow(3) / size
            return {"dx": torch.addcmul(d["dh"], d["dy"] * d["w"], inv[:, None]) - h * along[:, None],
                    "dw": torch.einsum("mj,mj,m->j", d["dy"], h, inv)}
        out = {"h": h} if "res" in d else {}
        if op == "norm":
            return {**out, "y": torch.einsum("mj,m,j->mj", h, inv, d["w"])}
        t = h * d["w"]
        top = t.abs().max(dim=1).values
        return {**out, "scale": top * inv / 448.0, "q": (t * (448.0 / top)[:, None]).to(torch.float8_e4m3fn).double()}
    z = d["z"] if "z" in d else None
    if op == "linear_grad":
        dz = d["dy"]
        if case["act"] == "relu":
            dz = torch.where(z > 0, dz, 0.0)
        elif case["act"] == "gelu":
            dz = dz * (torch.special.ndtr(z) + z * torch.exp(-z * z / 2) * (2 * math.pi) ** -0.5)
        elif case["act"] == "silu":
            e = torch.exp(-z)
            dz = dz * (1 + e + z * e) / (1 + e).square()
        return {"dx": torch.mm(dz, d["w"]), "dw": torch.mm(dz.t(), d["x"]), "db": torch.mv(dz.t(), torch.ones_like(dz[:, 0]))}
    if op == "linear8":
        z = torch.addmm(d["b"], d["x"] * d["sx"][:, None], (d["w"] * d["sw"][:, None]).t())
    else:
        z = torch.addmm(d["b"], d["x"], d["w"].t())
    if case["act"] == "relu":
        z = torch.where(z > 0, z, 0.0)
    elif case["act"] == "gelu":
        z = z * torch.special.ndtr(z)
    elif case["act"] == "silu":
        z = z / (1 + torch.exp(-z))
    return z + d["res"] if "res" in d else z
