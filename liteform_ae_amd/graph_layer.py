"""A graph layer from the package's operators: aggregation with a composed hyb format, norm with the residual stream's addition,
dense transform - forward, in 8 bits, and a training step.

    h, y <- rms_norm(A . y + h) * w;   y <- act(y W^T + b)                                        GraphLayer
    h, n <- layer_norm(A . y + h);     y <- (act(n Wg^T + bg) * (n Wu^T + bu)) Wd^T + bd          GatedLayer
    y <- table[id] * scale                                                                        NodeEmbedding, before the first layer

    python -m liteform_ae_amd.graph_layer --synthetic cfg2 --feat 128 --layers 2 --steps 5
    python -m liteform_ae_amd.graph_layer --synthetic cfg2 --feat 128 --layers 2 --steps 5 --gated --embedding --max-norm 1e-3 --rate 5

train a stack of such layers on a synthetic graph against random targets, serve the result in 16 and 8 bits and print the losses and
times.  The reference ends with the sparse product (proc05.spmm.end-to-end.py:127-190) and has no counterpart.
"""
from __future__ import annotations

import argparse
import time

from . import format_algos as fa
from . import layer_ops as lo
from .format_matrix_market import MTX


class Aggregation:
    """C = A . y and its gradient dy = A^T . dC, both with plans that are composed once.  y is float32 or bfloat16, C float32."""

    def __init__(self, g, feat_size: int, b_dtype: str = "f32"):
        torch = fa._torch()
        self.dtype = torch.float32 if b_dtype == "f32" else torch.bfloat16
        self._forward = self._plan(g, feat_size, b_dtype)
        coo = g.coo_mtx
        self._backward = self._plan(MTX.from_coo(coo.col, coo.row, (coo.shape[1], coo.shape[0]), data=coo.data), feat_size, b_dtype)

    @staticmethod
    def _plan(g, feat_size, b_dtype):
        parts, windows = fa.predict_launch_shape(g, feat_size, b_dtype)
        widths = fa.search_bucket_config(g, parts, fa.CostModelSettings(feat_size, parts, cost_model="gfx950"))
        return fa.HybSpMM(fa.build_hyb_format_device(g, widths), feat_size, b_dtype, windows=windows)

    def forward(self, y):
        lo.refuse_graph("y", y)
        return self._forward.run(y if y.dtype is self.dtype else y.to(self.dtype))

    def backward(self, dC):
        lo.refuse_graph("dC", dC)
        return self._backward.run(dC if dC.dtype is self.dtype else dC.to(self.dtype))


def _take(mine, kept):
    """What a call of ``forward`` kept: the latest that no ``backward`` has had yet, unless the caller names one."""
    if kept is None:
        if not mine:
            raise RuntimeError("no forward(keep=True) since the last update is left to take gradients of")
        kept = mine.pop()
    return kept


class GraphLayer:
    """One layer with its parameters, in float32 or bfloat16.  ``backward`` returns the gradients of a call of ``forward`` that kept what they need;
    torch builds no graph through a layer, and one is called under ``torch.no_grad()`` where tensors require gradients."""

    def __init__(self, aggregation: Aggregation, feat_size: int, activation: str = "gelu", dtype=None, generator=None, eps: float = 1e-6):
        torch = fa._torch()
        dtype = torch.float32 if dtype is None else dtype
        self.aggregation, self.activation, self.eps = aggregation, activation, eps
        self.norm = torch.ones(feat_size, dtype=dtype, device="cuda")
        self.weight = (torch.randn((feat_size, feat_size), device="cuda", generator=generator) * feat_size ** -0.5).to(dtype)
        self.bias = torch.zeros(feat_size, dtype=dtype, device="cuda")
        self._eight = None                          # [q, scale] of the last call in 8 bits; its type is the next one's, unless that names one
        self._kept = []                             # (n, h, z) of calls of forward whose gradients are still to come

    def parameters(self):
        return [self.norm, self.weight, self.bias]

    def forward(self, y, h, keep=False):
        """(y, h) of the next layer from those of this one.  ``keep=True`` keeps what ``backward`` needs, for each call of its own, until
        that takes it or ``update`` changes the parameters; ``keep=`` a list appends it there instead."""
        n, h = lo.rms_norm(self.aggregation.forward(y), self.norm, residual=h, eps=self.eps, out_dtype=self.weight.dtype)
        kept = keep if isinstance(keep, list) else self._kept if keep else None
        if kept is None:
            return lo.linear(n, self.weight, self.bias, activation=self.activation), h
        y, z = lo.linear(n, self.weight, self.bias, activation=self.activation, return_preactivation=True)
        kept.append((n, h, z))
        return y, h

    def backward(self, dy, dh, kept=None):
        """Gradients (dy, dh) of the layer's inputs and of its parameters from those of its outputs.  They are those of the latest
        ``forward(keep=True)`` that no ``backward`` has had yet, or of the call whose entry of its list is passed as ``kept``."""
        n, h, z = self._take(kept)
        dn, dweight, dbias = lo.linear_grad(dy, n, self.weight, z=z, activation=self.activation, bias_dtype=self.bias.dtype)
        dsum, dnorm = lo.rms_norm_grad(dn, h, self.norm, eps=self.eps, dh=dh)
        return self.aggregation.backward(dsum), dsum, [dnorm, dweight, dbias]

    def _take(self, kept):
        return _take(self._kept, kept)

    def weight_8bit(self, dtype=None):
        """The weight as it is now in 8 bits, for ``forward_8bit``: ``(q, scale)`` of ``quantize_rows``."""
        return lo.quantize_rows(self.weight, dtype)

    def _weights_8bit(self, dtype, weight):
        """What ``forward_8bit`` multiplies with: ``weight``, or the weights as they are now."""
        if weight is None:
            eight = self.weight_8bit(self._eight[0].dtype if dtype is None and self._eight else dtype)
            if self._eight is None:
                self._eight = []
            self._eight[:] = eight
            return eight
        if dtype is not None and weight[0].dtype is not dtype:
            raise ValueError(f"weight is of {weight[0].dtype}, dtype is {dtype}")
        return weight

    def forward_8bit(self, y, h, dtype=None, weight=None):
        """``forward`` with the dense product in 8 bits, ``dtype`` (None: that of the layer's call before, e4m3 for the first one and after
        ``update``).  The weight is taken into 8 bits in every call, since nothing tells who has written to it meanwhile.  A caller who
        knows passes ``weight``, what ``weight_8bit`` returned since the last change, and saves that pass over it."""
        eight = self._weights_8bit(dtype, weight)
        q, scale, h = lo.rms_norm_8bit(self.aggregation.forward(y), self.norm, residual=h, eps=self.eps, dtype=eight[0].dtype)
        return lo.linear_8bit(q, scale, *eight, self.bias, activation=self.activation, out_dtype=self.weight.dtype), h

    def update(self, grads, rate: float):
        for p, d in zip(self.parameters(), grads):
            p.add_(d.to(p.dtype), alpha=-rate)
        self._eight = None
        self._kept.clear()


class GatedLayer(GraphLayer):
    """A layer with layer norm and a gated feed-forward block of ``hidden`` features in the place of the one transform; else as ``GraphLayer``."""

    def __init__(self, aggregation: Aggregation, feat_size: int, hidden: int | None = None, activation: str = "silu", dtype=None, generator=None, eps: float = 1e-5):
        torch = fa._torch()
        dtype = torch.float32 if dtype is None else dtype
        hidden = 2 * feat_size if hidden is None else hidden

        def normal(rows, cols):
            return (torch.randn((rows, cols), device="cuda", generator=generator) * cols ** -0.5).to(dtype)

        self.aggregation, self.activation, self.eps = aggregation, activation, eps
        self.norm, self.shift = torch.ones(feat_size, dtype=dtype, device="cuda"), torch.zeros(feat_size, dtype=dtype, device="cuda")
        self.gates, self.gates_bias = normal(2 * hidden, feat_size), torch.zeros(2 * hidden, dtype=dtype, device="cuda")      # (the gate's rows first)
        self.weight, self.bias = normal(feat_size, hidden), torch.zeros(feat_size, dtype=dtype, device="cuda")
        self._eight = None                          # [q, scale] of both weights
        self._kept = []                             # (n, h, z, m) of calls of forward

    def parameters(self):
        return [self.norm, self.shift, self.gates, self.gates_bias, self.weight, self.bias]

    def forward(self, y, h, keep=False):
        n, h = lo.layer_norm(self.aggregation.forward(y), self.norm, self.shift, residual=h, eps=self.eps, out_dtype=self.weight.dtype)
        kept = keep if isinstance(keep, list) else self._kept if keep else None
        if kept is None:
            return lo.linear(lo.gated_linear(n, self.gates, self.gates_bias, activation=self.activation), self.weight, self.bias), h
        m, z = lo.gated_linear(n, self.gates, self.gates_bias, activation=self.activation, return_preactivation=True)
        kept.append((n, h, z, m))
        return lo.linear(m, self.weight, self.bias), h

    def backward(self, dy, dh, kept=None):
        n, h, z, m = self._take(kept)
        dm, dweight, dbias = lo.linear_grad(dy, m, self.weight, bias_dtype=self.bias.dtype)
        dn, dgates, dgates_bias = lo.gated_linear_grad(dm, n, self.gates, z, activation=self.activation, bias_dtype=self.gates_bias.dtype)
        dsum, dnorm, dshift = lo.layer_norm_grad(dn, h, self.norm, eps=self.eps, dh=dh, bias_dtype=self.shift.dtype)
        return self.aggregation.backward(dsum), dsum, [dnorm, dshift, dgates, dgates_bias, dweight, dbias]

    def weight_8bit(self, dtype=None):
        """Both weights as they are now in 8 bits: ``(q, scale)`` of the gated product's, then of the other's."""
        return (*lo.quantize_rows(self.gates, dtype), *lo.quantize_rows(self.weight, dtype))

    def forward_8bit(self, y, h, dtype=None, weight=None):
        """``forward`` with both products in 8 bits; what they read of the rows is taken into 8 bits row by row."""
        gates, gates_scale, weight, weight_scale = self._weights_8bit(dtype, weight)
        q, scale, h = lo.layer_norm_8bit(self.aggregation.forward(y), self.norm, self.shift, residual=h, eps=self.eps, dtype=gates.dtype)
        m = lo.gated_linear_8bit(q, scale, gates, gates_scale, self.gates_bias, activation=self.activation, out_dtype=self.weight.dtype)
        return lo.linear_8bit(*lo.quantize_rows(m, gates.dtype), weight, weight_scale, self.bias, out_dtype=self.weight.dtype), h


class NodeEmbedding:
    """Features of nodes by id out of a table that is trained: ``table[id] * scale``; an id outside of it (padding) has features of zeros."""

    def __init__(self, num_nodes: int, feat_size: int, scale: float = 1.0, dtype=None, generator=None):
        torch = fa._torch()
        self.table = torch.randn((num_nodes, feat_size), device="cuda", generator=generator).to(torch.float32 if dtype is None else dtype)
        self.scale = scale
        self._kept = []                             # ids of calls of forward

    def parameters(self):
        return [self.table]

    def forward(self, ids, keep=False):
        kept = keep if isinstance(keep, list) else self._kept if keep else None
        if kept is not None:
            kept.append(ids.clone())                # (the caller may read the next batch into them)
        return lo.embedding(ids, self.table, scale=self.scale)

    def backward(self, dy, kept=None):
        """``[gradient of the table]``, of the call of ``forward`` that ``GraphLayer.backward`` would take."""
        return [lo.embedding_grad(dy, _take(self._kept, kept), self.table.shape[0], scale=self.scale, out_dtype=self.table.dtype)]

    def update(self, grads, rate: float):
        self.table.add_(grads[0].to(self.table.dtype), alpha=-rate)
        self._kept.clear()


def train_step(layers, y, h, target, rate: float, max_norm: float | None = None, embedding: NodeEmbedding | None = None):
    """One step of plain gradient descent on mean((y - target)^2); returns the loss before it (a CUDA scalar).  A layer may stand in
    ``layers`` more than once.  With an ``embedding`` y are the ids of the nodes, whose features it gives, and it is trained too.  With
    ``max_norm`` the gradients of all parameters together are cut to that norm (``layer_ops.clip_gradients``), and ``(loss, norm)`` is returned."""
    torch = fa._torch()
    if embedding is not None:
        y = embedding.forward(y, keep=True)
    for layer in layers:
        y, h = layer.forward(y, h, keep=True)
    off = y.float() - target
    loss = off.square().mean()
    dy, dh = (off * (2.0 / off.numel())).to(y.dtype), torch.zeros_like(h)
    sums = {}
    for layer in reversed(layers):
        dy, dh, grads = layer.backward(dy.to(layer.weight.dtype), dh)
        sums[layer] = [a + b for a, b in zip(sums[layer], grads)] if layer in sums else grads
    if embedding is not None:
        sums[embedding] = embedding.backward(dy)
    norm = None
    if max_norm is not None:
        _, norm = lo.clip_gradients([g for grads in sums.values() for g in grads], max_norm, in_place=True)
    for layer, grads in sums.items():
        layer.update(grads, rate)
    return loss if norm is None else (loss, norm)


def main(argv=None):
    from .synthetic import make_workload
    ap = argparse.ArgumentParser(description="graph layers on a synthetic graph: training steps, then serving in 16 and 8 bits")
    ap.add_argument("--synthetic", default="cfg2", help="workload of liteform_ae_amd.synthetic (a square matrix)")
    ap.add_argument("--scale", type=float, default=1.0)
    ap.add_argument("--feat", type=int, default=128)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--rate", type=float, default=50.0)
    ap.add_argument("--gated", action="store_true", help="layers with layer norm and a gated feed-forward block")
    ap.add_argument("--embedding", action="store_true", help="the nodes' features are a table that is trained, looked up by id")
    ap.add_argument("--max-norm", type=float, default=None, help="the gradients of all parameters together are cut to this norm")
    a = ap.parse_args(argv)
    torch = fa._torch()
    g = make_workload(a.synthetic, scale=a.scale).matrix
    rows = g.num_src_nodes()
    if rows != g.num_dst_nodes():
        raise ValueError("a stack of layers needs a square matrix")
    gen = torch.Generator(device="cuda").manual_seed(0)
    aggregation = Aggregation(g, a.feat)
    layers = [(GatedLayer if a.gated else GraphLayer)(aggregation, a.feat, generator=gen) for _ in range(a.layers)]
    y, target = (torch.randn((rows, a.feat), device="cuda", generator=gen) for _ in range(2))
    h = torch.zeros_like(y)
    embedding = NodeEmbedding(rows, a.feat, generator=gen) if a.embedding else None
    ids = torch.arange(rows, device="cuda")
    losses = []
    for _ in range(a.steps):
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        result = train_step(layers, y if embedding is None else ids, h, target, a.rate, a.max_norm, embedding)
        loss, norm = (result, None) if a.max_norm is None else result
        losses.append(float(loss))
        print(f"loss {losses[-1]:.6f}  step(ms): {(time.perf_counter() - t0) * 1e3:.3f}" + ("" if norm is None else f"  norm: {float(norm):.3e}"))
    if embedding is not None:
        y = embedding.forward(ids)

    def serve(call):
        v, s = y, h
        for layer in layers:
            v, s = call(layer, v, s)
        return v

    eights = {layer: layer.weight_8bit() for layer in layers}            # (trained weights do not change any more)
    forward = type(layers[0]).forward if layers else GraphLayer.forward
    want = serve(forward)
    for name, call in (("float32", forward), ("8 bits", lambda layer, v, s: layer.forward_8bit(v, s, weight=eights[layer]))):
        best = float("inf")
        for _ in range(5):
            torch.cuda.synchronize()
            t0 = time.perf_counter()
            out = serve(call)
            torch.cuda.synchronize()
            best = min(best, time.perf_counter() - t0)
        off = float((out - want).norm() / want.norm())
        print(f"{name}: {best * 1e3:.3f} ms, off by {off:.2e}")
    return losses


if __name__ == "__main__":
    main()
