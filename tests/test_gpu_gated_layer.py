"""A stack that is trained from node ids - embedding, gated layers, clipping (graph_layer) - against the same stack in 64 bits."""
import math

import pytest

from helpers import skewed_matrix
from test_gpu_graph_layer import dense

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
np = pytest.importorskip("numpy")
ROWS, FEAT, HIDDEN = 300, 64, 100


@pytest.fixture(scope="module")
def gl():
    from liteform_ae_amd import graph_layer
    return graph_layer


def stack(gl, seed, dtype=torch.float32, count=2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = skewed_matrix(np.random.default_rng(5), ROWS, ROWS, mean_deg=5.0)
    aggregation = gl.Aggregation(g, FEAT, "f32" if dtype is torch.float32 else "bf16")
    layers = [gl.GatedLayer(aggregation, FEAT, HIDDEN, dtype=dtype, generator=gen) for _ in range(count)]
    for layer in layers:
        for p in (layer.norm, layer.shift, layer.gates_bias, layer.bias):
            p += (0.1 * torch.randn(p.shape, device="cuda", generator=gen)).to(dtype)
    embedding = gl.NodeEmbedding(200, FEAT, scale=2.0, dtype=dtype, generator=gen)
    ids = torch.randint(0, 200, (ROWS,), device="cuda", generator=gen)
    ids[::7] = -1                                                         # (nodes without features)
    h, target = (torch.randn((ROWS, FEAT), device="cuda", generator=gen) for _ in range(2))
    return dense(g), layers, embedding, ids, h.to(dtype), target


def layer64(A, layer, p, y, h):
    norm, shift, gates, gates_bias, weight, bias = p
    s = A @ y + h
    mean = s.mean(dim=1, keepdim=True)
    n = (s - mean) / torch.sqrt((s - mean).square().mean(dim=1, keepdim=True) + layer.eps) * norm + shift
    z = n @ gates.t() + gates_bias
    k = z.shape[1] // 2
    return (torch.nn.functional.silu(z[:, :k]) * z[:, k:]) @ weight.t() + bias, s


def stack64(A, layers, embedding, ids, h):
    """Parameters in 64 bits, by layer, and (y, h) of the last layer."""
    ps = {layer: [p.double().requires_grad_() for p in layer.parameters()] for layer in (*layers, embedding)}
    y = torch.where((ids >= 0)[:, None], ps[embedding][0][ids.clamp_min(0)] * embedding.scale, 0.0)
    s = h.double()
    for layer in layers:
        y, s = layer64(A, layer, ps[layer], y, s)
    return ps, y, s


def off(a, b):
    return float((a.double() - b).detach().norm() / b.detach().norm())


def test_forward_and_gradients(gl):
    A, layers, embedding, ids, h, target = stack(gl, 1)
    ps, y64, s64 = stack64(A, layers, embedding, ids, h)
    y, s = embedding.forward(ids, keep=True), h
    for layer in layers:
        y, s = layer.forward(y, s, keep=True)
    # two layers, each off by some 100 roundings of 2^-24 of values near one, and rows of up to 150 neighbours
    assert off(y, y64) <= 1e-5 and off(s, s64) <= 1e-5
    dy, dh = torch.randn_like(y), torch.randn_like(s)
    ((y64 * dy.double()).sum() + (s64 * dh.double()).sum()).backward()
    for layer in reversed(layers):
        dy, dh, grads = layer.backward(dy, dh)
        for got, want in zip(grads, ps[layer]):
            assert got.shape == want.shape and off(got, want.grad) <= 2e-5
    (got,) = embedding.backward(dy)
    assert off(got, ps[embedding][0].grad) <= 2e-5
    for layer in (*layers, embedding):
        with pytest.raises(RuntimeError, match="keep=True"):
            layer.backward(dy, dh) if layer is not embedding else layer.backward(dy)


def test_training_step_with_clipped_gradients(gl):
    for most in (1e-3, 1e3):
        A, layers, embedding, ids, h, target = stack(gl, 2)
        ps, y64, _ = stack64(A, [layers[0], layers[1], layers[0]], embedding, ids, h)       # (a layer that stands twice)
        loss64 = (y64 - target.double()).square().mean()
        loss64.backward()
        norm64 = math.sqrt(sum(float(p.grad.square().sum()) for each in ps.values() for p in each))
        factor, rate = min(1.0, most / (norm64 + 1e-6)), 0.5
        loss64 = loss64.detach()
        loss, norm = gl.train_step([layers[0], layers[1], layers[0]], ids, h, target, rate, max_norm=most, embedding=embedding)
        assert abs(float(loss) - float(loss64)) <= 1e-5 * float(loss64) and abs(float(norm) - norm64) <= 2e-5 * norm64
        for layer, each in ps.items():
            # the step of a parameter near one is known to half of its last place, 2^-24 of the values' norm at most, and to the gradient's 2e-5, twice
            for p, p64 in zip(layer.parameters(), each):
                step = rate * factor * p64.grad
                assert float((p.double() - (p64.detach() - step)).norm()) <= 4e-5 * float(step.norm()) + 2.0 ** -24 * float(p64.detach().norm() + step.norm())


def test_training_step_without_clipping_is_as_before(gl):
    """Without the new arguments a step returns the loss alone; a limit that cuts nothing changes nothing."""
    runs = []
    for most in (None, 1e9):
        _, layers, embedding, ids, h, target = stack(gl, 3)
        result = gl.train_step(layers, ids, h, target, 0.5, embedding=embedding, max_norm=most)
        assert (most is None) == isinstance(result, torch.Tensor)
        runs.append([result if most is None else result[0]] + [p for layer in (*layers, embedding) for p in layer.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_forward_in_8_bits(gl, dtype):
    _, layers, embedding, ids, h, _ = stack(gl, 4)
    c = e = embedding.forward(ids)
    d = f = h
    for layer in layers:
        c, d = layer.forward(c, d)
        weight = layer.weight_8bit(dtype)
        a, b = layer.forward_8bit(e, f, weight=weight)
        e, f = layer.forward_8bit(e, f, dtype)
        assert torch.equal(a, e) and torch.equal(b, f)
    # e4m3 rounds by 2^-4 / sqrt 3 of a value at most, both operands of both products of two layers; the products' sums average that
    assert 1e-4 < off(e, c.double()) < 0.15
    with pytest.raises(ValueError, match="dtype"):
        layer.forward_8bit(e, f, torch.int8 if dtype is not torch.int8 else torch.float8_e4m3fn, weight)


def test_bfloat16(gl):
    A, layers, embedding, ids, h, _ = stack(gl, 5, torch.bfloat16)
    ps, y64, s64 = stack64(A, layers, embedding, ids, h)
    y, s = embedding.forward(ids, keep=True), h
    for layer in layers:
        y, s = layer.forward(y, s, keep=True)
    assert y.dtype is s.dtype is torch.bfloat16
    # n, z, m, y and h of each layer are rounded by 2^-9 on average
    assert off(y, y64) < 2e-2 and off(s, s64) < 1e-2
    dy, dh = torch.randn_like(y), torch.randn_like(s)
    ((y64 * dy.double()).sum() + (s64 * dh.double()).sum()).backward()
    for layer in reversed(layers):
        dy, dh, grads = layer.backward(dy.to(torch.bfloat16), dh)
        for got, want in zip(grads, ps[layer]):
            assert got.dtype is torch.bfloat16 and off(got, want.grad) < 4e-2
    assert off(embedding.backward(dy)[0], ps[embedding][0].grad) < 4e-2


def test_a_step_in_a_graph(gl):
    """Forward, backward and clipping recorded once and replayed, between eager steps of the same stack."""
    from liteform_ae_amd import layer_ops as lo
    _, layers, embedding, ids, h, target = stack(gl, 6)
    gen = torch.Generator(device="cuda").manual_seed(7)
    dy, dh = (torch.randn((ROWS, FEAT), device="cuda", generator=gen) for _ in range(2))

    def step():
        kept, some = [[] for _ in layers], []
        y, s = embedding.forward(ids, keep=some), h
        for layer, each in zip(layers, kept):
            y, s = layer.forward(y, s, keep=each)
        a, b, grads = dy, dh, []
        for layer, each in zip(reversed(layers), reversed(kept)):
            a, b, more = layer.backward(a, b, each[0])
            grads += more
        clipped, norm = lo.clip_gradients(grads + embedding.backward(a, some[0]), 0.5, in_place=True)
        return [y, s, norm, *clipped]

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
        assert all(torch.equal(a, b) for a, b in zip(step(), want)), turn


def test_command(capsys):
    from liteform_ae_amd import graph_layer
    graph_layer.main(["--synthetic", "cfg2", "--scale", "0.02", "--feat", "64", "--steps", "2", "--rate", "0.5", "--gated", "--embedding", "--max-norm", "1"])
    out = capsys.readouterr().out
    assert "8 bits" in out and out.count("norm:") == 2
    graph_layer.main(["--synthetic", "cfg2", "--scale", "0.02", "--feat", "64", "--steps", "1", "--max-norm", "1", "--embedding"])
    assert "norm:" in capsys.readouterr().out


def test_inputs_that_require_gradients(gl):
    _, layers, embedding, ids, h, _ = stack(gl, 8)
    y = embedding.forward(ids)
    want = layers[0].forward(y, h)
    for a, b in ((y.clone().requires_grad_(), h), (y, h.clone().requires_grad_())):
        for call in (layers[0].forward, layers[0].forward_8bit):
            with pytest.raises(ValueError, match="no_grad"):
                call(a, b)
        with torch.no_grad():
            assert all(torch.equal(c, d) for c, d in zip(layers[0].forward(a, b), want))
    embedding.table.requires_grad_()
    with pytest.raises(ValueError, match="requires gradients"):
        embedding.forward(ids)
