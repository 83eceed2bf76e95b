"""A graph layer made of the package's operators (graph_layer) against the same layer in 64 bits, forward, in 8 bits and backward."""
import numpy as np
import pytest

from helpers import skewed_matrix

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def dense(g):
    return torch.from_numpy(np.asarray(g.coo_mtx.todense())).double().cuda()


def layer64(A, layer, y, h):
    """(y, h) of a layer, differentiable in 64 bits."""
    s = A @ y + h
    n = s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + layer.eps) * layer.p64[0]
    z = n @ layer.p64[1].t() + layer.p64[2]
    return z * torch.special.ndtr(z), s


@pytest.fixture(scope="module")
def setup():
    from liteform_ae_amd import graph_layer as gl
    rng = np.random.default_rng(5)
    g = skewed_matrix(rng, 300, 300, mean_deg=5.0)
    gen = torch.Generator(device="cuda").manual_seed(1)
    aggregation = gl.Aggregation(g, 64)
    layers = [gl.GraphLayer(aggregation, 64, generator=gen) for _ in range(3)]
    for layer in layers:
        layer.norm += 0.1 * torch.randn(64, device="cuda", generator=gen)
        layer.bias += 0.1 * torch.randn(64, device="cuda", generator=gen)
    y, h, target = (torch.randn((300, 64), device="cuda", generator=gen) for _ in range(3))
    return gl, g, layers, y, h, target


def test_forward_and_gradients(setup):
    gl, g, layers, y, h, target = setup
    A = dense(g)
    for layer in layers:
        layer.p64 = [p.detach().double().requires_grad_() for p in layer.parameters()]
    v, s = y.double().requires_grad_(), h.double().requires_grad_()
    a, b = v, s
    for layer in layers:
        a, b = layer64(A, layer, a, b)
    c, d = y, h
    for layer in layers:
        c, d = layer.forward(c, d, keep=True)
    # each of the three layers is off by some 100 roundings of 2^-24 of values near one, and rows of up to 150 neighbours
    assert float((c.double() - a).norm() / a.norm()) <= 1e-5 and float((d.double() - b).norm() / b.norm()) <= 1e-5
    dy, dh = torch.randn_like(c), torch.randn_like(d)
    ((a * dy.double()).sum() + (b * dh.double()).sum()).backward()
    for layer in reversed(layers):
        dy, dh, grads = layer.backward(dy, dh)
        for got, want in zip(grads, layer.p64):
            assert float((got.double() - want.grad).norm() / want.grad.norm()) <= 2e-5
    assert float((dy.double() - v.grad).norm() / v.grad.norm()) <= 2e-5
    assert float((dh.double() - s.grad).norm() / s.grad.norm()) <= 2e-5


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_forward_in_8_bits(setup, dtype):
    gl, g, layers, y, h, target = setup
    c, d, e, f = y, h, y, h
    for layer in layers:
        layer._eight = None
        c, d = layer.forward(c, d)
        e, f = layer.forward_8bit(e, f, dtype)
    # e4m3 rounds by 2^-4 / sqrt 3 of a value at most, both operands of each of three layers; the products' sums average that
    assert 1e-4 < float((e - c).norm() / c.norm()) < 0.1
    kept = layers[0]._eight
    assert kept[0].dtype is dtype
    layers[0].forward_8bit(y, h)
    assert layers[0]._eight is kept
    layers[0].update([torch.zeros_like(p) for p in layers[0].parameters()], 1.0)
    assert layers[0]._eight is None


def test_training_lowers_the_loss(setup):
    gl, g, layers, y, h, target = setup
    losses = [float(gl.train_step(layers, y, h, target, 5.0)) for _ in range(6)]
    assert all(b < a for a, b in zip(losses, losses[1:])), losses


def test_bfloat16_layer(setup):
    gl, g, _, y, h, _ = setup
    gen = torch.Generator(device="cuda").manual_seed(2)
    aggregation = gl.Aggregation(g, 64, "bf16")
    layer = gl.GraphLayer(aggregation, 64, dtype=torch.bfloat16, generator=gen)
    layer.p64 = [p.double() for p in layer.parameters()]
    yb, hb = y.bfloat16(), h.bfloat16()
    a, b = layer64(dense(g), layer, yb.double(), hb.double())
    c, d = layer.forward(yb, hb)
    assert c.dtype is d.dtype is torch.bfloat16
    # three roundings of 2^-9 on average each (n, y; h once)
    assert float((c.double() - a).norm() / a.norm()) < 1e-2 and float((d.double() - b).norm() / b.norm()) < 4e-3
    assert layer.forward_8bit(yb, hb)[0].dtype is torch.bfloat16


def test_command(capsys):
    from liteform_ae_amd import graph_layer
    losses = graph_layer.main(["--synthetic", "cfg2", "--scale", "0.02", "--feat", "64", "--steps", "3", "--rate", "5"])
    assert losses[2] < losses[1] < losses[0]
    assert "8 bits" in capsys.readouterr().out


def eight_by_hand(layer, y, h, dtype):
    from liteform_ae_amd import layer_ops as lo
    q, scale, s = lo.rms_norm_8bit(layer.aggregation.forward(y), layer.norm, residual=h, eps=layer.eps, dtype=dtype)
    return lo.linear_8bit(q, scale, *lo.quantize_rows(layer.weight, dtype), layer.bias, activation=layer.activation, out_dtype=layer.weight.dtype), s


def test_8_bits_of_the_type_that_is_asked_for(setup):
    gl, g, layers, y, h, target = setup
    layer = layers[1]
    for dtype in (torch.float8_e4m3fn, torch.int8, torch.float8_e4m3fn):
        for got, want in zip(layer.forward_8bit(y, h, dtype), eight_by_hand(layer, y, h, dtype)):
            assert torch.equal(got, want)
    weight = layer.weight_8bit(torch.int8)
    assert torch.equal(layer.forward_8bit(y, h, weight=weight)[0], eight_by_hand(layer, y, h, torch.int8)[0])
    assert torch.equal(layer.forward_8bit(y, h, torch.int8, weight)[0], eight_by_hand(layer, y, h, torch.int8)[0])
    with pytest.raises(ValueError, match="dtype"):
        layer.forward_8bit(y, h, torch.float8_e4m3fn, weight)


def test_8_bits_of_the_weight_as_it_is(setup):
    """Written to by an optimizer, past autograd's counter of changes, or by a replayed graph."""
    gl, g, _, y, h, _ = setup
    gen = torch.Generator(device="cuda").manual_seed(3)
    layer = gl.GraphLayer(gl.Aggregation(g, 64), 64, generator=gen)

    def check(change):
        before = layer.forward_8bit(y, h)[0]
        change()
        got = layer.forward_8bit(y, h)[0]
        assert torch.equal(got, eight_by_hand(layer, y, h, torch.float8_e4m3fn)[0])
        assert not torch.equal(got, before)

    def optimize():
        for p in layer.parameters():
            p.grad = torch.randn(p.shape, device="cuda", generator=gen)
        torch.optim.SGD(layer.parameters(), lr=0.1).step()

    check(optimize)
    check(lambda: layer.weight.copy_(torch.randn((64, 64), device="cuda", generator=gen)))
    check(lambda: layer.weight.data.mul_(torch.randn((64, 64), device="cuda", generator=gen)))
    layer.weight = torch.randn((64, 64), device="cuda", generator=gen)
    check(lambda: setattr(layer, "weight", torch.randn((64, 64), device="cuda", generator=gen)))
    turn = torch.randn((64, 64), device="cuda", generator=gen)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.weight.mul_(turn)
    for _ in range(3):
        check(graph.replay)


def test_gradients_of_calls_that_wait_for_them(setup):
    """Two calls before their gradients, newest first or out of lists in any order, are those of each call alone."""
    gl, g, layers, y, h, target = setup
    layer = layers[2]
    gen = torch.Generator(device="cuda").manual_seed(4)
    inputs = [tuple(torch.randn((300, 64), device="cuda", generator=gen) for _ in range(4)) for _ in range(2)]     # y, h, dy, dh
    alone = []
    for a, b, dy, dh in inputs:
        layer.forward(a, b, keep=True)
        alone.append(layer.backward(dy, dh))

    def same(got, want):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2]))

    for a, b, _, _ in inputs:
        layer.forward(a, b, keep=True)
    for i in (1, 0):
        same(layer.backward(*inputs[i][2:]), alone[i])
    with pytest.raises(RuntimeError, match="keep=True"):
        layer.backward(*inputs[0][2:])
    kept = []
    for a, b, _, _ in inputs:
        layer.forward(a, b, keep=kept)
    for i in (0, 1):
        same(layer.backward(*inputs[i][2:], kept[i]), alone[i])
    layer.forward(*inputs[0][:2], keep=True)
    layer.update([torch.zeros_like(p) for p in layer.parameters()], 1.0)
    with pytest.raises(RuntimeError, match="keep=True"):
        layer.backward(*inputs[0][2:])                                    # (of parameters that are no more)


def test_training_with_a_layer_that_stands_twice(setup):
    gl, g, layers, y, h, target = setup
    gen = torch.Generator(device="cuda").manual_seed(5)
    layer, other = (gl.GraphLayer(layers[0].aggregation, 64, generator=gen) for _ in range(2))
    A, rate = dense(g), 5.0
    for each in (layer, other):
        each.p64 = [p.double().requires_grad_() for p in each.parameters()]
    a, b = y.double(), h.double()
    for each in (layer, other, layer):
        a, b = layer64(A, each, a, b)
    loss = (a - target.double()).square().mean()
    loss.backward()
    got = gl.train_step([layer, other, layer], y, h, target, rate)
    assert float((got.double() - loss.detach()).abs() / loss.detach()) <= 1e-5
    for each in (layer, other):
        # the step of a parameter near one is known to half of its last place, 2^-24 of the values' norm at most, and to the gradient's 2e-5
        for p, p64 in zip(each.parameters(), each.p64):
            step = rate * p64.grad
            assert float((p.double() - (p64.detach() - step)).norm()) <= 2e-5 * float(step.norm()) + 2.0 ** -24 * float(p64.detach().norm() + step.norm())


def test_inputs_that_require_gradients(setup):
    gl, g, layers, y, h, target = setup
    layer = layers[0]
    want = layer.forward(y, h)
    for a, b in ((y.clone().requires_grad_(), h), (y, h.clone().requires_grad_())):
        for call in (layer.forward, layer.forward_8bit):
            with pytest.raises(ValueError, match="no_grad"):
                call(a, b)
        with torch.no_grad():
            assert all(torch.equal(c, d) for c, d in zip(layer.forward(a, b), want))
