"""Limits of clipping that cut nothing, and what node embeddings keep of a call."""
import math

import pytest

from test_gpu_layer_ops import BF16, F16, F32, gen

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lo():
    from liteform_ae_amd import layer_ops
    return layer_ops


def same(a, b):
    return a.dtype is b.dtype and a.shape == b.shape and torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, nan=7.0, posinf=8.0, neginf=9.0),
                                                                                                                     torch.nan_to_num(b, nan=7.0, posinf=8.0, neginf=9.0))


def test_an_infinite_limit_cuts_nothing(lo):
    """Whatever the norm: one that is infinite, of infinite elements or beyond float32, leaves all as it is; one that is NaN makes all NaN."""
    g = gen(81)
    for dtype in (F32, BF16, F16):
        for bad in (None, math.inf, -math.inf, 3e38, math.nan):
            if bad == 3e38 and dtype is F16:
                continue
            grads = [torch.randn(s, device="cuda", generator=g).to(dtype) for s in ((1000,), (30, 17), (3,))]
            if bad is not None:
                grads[0][[3, 5, 500]] = bad
            for eps in (0.0, 1e-6, math.inf):
                before = [t.clone() for t in grads]
                want = before if bad is None or not math.isnan(bad) else [torch.full_like(t, math.nan) for t in before]
                clipped, norm = lo.clip_gradients(grads, math.inf, eps=eps)
                assert all(map(same, clipped, want)) and all(map(same, grads, before)), (dtype, bad, eps)
                assert bad is None or (math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf)
                clipped, again = lo.clip_gradients([t.clone() for t in grads], math.inf, eps=eps, in_place=True)
                assert all(map(same, clipped, want)) and same(norm, again), (dtype, bad, eps)


def test_a_finite_limit_and_an_infinite_norm(lo):
    """Zeros, and NaN for what is infinite itself, in place and not."""
    for most in (0.0, 1.0, 3e38):
        grads = [torch.ones(100, device="cuda"), torch.ones((5, 5), device="cuda", dtype=BF16)]
        grads[0][7] = math.inf
        for in_place in (False, True):
            clipped, norm = lo.clip_gradients(grads, most, in_place=in_place)
            assert float(norm) == math.inf and bool(torch.isnan(clipped[0][7])) and int(torch.isnan(clipped[0]).sum()) == 1
            assert bool((torch.nan_to_num(clipped[0]) == 0).all()) and bool((clipped[1] == 0).all())


def test_ids_that_change_between_forward_and_backward():
    """A buffer of ids that the next batch is read into: each call's gradient is of the ids that it had."""
    from liteform_ae_amd import graph_layer, layer_ops as lo
    g = gen(82)
    embedding = graph_layer.NodeEmbedding(50, 24, generator=g)
    first, second = (torch.randint(0, 50, (300,), device="cuda", generator=g) for _ in range(2))
    dy = torch.randn((300, 24), device="cuda", generator=g)
    want = [lo.embedding_grad(dy, ids, 50) for ids in (first, second)]
    ids, some = first.clone(), []
    embedding.forward(ids, keep=True)
    embedding.forward(ids, keep=some)
    ids.copy_(second)
    embedding.forward(ids, keep=True)
    ids.zero_()
    assert torch.equal(embedding.backward(dy)[0], want[1]) and torch.equal(embedding.backward(dy)[0], want[0]) and torch.equal(embedding.backward(dy, some[0])[0], want[0])
