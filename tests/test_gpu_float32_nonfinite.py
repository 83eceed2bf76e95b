"""float32 products at the ends of the range: with many values that are not finite, right as any others and not much slower; of the smallest ones."""
import math

import pytest

from test_gpu_layer_ops import E, F32, TINY, gen, lo, normal  # noqa: F401 (lo: the fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def spoil(t, g, share):
    """Some values infinite, some NaN, and zeros for them to meet."""
    at = torch.rand(t.shape, device="cuda", generator=g)
    t[at < share] = math.inf
    t[(at >= share) & (at < 2 * share)] = -math.inf
    t[(at >= 2 * share) & (at < 3 * share)] = math.nan
    t[(at >= 0.5) & (at < 0.6)] = 0.0
    return t


def compare(got, a, b):
    """got = a b, where the terms of an output have an infinity, infinities of both signs, a NaN, or are finite."""
    want = a.double() @ b.double()
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got == math.inf, want == math.inf) and torch.equal(got == -math.inf, want == -math.inf)
    fine = torch.isfinite(want)
    bound = (a.nan_to_num(0, 0, 0).double().abs() @ b.nan_to_num(0, 0, 0).double().abs()) * (a.shape[1] + 24) * E + TINY[F32]
    assert bool(((got - want).abs() <= bound)[fine].all())
    return want


@pytest.mark.parametrize("share", [1e-5, 1e-3, 0.02])
def test_values_that_are_not_finite(lo, share):  # noqa: F811
    g = gen(71)
    for m, n, k, pad in [(17, 5, 3, 0), (33, 130, 70, 3), (64, 64, 64, 0), (130, 257, 513, 5), (300, 20, 9001, 0), (1100, 1030, 515, 1), (2050, 3000, 260, 0)]:
        x, w, dy = (spoil(normal(s, F32, g, 1.0, pad, pad // 3), g, share) for s in ((m, k), (n, k), (m, n)))
        compare(lo.linear(x, w), x, w.t())
        dx, dw, _ = lo.linear_grad(dy, x, w)
        compare(dx, dy, w)
        compare(dw, dy.t(), x)


def test_what_stands_beside_a_matrix_is_not_looked_at(lo):  # noqa: F811
    """NaN in the buffer behind every row, which tiles of k across read along: the same bits as without."""
    g = gen(72)
    for m, n, k in [(70, 100, 65), (1030, 1100, 515)]:
        plain = [normal(s, F32, g).contiguous() for s in ((m, n), (m, k), (n, k))]
        wide = []
        for t in plain:
            buffer = torch.full((t.shape[0] + 1, t.shape[1] + 7), math.nan, device="cuda")
            buffer[:-1, :t.shape[1]] = t
            wide.append(buffer[:-1, :t.shape[1]])
        for a, b in zip(lo.linear_grad(*plain)[:2], lo.linear_grad(*wide)[:2]):
            assert torch.equal(a, b)
        assert torch.equal(lo.linear(*plain[1:]), lo.linear(*wide[1:]))


def test_an_operand_of_nan_takes_a_few_times_as_long(lo):  # noqa: F811
    """The product is made twice: of planes, six bf16 products, and by float32 matrix instructions, which take as long as sixteen: 16 / 6 of its time,
    twice that with operands that are not staged, 6.4 in all.  (An output at a time took 80.)"""
    g = gen(73)
    x, w = normal((2048, 2048), F32, g), normal((2048, 2048), F32, g)

    def time(a):
        times = []
        for _ in range(9):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            lo.linear(a, w)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return sorted(times)[4]

    bad = torch.full_like(x, math.nan)
    time(x), time(bad)
    assert time(bad) <= 12 * time(x)


@pytest.mark.parametrize("power", [-100, -112, -118, -124, -130])
def test_values_near_the_smallest(lo, power):  # noqa: F811
    """What a value's three bfloat16 leave below 2^-126 is lost to the matrix instruction, and so is a sum below it at each of its instructions."""
    g = gen(74)
    lost = 2.0 ** -126
    for m, n, k in [(64, 70, 256), (300, 200, 1000), (40, 30, 9000)]:
        x, w = normal((m, k), F32, g) * 2.0 ** power, normal((n, k), F32, g)
        x64, w64 = x.double(), w.double()
        want = x64 @ w64.t()
        bound = (x64.abs() @ w64.abs().t()) * (k + 24) * E + 1.01 * lost * (x64.abs().sum(dim=1)[:, None] + w64.abs().sum(dim=1)) + 6 * (k // 32 + 1) * lost
        assert bool(((lo.linear(x, w).double() - want).abs() <= bound).all()), (m, n, k)
    x, w = normal((16, 300), F32, g) * 2.0 ** power, normal((40, 300), F32, g)         # (few rows: float32 instructions)
    x64, w64 = x.double(), w.double()
    assert bool(((lo.linear(x, w).double() - x64 @ w64.t()).abs() <= (x64.abs() @ w64.abs().t()) * 324 * E + TINY[F32]).all())
