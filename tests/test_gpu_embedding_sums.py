"""Gradients of embedding tables where one id has many rows: exact sums, and bounds of the additions that there are."""
import pytest

from test_gpu_layer_ops import BF16, E, F16, F32, TINY, U, gen, normal, within
from test_gpu_training_ops import ids_of

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
# ids, rows, columns: one id, some and many; spans of ids that end in, at and behind a workgroup's; sorted in one workgroup and in many; narrow and wide rows
SIZES = [(1, 1, 5), (7, 1, 64), (300, 2, 100), (8192, 1, 24), (8193, 3, 24), (40_000, 1, 64), (40_000, 1000, 100), (65_536, 10, 130), (65_537, 82, 33), (131_072, 200, 64),
         (300_000, 1, 64), (300_000, 9, 16), (300_000, 50, 130), (500_000, 50, 8), (20_000, 2, 1000), (20_000, 700, 600), (2_000_003, 9, 8), (2_500_001, 100_000, 12)]


@pytest.fixture(scope="module")
def lo():
    from liteform_ae_amd import layer_ops
    return layer_ops


def sums(ids, rows, dy):
    """Sums in 64 bits, and how many terms each has (few rows as a product: additions to one address would wait for one another)."""
    wide = ids.long()
    on = (wide >= 0) & (wide < rows)
    wide, dy = wide[on], dy[on].double()
    if rows <= 1000:
        want = (torch.arange(rows, device="cuda")[:, None] == wide).double() @ dy
    else:
        want = torch.zeros((rows, dy.shape[1]), device="cuda", dtype=torch.float64).index_add_(0, wide, dy)
    return want, torch.bincount(wide, minlength=rows)[:rows, None]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_sums_of_whole_numbers_are_exact(lo, dtype):
    """One entry that is lost, doubled or of another row is seen.  All sums stay below 2^24."""
    g = gen(71)
    for i, (n, rows, dim) in enumerate(SIZES):
        ids = ids_of(n, rows, g, ("even", "zipf")[i % 2], (torch.int64, torch.int32)[i % 2], bad=i % 3 != 0)
        dy = torch.randint(-3, 5, (n, dim), device="cuda", generator=g).to(dtype)
        one = torch.zeros((rows, dim), device="cuda", dtype=torch.float64)
        one[rows - 1] = dy.double().sum(dim=0)
        for given, want in ((ids, None), (ids.sort().values, None), (torch.full_like(ids, rows - 1), one)):
            want = sums(given, rows, dy)[0] if want is None else want
            assert torch.equal(lo.embedding_grad(dy, given, rows, out_dtype=F32).double(), want), (n, rows, dim)
            assert torch.equal(lo.embedding_grad(dy, given, rows, scale=-0.5, out_dtype=BF16), (want * -0.5).to(F32).to(BF16)), (n, rows, dim)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_sums_of_many_rows(lo, dtype):
    g = gen(72)
    for i, (n, rows, dim) in enumerate(SIZES):
        ids = ids_of(n, rows, g, ("zipf", "even")[i % 2], (torch.int64, torch.int32)[i % 2])
        dy, scale = normal((n, dim), dtype, g, 1.0, (0, 3)[i % 2], i % 2), (1.0, 0.3, -11.3)[i % 3]
        want, count = sums(ids, rows, dy)
        size, _ = sums(ids, rows, dy.abs())
        # 16 bits: up to 64 terms one after the other and those of up to 32 groups of threads in 32 bits, the rest in 64 bits, as all of float32 (and
        # of what it is compared with)
        off = size * ((96 * E if dtype is not F32 else 0.0) + (count + 100) * 2.0 ** -52)
        # the scale, the sum and the product are rounded to 32 bits
        bound = (want.abs() * 4 * E + off) * abs(scale) * 1.01
        for out in (F32, dtype):
            got = lo.embedding_grad(dy, ids, rows, scale=scale, out_dtype=out)
            within(got, want * scale, (want * scale).abs() * U[out] + bound * (1 + U[out]) + (count > 0) * TINY[out], (n, rows, dim))


@pytest.mark.parametrize("n,rows,dim", [(30_000, 200, 24), (50_000, 200, 24), (50_000, 3000, 24), (40_000, 2_000_000, 8), (9000, 8000, 1300), (2000, 30_000, 600)])
def test_both_ways_of_the_sort_and_the_sums_in_a_graph(lo, n, rows, dim):
    """Recorded once and replayed with other ids and rows in the same buffers, between eager calls."""
    g = gen(73)
    dy, ids = normal((n, dim), F32, g), ids_of(n, rows, g)
    lo.embedding_grad(dy, ids, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = lo.embedding_grad(dy, ids, rows)
    for _ in range(3):
        dy.copy_(normal((n, dim), F32, g))
        ids.copy_(ids_of(n, rows, g, "zipf"))
        want = lo.embedding_grad(dy, ids, rows)
        got.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
