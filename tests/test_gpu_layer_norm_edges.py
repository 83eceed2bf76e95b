"""Layer norm of rows whose elements are equal, or differ in their last places, at any distance from zero; sums of its gradient over many rows."""
import pytest

from test_gpu_layer_ops import BF16, E, F32, TINY, U, gen, normal, within
from test_gpu_training_ops import check_layer_grad, check_layer_norm, layer_reference

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
# rows of every number of threads and pieces, whole and not, and long ones
DIMS = [2, 3, 7, 9, 100, 127, 200, 500, 1000, 1025, 3001, 5000, 8191, 12_001, 20_001]


@pytest.fixture(scope="module")
def lo():
    from liteform_ae_amd import layer_ops
    return layer_ops


def magnitudes():
    """Values of 64 powers of ten, of both signs, with all their digits."""
    k = torch.arange(64, device="cuda", dtype=torch.float64)
    return ((1.0 + 0.9 * torch.frac(k * 0.61803398875)) * 10.0 ** (k - 25.5) * (1 - 2 * (k % 2))).to(F32)


@pytest.mark.parametrize("dim", DIMS)
def test_rows_of_equal_elements(lo, dim):
    """Of h - mean no more is left than 160 roundings (layer_reference) times sqrt(eps), whatever the size of h: y is the bias, and the gradient that of a row whose
    variance is 0."""
    values, g = magnitudes(), gen(61)
    x = values[:, None].repeat(1, dim)
    b = normal((1, dim), F32, g)[0]
    wide = b.double().expand_as(x)
    for eps in (1e-5, 1e-12):
        off = 160 * E + 4 * E * wide.abs()
        within(lo.layer_norm(x, None, b, eps=eps), wide, off, f"y, {eps}")
        within(lo.layer_norm(x, None, b, residual=torch.zeros_like(x), eps=eps)[0], wide, off, f"y with a residual, {eps}")
        q, scale = lo.layer_norm_8bit(x, None, b, eps=eps)
        top = wide.abs().amax(dim=1)
        within(scale * 448.0, top, 160 * E + 8 * E * top, f"scale, {eps}")
        within(q.double() * scale.double()[:, None], wide, torch.maximum(wide.abs() * 2.0 ** -4, top[:, None] / 448 * 2.0 ** -10) * (1 + 1e-3) + 2 * off, f"q, {eps}")
        dy, w = normal((len(x), dim), F32, g), normal((1, dim), F32, g)[0]
        dx, dw, db = lo.layer_norm_grad(dy, x, w, eps=eps, bias_dtype=F32)
        d = dy.double() * w.double()
        mean = d.mean(dim=1, keepdim=True)
        s = eps ** -0.5
        # a product, a mean of sums in 160 parts at most and the difference are rounded, and s is off by half of what the variance is, 160 roundings of eps
        within(dx, (d - mean) * s, s * (4 * E * d.abs() + 160 * E * d.abs().mean(dim=1, keepdim=True) + 160 * E * (d - mean).abs()), f"dx, {eps}")
        within(dw, torch.zeros_like(dw, dtype=torch.float64), dy.double().abs().sum(dim=0) * 160 * E, f"dw, {eps}")


@pytest.mark.parametrize("dim", DIMS)
def test_rows_that_differ_in_their_last_places(lo, dim):
    """Elements of 0 to 3 last places more than a value: nothing but these is left, and it has all its digits."""
    g = gen(62)
    bits = magnitudes()[8:].view(torch.int32)                             # (squares of differences below 10^-17 vanish beside either eps)
    x = (bits[:, None] + torch.randint(0, 4, (len(bits), dim), device="cuda", generator=g, dtype=torch.int32)).view(F32)
    x[:, 0] = bits.view(F32)
    x[:, -1] = (bits + 3).view(F32)                                       # (no two ends alike)
    w, b, dy = normal((1, dim), F32, g)[0], normal((1, dim), F32, g)[0], normal(x.shape, F32, g)
    for eps in (1e-5, 1e-12, 0.0):
        check_layer_norm(lo, x, w, b, None, eps, F32, (dim, eps))
        check_layer_grad(lo, dy, x, w, eps, None, (dim, eps))
    # one element of a row
    x = bits.view(F32)[:, None].repeat(1, dim)
    x[:, dim // 2] = (bits + 1).view(F32)
    for eps in (1e-5, 1e-12, 0.0):
        check_layer_norm(lo, x, w, b, None, eps, F32, (dim, eps))
        check_layer_grad(lo, dy, x, w, eps, None, (dim, eps))


def depth_of(rows, dim):
    """Additions that a term of dw and db goes through: rows of a thread, row groups of a workgroup, workgroups of a slice, slices."""
    threads = 8 if dim <= 64 else 16 if dim <= 128 else 32 if dim <= 256 else 64 if dim <= 1024 else 256 if dim <= 4096 else 512 if dim <= 8192 else 1024
    size = max(threads, 256)
    each = size // threads
    groups = min(-(-rows // each), 4 * 256 * 256 // size, max(1, (1 << 25) // dim))
    return -(-rows // (groups * each)) + each + -(-groups // 64) + 64


@pytest.mark.parametrize("rows,dim", [(1, 24), (1025, 3000), (70_001, 24), (40_003, 96), (20_003, 200), (9_001, 513), (3_001, 3000), (1_101, 12_000), (603, 17_000)])
def test_sums_over_many_rows(lo, rows, dim):
    """A row that is left out or counted twice is seen: the bound is that of the additions that there are, and sums of whole numbers are exact."""
    g = gen(63)
    h, w = normal((rows, dim), F32, g, 2.0), normal((1, dim), F32, g)[0]
    for dtype in (F32, BF16):
        dy = torch.randint(-8, 9, (rows, dim), device="cuda", generator=g).to(dtype)
        _, dw, db = lo.layer_norm_grad(dy, h, w, bias_dtype=F32)
        assert torch.equal(db.double(), dy.double().sum(dim=0))           # (below 2^24 in magnitude)
        _, t, _, _, t_off = layer_reference(h, None, None, None, 1e-5)
        terms = dy.double() * t
        bound = terms.abs().sum(dim=0) * (depth_of(rows, dim) + 2) * E + (dy.double().abs() * t_off).sum(dim=0)
        want = terms.sum(dim=0)
        within(dw, want, want.abs() * U[F32] + bound * 1.01 + TINY[F32], "dw")


@pytest.mark.parametrize("dim", [5, 100, 3001, 20_001])
def test_an_eps_beside_squares_that_overflow(lo, dim):
    """Variance and eps, each in the range of float32 or not, whose sum is beyond it."""
    g = gen(64)
    x, w, b, dy = normal((9, dim), F32, g), normal((1, dim), F32, g)[0], normal((1, dim), F32, g)[0], normal((9, dim), F32, g)
    for scale, eps in ((1e19, 3e38), (3e18, 3.4e38), (1e20, 3e38), (1e21, 1e38)):
        check_layer_norm(lo, x * scale, w, b, None, eps, F32, (dim, scale, eps))
        check_layer_grad(lo, dy, x * scale, w, eps, None, (dim, scale, eps))
