"""Layer norm, gated product, embedding and clipping (layer_ops) against their formulas in 64 bits.

Tolerances come from the arithmetic, as in test_gpu_layer_ops: u(T) is half the distance from 1 to the next value of a type; a sum of n terms
in 32 bits is off by at most n 2^-24 of the sum of its terms' magnitudes, whatever its order."""
import math

import pytest

from test_gpu_layer_ops import (ACTS, BIG, BF16, DIMS, E, E4M3, F16, F32, I8, SHAPES, TINY, U, act64, act_grad64, eight_within, gen, normal,  # noqa: F401
                                within)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lo():
    from liteform_ae_amd import layer_ops
    return layer_ops


# --------------------------------------------------------------------------- layer norm


def layer_reference(x, w, b, res, eps):
    """h, t, y, 1 / sigma and what t may be off by: sums of up to 100 terms one after the other, those of 64 lanes and 16 wavefronts, and h's rounding."""
    h = x.double() if res is None else x.double() + res.double()
    mean = h.mean(dim=1, keepdim=True)
    s = 1.0 / torch.sqrt((h - mean).square().mean(dim=1, keepdim=True) + eps)
    t = (h - mean) * s
    y = t * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    t_off = 160 * E * (1 + t.abs()) + (0.0 if res is None else 2 * E * s * (h.abs() + h.abs().mean(dim=1, keepdim=True)))
    return h, t, y, s, t_off


def check_layer_norm(lo, x, w, b, res, eps, out, what):
    h64, _, y64, _, t_off = layer_reference(x, w, b, res, eps)
    r = lo.layer_norm(x, w, b, residual=res, eps=eps, out_dtype=out)
    y, h = (r, None) if res is None else r
    assert y.dtype is out and y.is_contiguous()
    y_off = t_off * (1.0 if w is None else w.double().abs()) + 2 * E * (y64.abs() + (0.0 if b is None else b.double().abs()))
    within(y, y64, y64.abs() * U[out] + y_off * (1 + U[out]) + TINY[out], f"y, {what}")
    if h is not None:
        assert h.dtype is res.dtype
        within(h, h64, h64.abs() * (U[res.dtype] + E) + TINY[res.dtype], f"h, {what}")


@pytest.mark.parametrize("x_type,res_type,out", [(F32, None, F32), (F32, F32, F32), (BF16, BF16, BF16), (F32, BF16, BF16), (F16, F32, F16), (BF16, F16, F32), (F16, None, BF16)])
def test_layer_norm(lo, x_type, res_type, out):
    g = gen(1)
    for i, dim in enumerate(DIMS):
        rows, pad = 1 + i % 5, (0, 3, 8)[i % 3]
        x = normal((rows, dim), x_type, g, 2.0, pad, i % 2)
        res = None if res_type is None else normal((rows, dim), res_type, g, 3.0, pad)
        w = None if i % 7 == 6 else normal((1, dim), (F32, BF16, F16)[i % 3], g)[0].contiguous()
        b = None if i % 5 == 4 else normal((1, dim), (BF16, F16, F32)[i % 3], g)[0].contiguous()
        check_layer_norm(lo, x, w, b, res, 1e-5, out, dim)


def test_layer_norm_of_many_rows(lo):
    """More rows than the workgroups take at once, in rows of every number of threads."""
    g = gen(2)
    for rows, dim in [(70_001, 24), (40_000, 96), (20_003, 200), (9_001, 513), (3_000, 3000), (1_100, 12_000)]:
        x, res, w, b = normal((rows, dim), BF16, g), normal((rows, dim), BF16, g), normal((1, dim), BF16, g)[0], normal((1, dim), BF16, g)[0]
        check_layer_norm(lo, x, w, b, res, 1e-5, BF16, (rows, dim))


@pytest.mark.parametrize("dim", [3, 100, 513, 5000, 20_001])
def test_layer_norm_of_rows_far_from_zero(lo, dim):
    """Rows of 1000 and a little: the mean keeps what is left of it (a float32 mean alone is off by 3e-5, here 1 % of sigma)."""
    g = gen(3)
    x = normal((9, dim), F32, g, 3e-3)
    x += 1000.0
    check_layer_norm(lo, x, None, None, None, 0.0 if dim > 3 else 1e-12, F32, dim)
    dy = normal((9, dim), F32, g)
    check_layer_grad(lo, dy, x, None, 0.0 if dim > 3 else 1e-12, None, dim)


def test_layer_norm_of_equal_elements(lo):
    """What is left of (h - mean) is at most the rounding of the mean's correction, far below sqrt(eps)."""
    for dim in (1, 2, 7, 8, 100, 1000, 5000, 20_001):
        for value in (0.0, 1.0, 0.1, -1000.3, 3e38, 1e-40):
            x = torch.full((3, dim), value, device="cuda")
            b = torch.arange(dim, device="cuda", dtype=F32)
            y = lo.layer_norm(x, None, b, eps=1e-5)
            within(y, b.double().expand(3, dim), 2 * E * b.double().abs() + 1e-5, f"{dim} of {value}")


@pytest.mark.parametrize("dim", [5, 300, 3000, 20_001])
def test_layer_norm_of_rows_that_leave_the_range(lo, dim):
    """Squares, or the sum itself, overflow; squares vanish (without eps)."""
    g = gen(4)
    x = normal((6, dim), F32, g)
    x.clamp_(-4, 4)
    x[0] *= 8e37
    x[1] *= 1e25
    x[2] *= 1e-25
    x[3] *= 1e-30
    x[4] = x[4].abs() * 1e37 + 3e38
    w, b = normal((1, dim), F32, g)[0], normal((1, dim), F32, g)[0]
    x = torch.nan_to_num(x, posinf=3.4e38)
    check_layer_norm(lo, x, w, b, None, 0.0, F32, dim)
    # (row 4 lies ten sigma and more from zero: what the rounding of h itself would be, is in no bound, h being given)
    dy = normal((6, dim), F32, g)
    check_layer_grad(lo, dy, x[:4], w, 0.0, None, dim, dy4=True)


def test_layer_norm_keeps_inf_and_nan_in_their_rows(lo):
    g = gen(5)
    for dim in (7, 100, 700, 3000, 20_000):
        x, w, b = normal((5, dim), F32, g), normal((1, dim), F32, g)[0], normal((1, dim), F32, g)[0]
        x[1, dim // 2], x[2, dim - 1], x[3, 0] = math.inf, math.nan, -math.inf
        y = lo.layer_norm(x, w, b)
        assert bool(torch.isnan(y[1:4]).all())
        keep = [0, 4]
        _, _, y64, _, off = layer_reference(x[keep], w, b, None, 1e-5)
        within(y[keep], y64, off * w.double().abs() + 4 * E * (y64.abs() + b.double().abs()))
        q, scale = lo.layer_norm_8bit(x, w, b)
        assert bool(torch.isnan(scale[1:4]).all()) and bool(torch.isfinite(scale[keep]).all())


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("x_type,res_type", [(F32, None), (BF16, BF16), (F16, F32)])
def test_layer_norm_8bit(lo, x_type, res_type, dtype):
    g = gen(6)
    for i, dim in enumerate(DIMS):
        if dim == 1:
            continue                                                     # (y is b: nothing to scale)
        rows = 1 + i % 4
        x = normal((rows, dim), x_type, g, 2.0, i % 3)
        res = None if res_type is None else normal((rows, dim), res_type, g, 3.0)
        w, b = normal((1, dim), x_type, g)[0], normal((1, dim), x_type, g)[0]
        h64, _, y64, _, _ = layer_reference(x, w, b, res, 1e-5)
        q, scale, *h = lo.layer_norm_8bit(x, w, b, residual=res, eps=1e-5, dtype=dtype)
        assert q.dtype is dtype and scale.dtype is F32
        want = y64.abs().amax(dim=1)
        # the largest |y| is off by up to 160 roundings of 1 + |t|, a few of |h| / sigma; |y| of the others by as much
        off = 400 * E * (1 + y64.abs().amax(dim=1)) * (1 + w.double().abs().max())
        within(scale * (448.0 if dtype is E4M3 else 127.0), want, off + 8 * E * want, f"scale, {dim}")
        s = (want / (448.0 if dtype is E4M3 else 127.0))[:, None]
        half = s * 0.5 if dtype is I8 else torch.maximum(y64.abs() * 2.0 ** -4, s * 2.0 ** -10)
        within(q.double() * scale.double()[:, None], y64, half * (1 + 1e-3) + 2 * off[:, None], f"q, {dim}")
        if h:
            within(h[0], h64, h64.abs() * (U[res_type] + E))


def test_layer_norm_of_no_rows(lo):
    x = torch.empty((0, 64), device="cuda")
    y, h = lo.layer_norm(x, residual=x)
    assert y.shape == h.shape == (0, 64)
    q, s = lo.layer_norm_8bit(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    dx, dw, db = lo.layer_norm_grad(x, x, torch.ones(64, device="cuda"), bias_dtype=BF16)
    assert dx.shape == (0, 64) and bool((dw == 0).all()) and bool((db == 0).all()) and db.dtype is BF16


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_where_h_is_the_residual(lo, dtype):
    """The library may write h where the residual was; rows whose end reaches back into the piece before, which another wavefront may hold."""
    import ctypes as C
    from liteform_ae_amd import _lib
    lib, code = _lib.load(), {F32: _lib.LF_DTYPE_F32, BF16: _lib.LF_DTYPE_BF16}[dtype]
    g = gen(10)
    for dim in (5, 63, 513, 1025, 1540, 2049, 2050, 4095, 4097, 6150, 8191, 10_001, 16_383, 20_001):
        x, res = normal((700, dim), dtype, g), normal((700, dim), dtype, g)
        y, h = lo.layer_norm(x, residual=res, eps=1e-5)
        y2 = torch.empty_like(y)
        a = _lib.LayerNormArgs(x=x.data_ptr(), residual=res.data_ptr(), y=y2.data_ptr(), h=res.data_ptr(), ld_x=dim, ld_residual=dim, ld_y=dim, ld_h=dim, rows=700, dim=dim,
                               x_dtype=code, residual_dtype=code, y_dtype=code, eps=1e-5)
        _lib.check(lib.lf_layer_norm(C.byref(a), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(res, h) and torch.equal(y2, y), dim


def check_layer_grad(lo, dy, h, w, eps, dh, what, bias=F32, dy4=False):
    if dy4:
        dy = dy[:4]
    dx, dw, db = lo.layer_norm_grad(dy, h, w, eps=eps, dh=dh, bias_dtype=bias)
    h64, t, _, s, t_off = layer_reference(h, None, None, None, eps)
    dy64, rows = dy.double(), dy.shape[0]
    g = dy64 * (1.0 if w is None else w.double())
    mean = lambda v: v.mean(dim=1, keepdim=True)  # noqa: E731
    own = s * (g - mean(g) - t * mean(g * t))
    want = own + (0.0 if dh is None else dh.double())
    sums = 160 * E                                                       # as in layer_reference
    off = s * (4 * E * g.abs() + sums * mean(g.abs()) + t.abs() * (sums * mean((g * t).abs()) + mean(g.abs() * t_off)) + t_off * mean(g * t).abs())
    off = off + sums * own.abs() + 4 * E * want.abs() + (0.0 if dh is None else E * dh.double().abs())
    within(dx, want, want.abs() * U[h.dtype] + off * (1 + U[h.dtype]) + TINY[h.dtype], f"dx, {what}")
    if w is not None:
        want = (dy64 * t).sum(dim=0)
        off = (dy64 * t).abs().sum(dim=0) * (rows + 24) * E + (dy64.abs() * t_off).sum(dim=0)
        within(dw, want, want.abs() * U[w.dtype] + off * 1.01 + TINY[w.dtype], f"dw, {what}")
    if bias is not None:
        want = dy64.sum(dim=0)
        assert db.dtype is bias
        within(db, want, want.abs() * U[bias] + dy64.abs().sum(dim=0) * (rows + 24) * E * 1.01 + TINY[bias], f"db, {what}")


@pytest.mark.parametrize("dy_type,h_type", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16)])
def test_layer_norm_grad(lo, dy_type, h_type):
    g = gen(7)
    for i, dim in enumerate(DIMS):
        rows, pad = (1, 4, 37, 300)[i % 4], (0, 3, 8)[i % 3]
        h, dy = normal((rows, dim), h_type, g, 2.0, pad, i % 2), normal((rows, dim), dy_type, g, 1.0, pad)
        w = None if i % 7 == 6 else normal((1, dim), (F32, BF16, F16)[i % 3], g)[0].contiguous()
        dh = None if i % 3 == 0 else normal((rows, dim), h_type, g, 1.0, pad)
        check_layer_grad(lo, dy, h, w, 1e-5, dh, dim, (None, F32, BF16)[i % 3])


def test_layer_norm_grad_of_many_rows(lo):
    g = gen(8)
    for rows, dim in [(70_001, 24), (40_000, 96), (20_003, 200), (9_001, 513), (3_000, 3000), (1_100, 12_000), (600, 17_000)]:
        h, dy, dh = (normal((rows, dim), BF16, g) for _ in range(3))
        w = normal((1, dim), BF16, g)[0]
        check_layer_grad(lo, dy, h, w, 1e-5, dh, (rows, dim), BF16)


def test_layer_norm_grad_against_differences(lo):
    """The derivative of sum(dy y) along a direction, by differences of the formula in 64 bits."""
    g = gen(9)
    for dim in (9, 130, 1000):
        x, dy, w, b = normal((4, dim), F32, g), normal((4, dim), F32, g), normal((1, dim), F32, g)[0], normal((1, dim), F32, g)[0]
        dx, dw, db = lo.layer_norm_grad(dy, x, w, bias_dtype=F32)
        args = [x.double(), w.double(), b.double()]
        for i, grad in enumerate((dx, dw, db)):
            along, step = torch.randn(args[i].shape, device="cuda", dtype=torch.float64, generator=g), 1e-5

            def loss(sign):
                moved = [v + sign * step * along if j == i else v for j, v in enumerate(args)]
                return (layer_reference(moved[0], moved[1], moved[2], None, 1e-5)[2] * dy.double()).sum()

            slope = float((loss(1) - loss(-1)) / (2 * step))
            # differences are off by step^2 of the third derivative, gradients by some 100 roundings of a sum of 4 dim terms of about one
            assert abs(float((grad.double() * along).sum()) - slope) <= 1e-4 * math.sqrt(4 * dim)


# --------------------------------------------------------------------------- gated product


def check_gated(lo, shape, x_type, act, bias, out, g, pad=0, offset=0):
    m, n, k = shape
    x = normal((m, k), x_type, g, 1.0, pad, offset)
    w = normal((2 * n, k), x_type, g, max(k, 1) ** -0.5, pad, offset)
    b = None if bias is None else normal((1, 2 * n), bias, g)[0]
    y, z = lo.gated_linear(x, w, b, activation=act, out_dtype=out, return_preactivation=True)
    assert y.shape == (m, n) and z.shape == (m, 2 * n) and y.dtype is out and z.dtype is x_type
    x64, w64 = x.double(), w.double()
    z64 = x64 @ w64.t() + (0.0 if b is None else b.double())
    # sums in 32 bits of products that are exact (16 bits) or off by 2^-22 (float32: what is left of the cut), the bias among them
    z_off = (x64.abs() @ w64.abs().t() + (0.0 if b is None else b.double().abs())) * (k + 24) * E
    within(z, z64, z64.abs() * U[x_type] + z_off + TINY[x_type], f"z {shape}")
    gate_within(y, z64, z_off, act, out, f"y {shape}")
    assert torch.equal(y, lo.gated_linear(x, w, b, activation=act, out_dtype=out))


def gate_within(y, z64, z_off, act, out, what):
    n = z64.shape[1] // 2
    g64, u64 = z64[:, :n], z64[:, n:]
    a64 = act64(g64, act)
    a_off = z_off[:, :n] if act is None else 1.13 * z_off[:, :n] + (g64.abs() + 1) * 16 * E      # |act'| <= 1.13, exp and erf to a few units
    y64 = a64 * u64
    off = a_off * (u64.abs() + z_off[:, n:]) + a64.abs() * z_off[:, n:] + E * y64.abs()
    within(y, y64, y64.abs() * U[out] + off * (1 + U[out]) + TINY[out], what)


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_gated(lo, x_type):
    g = gen(11)
    for i, shape in enumerate(SHAPES):
        check_gated(lo, shape, x_type, ACTS[i % 4], (None, x_type, F32)[i % 3], (x_type, F32)[i % 5 == 4], g)


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_gated_of_rows_inside_wider_buffers(lo, x_type):
    g = gen(12)
    for i, shape in enumerate(SHAPES[:-2]):
        check_gated(lo, shape, x_type, ACTS[(i + 1) % 4], x_type, x_type, g, pad=(1, 8, 3)[i % 3], offset=(0, 1, 8, 5)[i % 4])


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_gated_of_many_tiles(lo, x_type):
    g = gen(13)
    for i, shape in enumerate(BIG):
        check_gated(lo, shape, x_type, ACTS[i + 2], x_type, x_type, g)
        check_gated(lo, shape, x_type, "relu", None, F32, g)
        check_gated(lo, shape, x_type, "silu", None, x_type, g, pad=3, offset=1)


# outputs that end inside a tile of each size, before, at and after the middle of one
@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_gated_at_the_ends_of_tiles(lo, x_type):
    g = gen(14)
    for n in (15, 16, 17, 31, 32, 33, 47, 48, 64, 80, 127, 128, 129, 144):
        for m, k in ((40, 72), (130, 136), (2100, 64)):
            check_gated(lo, (m, n, k), x_type, "silu", x_type, x_type, g)


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_gated_of_long_sums(lo, x_type):
    """Few outputs, many products: k is cut up."""
    g = gen(15)
    for shape in [(40, 30, 40_000), (130, 100, 20_007), (16, 16, 100_003), (300, 20, 9_000), (1, 24, 30_000)]:
        check_gated(lo, shape, x_type, "gelu", x_type, x_type, g)


@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_gated_8bit(lo, dtype):
    g = gen(16)
    for i, (m, n, k) in enumerate(SHAPES + BIG + [(40, 30, 40_000), (130, 100, 20_007)]):
        pad, out = (0, 3, 16)[i % 3], (BF16, F32, F16)[i % 3]
        x, sx = lo.quantize_rows(normal((m, max(k, 1)), F32, g), dtype)
        w, sw = lo.quantize_rows(normal((2 * n, max(k, 1)), F32, g, max(k, 1) ** -0.5), dtype)
        wide = torch.zeros((m, k + pad), device="cuda", dtype=dtype)
        wide[:, :k] = x[:, :k]
        x, w = wide[:, :k], w[:, :k]
        b = None if i % 2 else normal((1, 2 * n), F32, g)[0]
        act = ACTS[i % 4]
        y = lo.gated_linear_8bit(x, sx, w, sw, b, activation=act, out_dtype=out)
        x64, w64 = x.double() * sx.double()[:, None], w.double() * sw.double()[:, None]
        z64 = x64 @ w64.t() + (0.0 if b is None else b.double())
        # (as for linear_8bit)
        off = (x64.abs() @ w64.abs().t()) * (8 * E if dtype is I8 else 2.0 ** -10 + (k + 16) * E) + (0.0 if b is None else b.double().abs()) * 4 * E
        gate_within(y, z64, off + z64.abs() * 4 * E, act, out, f"{(m, n, k)}")


def test_gated_keeps_inf_and_nan(lo):
    """Of x in their rows; of a weight in their columns, whether of the gate or of the other half."""
    g = gen(17)
    for x_type in (F32, BF16, F16):
        for m, n, k in [(5, 30, 100), (90, 70, 333), (300, 200, 256)]:
            x, w = normal((m, k), x_type, g), normal((2 * n, k), x_type, g)
            x[1, 2] = math.nan
            w[3, 5], w[n + 7, 6] = math.nan, math.inf
            y = lo.gated_linear(x, w, activation=None)
            bad = torch.zeros((m, n), dtype=torch.bool, device="cuda")
            bad[1] = bad[:, 3] = bad[:, 7] = True
            assert bool((~torch.isfinite(y[bad])).all()) and bool(torch.isfinite(y[~bad]).all())
            assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[:, 3]).all())


def check_gated_grad(lo, shape, x_type, act, bias, g, pad=0, offset=0):
    m, n, k = shape
    x, w = normal((m, k), x_type, g, 1.0, pad, offset), normal((2 * n, k), x_type, g, 1.0, pad)
    dy, z = normal((m, n), x_type, g, 1.0, pad, offset), normal((m, 2 * n), x_type, g, 1.0, offset)
    dx, dw, db = lo.gated_linear_grad(dy, x, w, z, activation=act, bias_dtype=bias)
    g64, u64, dy64 = z[:, :n].double(), z[:, n:].double(), dy.double()
    dz = torch.cat([dy64 * u64 * act_grad64(g64, act), dy64 * act64(g64, act)], dim=1)
    # dz as the products take it: rounded to the type; the activation and its derivative are known to 16 units
    units = torch.cat([dy64.abs() * u64.abs(), dy64.abs() * (1 + g64.abs())], dim=1) * 16 * E
    dz_off = dz.abs() * (U[x_type] + 2 * E) + units + TINY[x_type]
    x64, w64 = x.double(), w.double()
    off = (dz.abs() @ w64.abs()) * (2 * n + 24) * E + (dz_off @ w64.abs()) * 1.001
    want = dz @ w64
    within(dx, want, want.abs() * U[x_type] + off + TINY[x_type], f"dx {shape}")
    off = (dz.abs().t() @ x64.abs()) * (m + 24) * E + (dz_off.t() @ x64.abs()) * 1.001
    want = dz.t() @ x64
    within(dw, want, want.abs() * U[x_type] + off + TINY[x_type], f"dw {shape}")
    if bias is None:
        assert db is None
        return
    assert db.dtype is bias
    want = dz.sum(dim=0)
    off = dz.abs().sum(dim=0) * (m + 24) * E + units.sum(dim=0) * 1.001
    within(db, want, want.abs() * U[bias] + off + TINY[bias], f"db {shape}")


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_gated_grad(lo, x_type):
    g = gen(18)
    for i, shape in enumerate(SHAPES):
        check_gated_grad(lo, shape, x_type, ACTS[i % 4], (None, x_type, F32)[i % 3], g, pad=(0, 3, 8)[i % 3], offset=(0, 1, 8)[i % 3])


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_gated_grad_of_many_tiles(lo, x_type):
    g = gen(19)
    for i, shape in enumerate([(2100, 1030, 520), (5000, 1000, 300), (9000, 33, 70)]):
        check_gated_grad(lo, shape, x_type, ACTS[1 + i], x_type, g)


def test_gated_grad_of_what_is_wanted(lo):
    g = gen(20)
    x, w, dy, z = normal((70, 40), BF16, g), normal((60, 40), BF16, g), normal((70, 30), BF16, g), normal((70, 60), BF16, g)
    dx, dw, db = lo.gated_linear_grad(dy, x, w, z, bias_dtype=F32)
    for want in range(8):
        got = lo.gated_linear_grad(dy, x, w, z, bias_dtype=F32 if want & 4 else None, want_dx=bool(want & 1), want_dweight=bool(want & 2))
        for bit, a, b in zip((1, 2, 4), got, (dx, dw, db)):
            assert (a is None) == (not want & bit) and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("act", ACTS)
def test_gated_grad_against_differences(lo, act):
    g = gen(21)
    m, n, k = 11, 20, 30
    x, w, b, dy = normal((m, k), F32, g), normal((2 * n, k), F32, g, k ** -0.5), normal((1, 2 * n), F32, g)[0], normal((m, n), F32, g)
    _, z = lo.gated_linear(x, w, b, activation=act, return_preactivation=True)
    grads = lo.gated_linear_grad(dy, x, w, z, activation=act, bias_dtype=F32)
    args = [x.double(), w.double(), b.double()]
    for i, grad in enumerate(grads):
        along, step = torch.randn(args[i].shape, device="cuda", dtype=torch.float64, generator=g), 1e-6

        def loss(sign):
            moved = [v + sign * step * along if j == i else v for j, v in enumerate(args)]
            t = moved[0] @ moved[1].t() + moved[2]
            return (act64(t[:, :n], act) * t[:, n:] * dy.double()).sum()

        slope = float((loss(1) - loss(-1)) / (2 * step))
        # (a corner of relu that a step passes changes the difference by at most the step, 1e-6, times dy u)
        assert abs(float((grad.double() * along).sum()) - slope) <= 1e-3 * math.sqrt(along.numel())


@pytest.mark.parametrize("x_type", [F32, BF16])
def test_gated_of_sizes_of_zero(lo, x_type):
    for m, n, k in [(0, 5, 7), (4, 0, 7), (4, 5, 0), (0, 0, 7), (0, 5, 0), (4, 0, 0)]:
        x, w = torch.ones((m, k), device="cuda", dtype=x_type), torch.ones((2 * n, k), device="cuda", dtype=x_type)
        b = torch.full((2 * n,), 2.0, device="cuda", dtype=x_type)
        y, z = lo.gated_linear(x, w, b, activation=None, return_preactivation=True)
        assert y.shape == (m, n) and z.shape == (m, 2 * n)
        assert bool((y == (k + 2) ** 2).all())
        dx, dw, db = lo.gated_linear_grad(torch.ones((m, n), device="cuda", dtype=x_type), x, w, z, activation=None, bias_dtype=F32)
        assert dx.shape == (m, k) and dw.shape == (2 * n, k) and db.shape == (2 * n,)
        assert bool((dx == 2 * n * (k + 2)).all()) and bool((dw == m * (k + 2)).all()) and bool((db == m * (k + 2)).all())


# --------------------------------------------------------------------------- embedding


def ids_of(n, rows, g, spread="even", dtype=torch.int64, bad=True):
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    v = (u * rows if spread == "even" else rows ** u - 1).long().clamp_(0, max(rows - 1, 0))
    if bad and n > 3:
        v[::5] = torch.tensor([-1, rows, -(1 << 31), (1 << 31) - 1], device="cuda")[torch.arange(len(v[::5]), device="cuda") % 4]
    return v.to(dtype)


@pytest.mark.parametrize("x_type,out", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, F32)])
def test_embedding(lo, x_type, out):
    g = gen(31)
    for i, dim in enumerate([1, 2, 7, 8, 9, 63, 64, 65, 100, 128, 200, 256, 257, 500, 512, 1000, 1030, 4096, 5001]):
        n, rows = (1, 5, 64, 300, 1000)[i % 5], (1, 47, 1000)[i % 3]
        table = normal((rows, dim), x_type, g, 1.0, (0, 3, 8)[i % 3], i % 2)
        ids = ids_of(n, rows, g, dtype=(torch.int64, torch.int32)[i % 2])
        scale = (1.0, math.sqrt(dim), -0.3)[i % 3]
        y = lo.embedding(ids, table, scale=scale, out_dtype=out)
        assert y.dtype is out and y.shape == (n, dim) and y.is_contiguous()
        wide = ids.long()
        on = (wide >= 0) & (wide < rows)
        want = torch.where(on[:, None], table.double()[torch.where(on, wide, 0)] * scale, 0.0)
        # the scale and the product are rounded to 32 bits, then y
        within(y, want, want.abs() * (U[out] + 3 * E) + TINY[out], f"{dim}")
        assert bool((y[~on] == 0).all())


def test_embedding_of_ids_in_a_wider_buffer(lo):
    g = gen(32)
    table = normal((50, 40), F32, g)
    for dtype in (torch.int64, torch.int32):
        wide = torch.randint(0, 50, (64, 3), device="cuda", generator=g).to(dtype)
        for ids in (wide[:, 1], wide[:, 2], wide[::2, 0], wide[0, :1].expand(9)):
            assert torch.equal(lo.embedding(ids, table), table[ids.long()])
            dy = normal((ids.shape[0], 40), F32, g)
            assert torch.equal(lo.embedding_grad(dy, ids, 50), lo.embedding_grad(dy, ids.contiguous(), 50))


def check_embedding_grad(lo, ids, rows, dim, dy_type, out, scale, g, pad=0, offset=0, what=""):
    n = ids.shape[0]
    dy = normal((n, dim), dy_type, g, 1.0, pad, offset)
    got = lo.embedding_grad(dy, ids, rows, scale=scale, out_dtype=out)
    assert got.shape == (rows, dim) and got.dtype is out
    wide = ids.long()
    on = (wide >= 0) & (wide < rows)
    want = torch.zeros((rows, dim), device="cuda", dtype=torch.float64).index_add_(0, wide[on], dy[on].double())
    size = torch.zeros((rows, dim), device="cuda", dtype=torch.float64).index_add_(0, wide[on], dy[on].double().abs())
    count = torch.bincount(wide[on], minlength=rows)[:rows, None]
    bound = (want * scale).abs() * U[out] + size * abs(scale) * (count + 4) * E + (count > 0) * TINY[out]
    within(got, want * scale, bound, f"{what} {n} ids of {rows}, {dim}")
    assert torch.equal(got, lo.embedding_grad(dy, ids, rows, scale=scale, out_dtype=out))


#       ids, rows: none, one; one and more digits of the sort; one tile of it, some, and more workgroups than one
GRADS = [(0, 10), (1, 1), (1, 70_000), (5, 3), (63, 1000), (64, 2047), (65, 2048), (700, 5), (1000, 4000), (4095, 100), (4096, 3_000_000), (4097, 2_000), (8192, 70_000), (8193, 70_000),
         (20_000, 50_000), (100_001, 30_000), (300_000, 1), (300_000, 9), (9000, 5_000_000), (2_500_001, 1_000_000)]


@pytest.mark.parametrize("dy_type,out", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16)])
def test_embedding_grad(lo, dy_type, out):
    g = gen(33)
    for i, (n, rows) in enumerate(GRADS):
        dim = (1, 8, 33, 64, 100, 130, 257)[i % 7] if rows * 257 < 1e8 else 12
        ids = ids_of(n, rows, g, ("even", "zipf")[i % 2], (torch.int64, torch.int32)[i % 2], bad=i % 3 != 0)
        check_embedding_grad(lo, ids, rows, dim, dy_type, out, (1.0, 11.3, -0.2)[i % 3], g, (0, 3, 8)[i % 3], i % 2)


@pytest.mark.parametrize("dy_type", [F32, BF16])
def test_embedding_grad_of_wide_rows(lo, dy_type):
    g = gen(34)
    for n, rows, dim in [(3000, 200, 513), (3000, 4000, 1024), (12_000, 40, 2000), (500, 900, 5001), (30_000, 2, 600)]:
        check_embedding_grad(lo, ids_of(n, rows, g, "zipf"), rows, dim, dy_type, dy_type, 2.0, g)


def test_embedding_grad_of_special_ids(lo):
    g = gen(35)
    for n, dim in [(10, 100), (5000, 24), (40_000, 64), (20_000, 600)]:
        for ids in (torch.full((n,), 7, device="cuda"), torch.full((n,), -1, device="cuda"), torch.full((n,), 999, device="cuda"), torch.full((n,), 0, device="cuda"),
                    torch.arange(n, device="cuda") % 1000, torch.arange(n, device="cuda") * 1000 // n, 999 - torch.arange(n, device="cuda") * 1000 // n):
            check_embedding_grad(lo, ids, 1000, dim, F32, F32, 1.0, g)


def test_embedding_grad_against_differences(lo):
    g = gen(36)
    table, ids = normal((30, 9), F32, g), ids_of(200, 30, g)
    dy = normal((200, 9), F32, g)
    grad = lo.embedding_grad(dy, ids, 30, scale=3.0)
    along = normal((30, 9), F32, g)
    # (linear: the difference is the slope, off by the roundings of 1800 terms of about 3)
    slope = ((lo.embedding(ids, table + along, scale=3.0).double() - lo.embedding(ids, table, scale=3.0).double()) * dy.double()).sum()
    assert abs(float((grad.double() * along.double()).sum() - slope)) <= 1800 * 3 * 10 * E * 4


def test_embedding_of_tables_past_32_bits(lo):
    """Offsets of 64 bits: a table of more than 2^32 bytes, and gradients of it."""
    rows, dim = 1_200_000, 1024
    table = torch.zeros((rows, dim), device="cuda", dtype=F32)
    ids = torch.tensor([rows - 1, 0, 600_000, 1_048_577, rows], device="cuda")
    table[ids[:4]] = torch.arange(1, 5, device="cuda", dtype=F32)[:, None]
    y = lo.embedding(ids, table)
    assert y[:, 0].tolist() == [1, 2, 3, 4, 0] and bool((y == y[:, :1]).all())
    del table
    grad = lo.embedding_grad(y, ids, rows)
    assert torch.equal(grad[ids[:4]], y[:4]) and float(grad.sum(dtype=torch.float64)) == 10 * dim


def test_embedding_of_nothing(lo):
    table, none = torch.ones((5, 8), device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    assert lo.embedding(none, table).shape == (0, 8)
    assert bool((lo.embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), table[:0]) == 0).all())
    grad = lo.embedding_grad(table[:0], none, 6)
    assert grad.shape == (6, 8) and bool((grad == 0).all())
    assert lo.embedding_grad(table, torch.zeros(5, dtype=torch.int32, device="cuda"), 0).shape == (0, 8)


def test_embedding_grad_keeps_inf_and_nan_in_their_rows(lo):
    ids = torch.tensor([0, 1, 2, 1, 3, -1], device="cuda")
    dy = torch.ones((6, 20), device="cuda")
    dy[1, 3], dy[2, 4], dy[5] = math.inf, math.nan, math.nan
    grad = lo.embedding_grad(dy, ids, 5)
    want = torch.tensor([1.0, 2.0, 1.0, 1.0, 0.0], device="cuda")[:, None].repeat(1, 20)
    want[1, 3], want[2, 4] = math.inf, math.nan
    assert torch.equal(torch.nan_to_num(grad, nan=-7.0), torch.nan_to_num(want, nan=-7.0))


# --------------------------------------------------------------------------- norm of all gradients


def check_clip(lo, grads, most, eps=1e-6):
    before = [t.clone() for t in grads]
    norm64 = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
    norm = lo.gradient_norm(grads)
    assert norm.dtype is F32 and norm.shape == ()
    # squares and their sum are in 64 bits: the root is rounded once
    assert abs(float(norm) - norm64) <= (E + 1e-12) * norm64 + 2.0 ** -149
    clipped, again = lo.clip_gradients(grads, most, eps=eps)
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(grads, before))
    factor = 1.0 if norm64 == 0 else min(1.0, most / (norm64 + eps))
    for t, c in zip(grads, clipped):
        assert c.shape == t.shape and c.dtype is t.dtype
        # norm, sum, quotient and product are rounded, then the result
        within(c.reshape(-1, 1), t.double().reshape(-1, 1) * factor, (t.double().abs() * factor * (U[t.dtype] + 6 * E) + TINY[t.dtype]).reshape(-1, 1))
    inplace, third = lo.clip_gradients(grads, most, eps=eps, in_place=True)
    assert all(a is b for a, b in zip(inplace, grads)) and torch.equal(third, norm)
    assert all(torch.equal(a, b) for a, b in zip(inplace, clipped))


@pytest.mark.parametrize("most", [1e-3, 1.0, 1e9, 0.0, math.inf])
def test_clip(lo, most):
    g = gen(41)
    for shapes in ([(1,)], [(7,)], [(8,)], [(100_003,)], [(3, 5), (128,), (128, 128), (1, 1)], [(2, 3, 4, 5), (0,), (0, 4), (4, 0), (16384,), (16385,), (16383,)],
                   [(17, 31)] * 200, [(), (3_000_001,), (512, 1024)]):
        for kinds in ((F32,), (BF16,), (F16,), (F32, BF16, F16)):
            check_clip(lo, [torch.randn(s, device="cuda", generator=g).to(kinds[i % len(kinds)]) for i, s in enumerate(shapes)], most)


def test_clip_of_rows_inside_wider_buffers(lo):
    g = gen(42)
    wide = torch.randn((70, 50), device="cuda", generator=g)
    keep = wide.clone()
    check_clip(lo, [wide[:, :20], wide[:, 20:49], wide[:69, 49:]], 1.0)
    assert bool((wide[69, 49:] == keep[69, 49:]).all())                  # (what lies outside is left alone)
    for off in (0, 1, 3):
        flat = torch.randn(3000, device="cuda", generator=g).to(BF16)
        keep = flat.clone()
        check_clip(lo, [flat[off:off + 1000], flat[1000 + off:1000 + off + 77], flat[2001:2002]], 0.5)
        rest = torch.ones(3000, dtype=torch.bool, device="cuda")
        rest[off:off + 1000] = rest[1000 + off:1077 + off] = rest[2001] = False
        assert torch.equal(flat[rest], keep[rest])


def test_clip_of_large_and_small_values(lo):
    """Squares beyond the range of 32 bits, either way."""
    g = gen(43)
    for scale in (1e30, 1e-30, 1e-42):
        check_clip(lo, [torch.randn(1000, device="cuda", generator=g) * scale, torch.randn((20, 30), device="cuda", generator=g) * scale], scale, eps=0.0 if scale < 1 else 1e-6)
    check_clip(lo, [torch.zeros(100, device="cuda"), torch.zeros((4, 4), device="cuda", dtype=BF16)], 1.0)
    check_clip(lo, [torch.zeros(100, device="cuda")], 0.0, eps=0.0)
    check_clip(lo, [], 1.0)


def test_clip_of_inf_and_nan(lo):
    a, b = torch.ones(100, device="cuda"), torch.ones((5, 5), device="cuda", dtype=BF16)
    a[3] = math.nan
    clipped, norm = lo.clip_gradients([a, b], 1.0)
    assert math.isnan(float(norm)) and all(bool(torch.isnan(t).all()) for t in clipped)
    a[3] = -math.inf
    clipped, norm = lo.clip_gradients([a, b], 1.0)
    assert float(norm) == math.inf and bool(torch.isnan(clipped[0][3])) and bool((clipped[1] == 0).all()) and int(torch.isnan(clipped[0]).sum()) == 1


def test_clip_of_the_same_tensor_twice(lo):
    """Counted twice; in place it would be cut once or twice, and is refused."""
    g = gen(44)
    t = torch.randn(1000, device="cuda", generator=g)
    clipped, norm = lo.clip_gradients([t, t], 1.0)
    assert torch.equal(clipped[0], clipped[1]) and abs(float(norm) - math.sqrt(2) * float(t.double().norm())) <= 1e-5 * float(norm)
    keep = t.clone()
    for pair in ([t, t], [t, t[10:20]], [t[:500], t[499:]], [t.view(10, 100)[:, :60], t.view(10, 100)[:, 59:]], [t.view(10, 100)[:, :60], t.view(20, 50)[:, 40:]]):
        with pytest.raises(ValueError, match="lies on another"):
            lo.clip_gradients(pair, 1.0, in_place=True)
    assert torch.equal(t, keep)


def test_clip_in_place_is_seen_by_autograd(lo):
    t = torch.ones(10, device="cuda")
    version = t._version
    lo.clip_gradients([t], 1.0, in_place=True)
    assert t._version == version + 1


# --------------------------------------------------------------------------- streams, graphs, refusals


def calls(lo, g):
    x, w, w2 = normal((300, 200), BF16, g), normal((1, 200), BF16, g)[0], normal((96, 200), BF16, g)
    dy, z, ids = normal((300, 48), BF16, g), normal((300, 96), BF16, g), ids_of(9000, 500, g, "zipf")
    few, long_x, long_w = normal((3, 200), BF16, g), normal((40, 9000), BF16, g), normal((60, 9000), BF16, g)
    de, grads = normal((9000, 40), BF16, g), [normal((30, 70), F32, g) for _ in range(5)]
    rows = normal((600, 40), F32, g)
    return [lambda: lo.layer_norm(x, w, w, residual=x), lambda: lo.layer_norm_8bit(x, w, w), lambda: lo.layer_norm_grad(x, x, w, bias_dtype=F32),
            lambda: lo.gated_linear(x, w2, return_preactivation=True), lambda: (lo.gated_linear(few, w2),), lambda: (lo.gated_linear(long_x, long_w),),
            lambda: lo.gated_linear_grad(dy, x, w2, z, bias_dtype=F32), lambda: (lo.embedding(ids, rows),), lambda: (lo.embedding_grad(de, ids, 500),),
            lambda: (lo.embedding_grad(de[:3000], ids[:3000], 500),), lambda: (*lo.clip_gradients(grads, 1.0)[0], lo.gradient_norm(grads))]


def test_on_a_stream_of_its_own_and_in_a_graph(lo):
    for number, call in enumerate(calls(lo, gen(51))):
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = call()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), number
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for _ in range(3):
            for t in got:
                t.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), number
            again = call()                                               # (eager work between the replays)
            assert all(torch.equal(a, b) for a, b in zip(again, want)), number


def test_refusals(lo):
    x, w = torch.ones((4, 8), device="cuda"), torch.ones(8, device="cuda")
    cpu, ids, table = torch.ones((4, 8)), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones((5, 8), device="cuda")
    half = x.to(BF16)
    bad = [lambda: lo.layer_norm(cpu), lambda: lo.layer_norm(x, w[:7]), lambda: lo.layer_norm(x, w, w[:7]), lambda: lo.layer_norm(x, residual=x[:3]),
           lambda: lo.layer_norm(x.long()), lambda: lo.layer_norm(x, eps=-1.0), lambda: lo.layer_norm(x, out_dtype=torch.int8), lambda: lo.layer_norm_8bit(x, dtype=F32),
           lambda: lo.layer_norm(x[:, :0]), lambda: lo.layer_norm(x.t()), lambda: lo.layer_norm(x[0]),
           lambda: lo.layer_norm_grad(x, x, w[:7]), lambda: lo.layer_norm_grad(x[:3], x, w), lambda: lo.layer_norm_grad(x, x, dh=half),
           lambda: lo.layer_norm_grad(x, x, bias_dtype=torch.int8),
           lambda: lo.gated_linear(x, x[:3]), lambda: lo.gated_linear(x, x[:, :7]), lambda: lo.gated_linear(x, half), lambda: lo.gated_linear(x, x, w[:3]),
           lambda: lo.gated_linear(x, w), lambda: lo.gated_linear(x, x, activation="tanh"), lambda: lo.gated_linear(x, x, out_dtype=torch.int8),
           lambda: lo.gated_linear(x.to(E4M3), x.to(E4M3)), lambda: lo.gated_linear_8bit(x, w[:4], x, w[:4]), lambda: lo.gated_linear(x, cpu),
           lambda: lo.gated_linear_8bit(x.to(E4M3), w[:3], x.to(E4M3), w[:4]), lambda: lo.gated_linear_8bit(x.to(E4M3), w[:4], x.to(E4M3), w[:2]),
           lambda: lo.gated_linear_8bit(x.to(E4M3), w[:4], x.to(I8), w[:4]),
           lambda: lo.gated_linear_grad(x[:, :3], x, x, x[:, :4]), lambda: lo.gated_linear_grad(x[:, :2], x, x, x[:, :3]), lambda: lo.gated_linear_grad(half[:, :2], x, x, x[:, :4]),
           lambda: lo.gated_linear_grad(x[:, :2], x, x, half[:, :4]), lambda: lo.gated_linear_grad(x[:, :2], x, x, None),
           lambda: lo.embedding(ids.float(), table), lambda: lo.embedding(ids.cpu(), table), lambda: lo.embedding(ids[:, None], table), lambda: lo.embedding(ids, table[0]),
           lambda: lo.embedding(ids, table.cpu()), lambda: lo.embedding(ids, table, out_dtype=torch.int8), lambda: lo.embedding(ids, table[:, :0]),
           lambda: lo.embedding_grad(x, ids[:3], 5), lambda: lo.embedding_grad(x, ids, -1), lambda: lo.embedding_grad(x.long(), ids, 5),
           lambda: lo.clip_gradients([x, cpu], 1.0), lambda: lo.clip_gradients([x.long()], 1.0), lambda: lo.clip_gradients([x], -1.0), lambda: lo.clip_gradients([x], math.nan),
           lambda: lo.clip_gradients([x], 1.0, eps=-1.0), lambda: lo.gradient_norm([x.expand(3, 4, 8)]), lambda: lo.gradient_norm([x.t()[:, :2]])]
    for number, call in enumerate(bad):
        with pytest.raises((ValueError, AttributeError)):
            call()
            pytest.fail(f"call {number} was not refused")
    torch.cuda.synchronize()


def test_tensors_that_require_gradients(lo):
    x, w = torch.ones((4, 8), device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    plain = x.detach()
    for call in (lambda: lo.layer_norm(x), lambda: lo.layer_norm(plain, w), lambda: lo.layer_norm(plain, None, w), lambda: lo.layer_norm_8bit(x), lambda: lo.layer_norm_grad(x, plain),
                 lambda: lo.gated_linear(x, plain), lambda: lo.gated_linear(plain, x), lambda: lo.gated_linear_grad(x[:, :2], plain, plain, plain[:, :4]),
                 lambda: lo.embedding(ids, x), lambda: lo.embedding_grad(x, ids, 3), lambda: lo.clip_gradients([x], 1.0), lambda: lo.gradient_norm([x])):
        with pytest.raises(ValueError, match="requires gradients"):
            call()
        with torch.no_grad():
            call()
