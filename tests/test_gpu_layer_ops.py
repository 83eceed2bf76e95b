"""The operators of a graph layer beside the sparse product (layer_ops) against their formulas in 64 bits.

Tolerances come from the arithmetic: u(T) is half the distance from 1 to the next value of a type; a sum of n terms in
32 bits is off by at most n 2^-24 of the sum of its terms' magnitudes, whatever its order."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, BF16, F16, E4M3, I8 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}         # the smallest steps of the types
E = 2.0 ** -24
TOP = {E4M3: 448.0, I8: 127.0}


@pytest.fixture(scope="module")
def lo():
    from liteform_ae_amd import layer_ops
    return layer_ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, g, scale=1.0, pad=0, offset=0):
    """Normal values; `pad` more columns in the buffer behind a row, and `offset` before its first one."""
    t = torch.randn((shape[0], offset + shape[1] + pad), device="cuda", generator=g).mul_(scale).to(dtype)
    return t[:, offset:offset + shape[1]]


def within(got, want, bound, what=""):
    assert got.shape == want.shape
    got = got.double()
    assert bool(torch.isfinite(got).all()), what
    excess = ((got - want).abs() - bound).max().item() if got.numel() else 0.0
    assert excess <= 0, f"{what}: {excess} over its bound"


# --------------------------------------------------------------------------- norm

DIMS = [1, 2, 3, 7, 8, 9, 31, 63, 64, 65, 100, 128, 129, 255, 256, 257, 500, 512, 513, 1001, 1024, 1030, 2048, 2049, 4096, 4097, 8191, 8192, 8200, 16384, 16385, 32761,
        40_000, 70_003]


def norm_reference(x, w, res, eps):
    h = x.double() if res is None else x.double() + res.double()
    s = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    return h, s, h * s * (1.0 if w is None else w.double())


@pytest.mark.parametrize("x_type,res_type,out", [(F32, None, F32), (F32, F32, F32), (BF16, BF16, BF16), (F32, BF16, BF16), (F16, F32, F16), (BF16, F16, F32), (F16, None, BF16)])
def test_norm(lo, x_type, res_type, out):
    g = gen(1)
    for i, dim in enumerate(DIMS):
        rows, pad = 1 + i % 5, (0, 3, 8)[i % 3]
        x = normal((rows, dim), x_type, g, 2.0, pad, i % 2)
        res = None if res_type is None else normal((rows, dim), res_type, g, 3.0, pad)
        w = None if i % 7 == 6 else normal((1, dim), (F32, BF16, F16)[i % 3], g)[0].contiguous()
        h64, _, y64 = norm_reference(x, w, res, 1e-6)
        r = lo.rms_norm(x, w, residual=res, eps=1e-6, out_dtype=out)
        y, h = (r, None) if res is None else r
        assert y.dtype is out and y.is_contiguous()
        # a sum of squares of up to 72 in a thread and of 16 wavefronts' (rounded both ways; half of it in the root), a few more roundings
        within(y, y64, y64.abs() * (U[out] + 64 * E) + TINY[out], f"y, {dim}")
        if h is not None:
            assert h.dtype is res_type
            within(h, h64, h64.abs() * (U[res_type] + E) + TINY[res_type], f"h, {dim}")


def test_norm_of_many_rows(lo):
    """More rows than the workgroups take at once, in rows of every number of threads."""
    g = gen(2)
    for rows, dim in [(70_001, 24), (40_000, 96), (20_003, 200), (9_001, 513), (3_000, 3000), (1_100, 12_000)]:
        x, res, w = normal((rows, dim), BF16, g), normal((rows, dim), BF16, g), normal((1, dim), BF16, g)[0]
        h64, _, y64 = norm_reference(x, w, res, 1e-5)
        y, h = lo.rms_norm(x, w, residual=res, eps=1e-5)
        within(y, y64, y64.abs() * (U[BF16] + 64 * E) + TINY[BF16])
        within(h, h64, h64.abs() * (U[BF16] + E))


def test_norm_of_no_rows(lo):
    x = torch.empty((0, 64), device="cuda")
    y, h = lo.rms_norm(x, residual=x)
    assert y.shape == h.shape == (0, 64)
    q, s = lo.rms_norm_8bit(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    dx, dw = lo.rms_norm_grad(x, x, torch.ones(64, device="cuda"))
    assert dx.shape == (0, 64) and bool((dw == 0).all())


def eight_within(q, scale, y64, dtype):
    want = y64.abs().amax(dim=1) / TOP[dtype]
    within(scale, want, want * 80 * E + TINY[F32], "scale")
    # half a step: of int8 half the scale, of e4m3 2^-4 of the value or 2^-10 of the scale
    s = want[:, None]
    half = s * 0.5 if dtype is I8 else torch.maximum(y64.abs() * 2.0 ** -4, s * 2.0 ** -10)
    within(q.double() * scale.double()[:, None], y64, half * (1 + 1e-4) + TINY[F32], "q")


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("x_type,res_type", [(F32, None), (BF16, BF16), (F16, F32)])
def test_norm_8bit(lo, x_type, res_type, dtype):
    g = gen(3)
    for i, dim in enumerate(DIMS):
        rows = 1 + i % 4
        x = normal((rows, dim), x_type, g, 2.0, i % 3)
        res = None if res_type is None else normal((rows, dim), res_type, g, 3.0)
        w = normal((1, dim), x_type, g)[0]
        h64, _, y64 = norm_reference(x, w, res, 1e-6)
        q, scale, *h = lo.rms_norm_8bit(x, w, residual=res, eps=1e-6, dtype=dtype)
        assert q.dtype is dtype and scale.dtype is F32
        eight_within(q, scale, y64, dtype)
        if h:
            within(h[0], h64, h64.abs() * (U[res_type] + E))


@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_quantize_rows(lo, dtype):
    g = gen(4)
    for x_type in (F32, BF16, F16):
        for rows, dim, pad in [(1, 1, 0), (3, 5, 2), (130, 100, 4), (7, 4096, 0), (2, 32768, 0), (3, 100_001, 3), (4000, 72, 0)]:
            x = normal((rows, dim), x_type, g, 5.0, pad)
            q, scale = lo.quantize_rows(x, dtype)
            eight_within(q, scale, x.double(), dtype)
            top = q.double().abs().amax(dim=1)
            assert bool((top == TOP[dtype]).all())                       # the largest element takes the largest value


@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_8bit_rows_at_the_ends(lo, dtype):
    """Zeros, rows so small that 448 / max overflows, rows whose squares overflow, Inf and NaN - none of which touches the rows beside it."""
    g = gen(5)
    x = normal((8, 300), F32, g)
    x[1] = 0
    x[2] *= 1e-42
    x[3] *= 1e25
    x[4, 7] = math.inf
    x[5, 299] = math.nan
    x[6] *= 1e-20
    q, s = lo.quantize_rows(x, dtype)
    ok = [0, 2, 3, 6, 7]
    want = x.double().abs().amax(dim=1) / TOP[dtype]
    for r in ok:
        assert abs(s[r].item() - want[r].item()) <= want[r].item() * 4 * E + TINY[F32]
    for r in (0, 3, 6, 7):
        eight_within(q[r:r + 1], s[r:r + 1], x[r:r + 1].double(), dtype)
    assert s[1].item() == 0 and bool((q[1].float() == 0).all())
    assert bool(torch.isnan(s[4:6]).all())
    q, s = lo.rms_norm_8bit(x, dtype=dtype)
    assert s[1].item() == 0 and bool((q[1].float() == 0).all()) and bool(torch.isnan(s[4:6]).all())
    y64 = norm_reference(x, None, None, 1e-6)[2]
    for r in (0, 6, 7):
        eight_within(q[r:r + 1], s[r:r + 1], y64[r:r + 1], dtype)


def test_norm_keeps_inf_and_nan_in_their_rows(lo):
    x = torch.randn((5, 1001), device="cuda", generator=gen(6)).to(F16)
    x[1, 1000] = math.inf
    x[3, 0] = math.nan
    y = lo.rms_norm(x)
    y64 = norm_reference(x, None, None, 1e-6)[2]
    for r in (0, 2, 4):
        within(y[r], y64[r], y64[r].abs() * (U[F16] + 64 * E) + TINY[F16])
    assert bool(torch.isnan(y[3]).all())
    assert bool(torch.isnan(y[1, 1000])) and bool((y[1, :1000] == 0).all())       # 0 = finite / inf
    zero = lo.rms_norm(torch.zeros((2, 64), device="cuda"))
    assert bool((zero == 0).all())


def grad_reference(dy, h, w, eps, dh):
    d, h = dy.double(), h.double()
    g = d if w is None else d * w.double()
    s = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    k = (g * h).mean(dim=1, keepdim=True) * s * s
    dx = s * (g - h * k) + (0.0 if dh is None else dh.double())
    size = s * (g.abs() + h.abs() * (g * h).abs().mean(dim=1, keepdim=True) * s * s) + (0.0 if dh is None else dh.double().abs())
    return dx, size, (d * h * s).sum(dim=0), (d * h * s).abs().sum(dim=0)


@pytest.mark.parametrize("dy_type,h_type", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16)])
def test_norm_grad(lo, dy_type, h_type):
    g = gen(7)
    for i, dim in enumerate(DIMS):
        rows, pad = (1, 3, 300, 17)[i % 4], (0, 5, 8)[i % 3]
        h = normal((rows, dim), h_type, g, 2.0, pad)
        dy = normal((rows, dim), dy_type, g, 1.0, 0, i % 2)
        w = None if i % 6 == 5 else normal((1, dim), (F32, h_type)[i % 2], g)[0]
        dh = None if i % 3 == 1 else normal((rows, dim), h_type, g, 1.0, pad)
        dx, dw = lo.rms_norm_grad(dy, h, w, eps=1e-6, dh=dh)
        dx64, size, dw64, dw_size = grad_reference(dy, h, w, 1e-6, dh)
        assert dx.dtype is h_type
        within(dx, dx64, dx64.abs() * U[h_type] + size * 128 * E + TINY[h_type], f"dx, {dim}")
        if w is None:
            assert dw is None
        else:
            within(dw, dw64, dw64.abs() * U[w.dtype] + dw_size * (rows + 70) * E + TINY[w.dtype], f"dw, {dim}")


def test_norm_grad_of_many_rows(lo):
    g = gen(8)
    for rows, dim in [(100_003, 40), (50_000, 128), (9_001, 1001), (2_500, 4000)]:
        h, dy, w = normal((rows, dim), BF16, g), normal((rows, dim), BF16, g), normal((1, dim), F32, g)[0]
        dx, dw = lo.rms_norm_grad(dy, h, w)
        dx64, size, dw64, dw_size = grad_reference(dy, h, w, 1e-6, None)
        within(dx, dx64, dx64.abs() * U[BF16] + size * 128 * E + TINY[BF16])
        within(dw, dw64, dw64.abs() * U[F32] + dw_size * 400 * E)         # chains of at most 300 rows, then a tree
        again = lo.rms_norm_grad(dy, h, w)
        assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def test_norm_grad_against_differences(lo):
    g = gen(9)
    rows, dim, step = 6, 200, 1e-5
    x, res, w, c, ch = (normal(s, F32, g).double() for s in ((rows, dim), (rows, dim), (1, dim), (rows, dim), (rows, dim)))
    w = w[0]

    def loss(x, r, w):                                      # c . y + ch . h
        h, _, y = norm_reference(x, w, r, 1e-6)
        return ((c * y).sum() + (ch * h).sum()).item()

    _, h = lo.rms_norm(x.float(), w.float(), residual=res.float())
    dx, dw = lo.rms_norm_grad(c.float(), h, w.float(), dh=ch.float())
    for k in range(5):
        vx, vw = normal((rows, dim), F32, g).double(), normal((1, dim), F32, g).double()[0]
        along_x = (loss(x + step * vx, res, w) - loss(x - step * vx, res, w)) / (2 * step)
        along_r = (loss(x, res + step * vx, w) - loss(x, res - step * vx, w)) / (2 * step)
        along_w = (loss(x, res, w + step * vw) - loss(x, res, w - step * vw)) / (2 * step)
        got_x, got_w = (dx.double() * vx).sum().item(), (dw.double() * vw).sum().item()
        # differences: third derivatives times step^2 and the sums' 2^-53 over step, about 1e-7 of the terms; floats 1e-5 of them
        for got, want, size in ((got_x, along_x, (dx.double() * vx).abs().sum()), (got_x, along_r, (dx.double() * vx).abs().sum()),
                                (got_w, along_w, (dw.double() * vw).abs().sum())):
            assert abs(got - want) <= 1e-5 * size.item()


# --------------------------------------------------------------------------- product

#        rows, n, k: one row to many tiles, sizes that fit no tile, k of less than a step and of nothing
SHAPES = [(1, 1, 1), (1, 64, 256), (1, 1000, 4096), (2, 17, 33), (7, 100, 129), (13, 1001, 1000), (16, 48, 4000), (17, 16, 64), (33, 130, 70), (64, 64, 64), (65, 257, 31),
          (100, 47, 100), (128, 128, 128), (200, 33, 2050), (257, 255, 513), (300, 300, 8), (1000, 515, 1001), (2049, 70, 40), (3, 5, 0), (40, 9, 0)]
BIG = [(4100, 4000, 520), (5000, 2600, 1031)]                             # enough tiles for the largest ones
ACTS = [None, "relu", "gelu", "silu"]


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid(z) if act == "silu" else z


def act_grad64(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def check_linear(lo, shape, x_type, act, bias, res, out, g, pad=0, offset=0):
    m, n, k = shape
    x = normal((m, k), x_type, g, 1.0, pad, offset)
    w = normal((n, k), x_type, g, max(k, 1) ** -0.5, pad, offset)
    b = None if bias is None else normal((1, n), bias, g)[0]
    r = None if res is None else normal((m, n), res, g, 1.0, pad)
    y, z = lo.linear(x, w, b, activation=act, residual=r, out_dtype=out, return_preactivation=True)
    x64, w64 = x.double(), w.double()
    z64 = x64 @ w64.t() + (0.0 if b is None else b.double())
    # sums in 32 bits of products that are exact (16 bits) or off by 2^-22 (float32: what is left of the cut), the bias among them
    z_off = (x64.abs() @ w64.abs().t() + (0.0 if b is None else b.double().abs())) * (k + 24) * E
    within(z, z64, z64.abs() * U[x_type] + z_off + TINY[x_type], f"z {shape}")
    y64 = act64(z64, act)
    a_off = 0.0 if act is None else 1.13 * z_off + (z64.abs() + 1) * 16 * E     # |act'| <= 1.13, exp and erf to a few units
    a_off = z_off if act is None else a_off
    if r is not None:
        y64 = y64 + r.double()
    within(y, y64, y64.abs() * (U[out] + E) + a_off + E * (act64(z64, act).abs()) + TINY[out], f"y {shape}")
    assert torch.equal(y, lo.linear(x, w, b, activation=act, residual=r, out_dtype=out))


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_linear(lo, x_type):
    g = gen(11)
    for i, shape in enumerate(SHAPES):
        check_linear(lo, shape, x_type, ACTS[i % 4], (None, x_type, F32)[i % 3], (None, x_type, F32, BF16)[(i // 2) % 4], (x_type, F32)[i % 5 == 4], g)


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_linear_of_rows_inside_wider_buffers(lo, x_type):
    g = gen(12)
    for i, shape in enumerate(SHAPES[:-2]):
        check_linear(lo, shape, x_type, ACTS[(i + 1) % 4], x_type, x_type, x_type, g, pad=(1, 8, 3)[i % 3], offset=(0, 1, 8, 5)[i % 4])


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_linear_of_many_tiles(lo, x_type):
    g = gen(13)
    for i, shape in enumerate(BIG):
        check_linear(lo, shape, x_type, ACTS[i + 2], x_type, x_type, x_type, g)
        check_linear(lo, shape, x_type, "relu", None, None, x_type, g, pad=3, offset=1)


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_linear_of_long_sums(lo, x_type):
    """Few outputs, many products: k is cut up."""
    g = gen(14)
    for shape in [(40, 30, 40_000), (130, 100, 20_007), (16, 16, 100_003), (300, 20, 9_000)]:
        check_linear(lo, shape, x_type, "gelu", x_type, x_type, x_type, g)


@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_linear_8bit(lo, dtype):
    g = gen(15)
    for i, (m, n, k) in enumerate(SHAPES + BIG + [(40, 30, 40_000), (130, 100, 20_007)]):
        pad, out = (0, 3, 16)[i % 3], (BF16, F32, F16)[i % 3]
        x, sx = lo.quantize_rows(normal((m, max(k, 1)), F32, g), dtype)
        w, sw = lo.quantize_rows(normal((n, max(k, 1)), F32, g, max(k, 1) ** -0.5), dtype)
        wide = torch.zeros((m, k + pad), device="cuda", dtype=dtype)
        wide[:, :k] = x[:, :k]
        x, w = wide[:, :k], w[:, :k]
        b = None if i % 2 else normal((1, n), F32, g)[0]
        r = normal((m, n), out, g) if i % 3 else None
        act = ACTS[i % 4]
        y = lo.linear_8bit(x, sx, w, sw, b, activation=act, residual=r, out_dtype=out)
        x64, w64 = x.double() * sx.double()[:, None], w.double() * sw.double()[:, None]
        z64 = x64 @ w64.t() + (0.0 if b is None else b.double())
        # int8 sums are exact.  The instruction for e4m3 adds its products in groups of eight and cuts each below 2^-13 of the group's
        # largest one: seven of them lose at most 7 * 2^-13 of it
        off = (x64.abs() @ w64.abs().t()) * (8 * E if dtype is I8 else 2.0 ** -10 + (k + 16) * E) + (0.0 if b is None else b.double().abs()) * 4 * E
        y64 = act64(z64, act)
        off = off if act is None else 1.13 * off + (z64.abs() + 1) * 16 * E
        off = off + y64.abs() * 4 * E
        if r is not None:
            y64 = y64 + r.double()
        within(y, y64, y64.abs() * (U[out] + E) + off + TINY[out], f"{(m, n, k)}")


def test_int8_sums_are_exact(lo):
    """Of the longest rows that are taken, whose sums pass 2^24."""
    k = (1 << 17) - 1
    for m, n in [(1, 20), (20, 20)]:
        x = torch.full((m, k), -128, device="cuda", dtype=I8)
        w = torch.full((n, k), -128, device="cuda", dtype=I8)
        w[1::2] = 127
        w[1::2, -1] = 126
        y = lo.linear_8bit(x, torch.ones(m, device="cuda"), w, torch.ones(n, device="cuda"), out_dtype=F32)
        want = (x.double() @ w.double().t()).float()
        assert torch.equal(y, want)


def test_float32_products_keep_inf_nan_and_large_values(lo):
    g = gen(16)
    for m, n, k in [(3, 20, 70), (40, 50, 100), (200, 300, 260), (40, 30, 9000)]:
        x, w = normal((m, k), F32, g), normal((n, k), F32, g)
        x[0, 3] = math.inf
        x[1, 5], w[4, 5] = 3.0e38, 2.0 ** -10                          # just below the largest, times exact powers of two
        x[1, :5] = 0
        x[1, 6:] = 0
        x[2, 7] = math.nan
        w[:, 3] = torch.where(w[:, 3].abs() < 0.1, torch.ones_like(w[:, 3]), w[:, 3])
        w[5, 3] = 0.0
        y = lo.linear(x, w)
        assert bool(torch.isnan(y[2]).all())
        sign = torch.sign(w[:, 3])
        keep = sign != 0
        assert bool((y[0][keep] == sign[keep] * math.inf).all()) and bool(torch.isnan(y[0, 5]))
        assert y[1, 4].item() == pytest.approx(3.0e38 * 2.0 ** -10, rel=1e-6)
        z64 = x[3:].double() @ w.double().t()
        within(y[3:], z64, (x[3:].double().abs() @ w.double().abs().t()) * (k + 24) * E)


def test_float32_values_far_apart(lo):
    """A row with one value 1e20 times the others: where its weight is 0 the others must come out whole."""
    g = gen(17)
    for m, n, k in [(5, 40, 200), (64, 70, 300), (140, 200, 300)]:
        x, w = normal((m, k), F32, g), normal((n, k), F32, g)
        x[:, 11] = 1e20
        w[:, 11] = 0
        z64 = x.double() @ w.double().t()
        within(lo.linear(x, w), z64, (x.double().abs() @ w.double().abs().t()) * (k + 24) * E)


@pytest.mark.parametrize("x_type", [BF16, F16])
def test_products_keep_inf_and_nan_in_their_rows(lo, x_type):
    g = gen(18)
    for m, n, k in [(5, 30, 100), (90, 70, 333)]:
        x, w = normal((m, k), x_type, g), normal((n, k), x_type, g)
        x[1, 2], x[2, k - 1] = math.inf, math.nan
        y = lo.linear(x, w)
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isinf(y[1]).all())
        keep = [r for r in range(m) if r not in (1, 2)]
        z64 = x[keep].double() @ w.double().t()
        within(y[keep], z64, z64.abs() * U[x_type] + (x[keep].double().abs() @ w.double().abs().t()) * (k + 24) * E + TINY[x_type])


def check_grad(lo, shape, x_type, act, bias, g, pad=0, offset=0):
    m, n, k = shape
    x, w = normal((m, k), x_type, g, 1.0, pad, offset), normal((n, k), x_type, g, 1.0, pad)
    dy = normal((m, n), x_type, g, 1.0, pad, offset)
    z = None if act is None else normal((m, n), x_type, g, 1.0, offset)
    dx, dw, db = lo.linear_grad(dy, x, w, z=z, activation=act, bias_dtype=bias)
    dz = dy.double() if act is None else dy.double() * act_grad64(z.double(), act)
    # dz as the products take it: rounded to the type behind an activation, whose derivative is known to 16 units
    dz_off = 0.0 if act is None else dz.abs() * U[x_type] + dy.double().abs() * 16 * E + TINY[x_type]
    x64, w64 = x.double(), w.double()
    off = (dz.abs() @ w64.abs()) * (n + 24) * E + (0.0 if act is None else dz_off @ w64.abs()) * 1.001
    want = dz @ w64
    within(dx, want, want.abs() * U[x_type] + off + TINY[x_type], f"dx {shape}")
    off = (dz.abs().t() @ x64.abs()) * (m + 24) * E + (0.0 if act is None else dz_off.t() @ x64.abs()) * 1.001
    want = dz.t() @ x64
    within(dw, want, want.abs() * U[x_type] + off + TINY[x_type], f"dw {shape}")
    if bias is None:
        assert db is None
    else:
        want = dz.sum(dim=0)
        within(db, want, want.abs() * U[bias] + (dz.abs() + dy.double().abs()).sum(dim=0) * (m + 40) * E + TINY[bias], f"db {shape}")
    again = lo.linear_grad(dy, x, w, z=z, activation=act, bias_dtype=bias)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_linear_grad(lo, x_type):
    g = gen(21)
    for i, shape in enumerate(SHAPES[:-2] + [(20_000, 47, 100), (9_001, 128, 70), (70_000, 16, 16)]):
        check_grad(lo, shape, x_type, ACTS[i % 4], (x_type, F32, None)[i % 3], g, pad=(0, 3, 8)[i % 3], offset=(0, 1, 0, 4)[i % 4])


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_linear_grad_of_many_tiles(lo, x_type):
    g = gen(22)
    check_grad(lo, (4100, 3900, 4000), x_type, "gelu", x_type, g)
    check_grad(lo, (4100, 3901, 4005), x_type, None, F32, g, pad=1)


@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_linear_grad_at_the_ends_of_matrices(lo, x_type):
    """Matrices of a few elements and lengths around a step, in buffers that hold NaN behind every row and behind the last one."""
    g = gen(25)

    def among_nan(rows, cols, pad):
        flat = torch.full((rows * (cols + pad) + 64,), float("nan"), device="cuda", dtype=x_type)
        t = flat[:rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        return t.copy_(normal((rows, cols), x_type, g))

    for m in (1, 2, 9, 17, 31, 32, 33, 36, 40, 41, 63, 64, 65, 70, 72, 73, 137):
        for n in (1, 3, 8, 17):
            for k in (1, 2, 7, 8, 65):
                for pad in (0, 3):
                    dy, x, w = among_nan(m, n, pad), among_nan(m, k, pad), among_nan(n, k, pad)
                    dx, dw, _ = lo.linear_grad(dy, x, w)
                    want = dy.double() @ w.double()
                    within(dx, want, want.abs() * U[x_type] + (dy.double().abs() @ w.double().abs()) * (n + 24) * E + TINY[x_type], f"dx {(m, n, k, pad)}")
                    want = dy.double().t() @ x.double()
                    within(dw, want, want.abs() * U[x_type] + (dy.double().abs().t() @ x.double().abs()) * (m + 24) * E + TINY[x_type], f"dw {(m, n, k, pad)}")


def test_linear_grad_of_what_is_wanted(lo):
    g = gen(23)
    x, w, dy = normal((300, 64), BF16, g), normal((128, 64), BF16, g), normal((300, 128), BF16, g)
    dx, dw, db = lo.linear_grad(dy, x, w, bias_dtype=F32)
    only = lo.linear_grad(dy, x, w, want_dx=False)
    assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
    only = lo.linear_grad(dy, x, w, want_dweight=False, bias_dtype=F32)
    assert only[1] is None and torch.equal(only[0], dx) and torch.equal(only[2], db)
    none = lo.linear_grad(dy[:0], x[:0], w, bias_dtype=F32)
    assert none[0].shape == (0, 64) and bool((none[1] == 0).all()) and bool((none[2] == 0).all())


@pytest.mark.parametrize("act", ACTS)
def test_linear_grad_against_differences(lo, act):
    g = gen(24)
    m, n, k, step = 9, 33, 20, 1e-5
    x, w, c = (normal(s, F32, g).double() for s in ((m, k), (n, k), (m, n)))
    b = normal((1, n), F32, g).double()[0]

    def loss(x, w, b):
        return (c * act64(x @ w.t() + b, act)).sum().item()

    _, z = lo.linear(x.float(), w.float(), b.float(), activation=act, return_preactivation=True)
    dx, dw, db = lo.linear_grad(c.float(), x.float(), w.float(), z=z, activation=act, bias_dtype=F32)
    for _ in range(4):
        vx, vw, vb = normal((m, k), F32, g).double(), normal((n, k), F32, g).double(), normal((1, n), F32, g).double()[0]
        for d, v, at in ((dx, vx, 0), (dw, vw, 1), (db, vb, 2)):
            move = [torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)]
            move[at] = step * v
            along = (loss(x + move[0], w + move[1], b + move[2]) - loss(x - move[0], w - move[1], b - move[2])) / (2 * step)
            # relu's kinks: an element within a step of one (|z| < 1e-4, none or a few of 297) may move by its whole term
            size = (d.double() * v).abs().sum().item()
            kink = 0.0
            if act == "relu":
                near = (z.double().abs() < 2e-4).double()
                kink = (near * c.abs()).sum().item() * 20
            assert abs((d.double() * v).sum().item() - along) <= 2e-5 * size + kink


# --------------------------------------------------------------------------- how they are called


def test_rows_past_32_bits(lo):
    """Element offsets of more than 2^32: the last rows of matrices of 9 GB."""
    g = gen(31)
    rows, dim = 70_000_000, 64
    x = torch.empty((rows, dim), device="cuda", dtype=BF16)
    x[:1000] = normal((1000, dim), BF16, g)
    x[1000:-1000] = 1.0
    x[-1000:] = normal((1000, dim), BF16, g)
    w = normal((32, dim), BF16, g)
    y = lo.linear(x, w)
    for part in (slice(0, 1000), slice(rows - 1000, rows)):
        z64 = x[part].double() @ w.double().t()
        within(y[part], z64, z64.abs() * U[BF16] + (x[part].double().abs() @ w.double().abs().t()) * 90 * E + TINY[BF16])
    del y
    y = lo.rms_norm(x)
    for part in (slice(0, 1000), slice(rows - 1000, rows)):
        y64 = norm_reference(x[part], None, None, 1e-6)[2]
        within(y[part], y64, y64.abs() * (U[BF16] + 64 * E) + TINY[BF16])


def test_on_a_stream_of_its_own_and_in_a_graph(lo):
    g = gen(32)
    x, w, b, res = normal((130, 256), BF16, g), normal((96, 256), BF16, g), normal((1, 96), BF16, g)[0], normal((130, 256), BF16, g)
    weight = normal((1, 256), BF16, g)[0]

    def layer():
        y, h = lo.rms_norm(x, weight, residual=res)
        out, z = lo.linear(y, w, b, activation="gelu", return_preactivation=True)
        grads = lo.linear_grad(out, y, w, z=z, activation="gelu", bias_dtype=F32)
        dx, dw = lo.rms_norm_grad(grads[0], h, weight)
        q, s, _ = lo.rms_norm_8bit(x, weight, residual=res)
        qw, sw = lo.quantize_rows(w)
        return [y, h, out, z, *grads, dx, dw, s, lo.linear_8bit(q, s, qw, sw)]

    want = [t.clone() for t in layer()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = layer()
    for k in range(3):
        x.copy_(normal((130, 256), BF16, g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        again = layer()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, again)), k


def test_refusals(lo):
    g = gen(33)
    x, w = normal((8, 64), BF16, g), normal((32, 64), BF16, g)
    for call in (
        lambda: lo.rms_norm(x.cpu()),
        lambda: lo.rms_norm(x.double()),
        lambda: lo.rms_norm(x[0]),
        lambda: lo.rms_norm(x.t()),                                      # columns, not rows
        lambda: lo.rms_norm(x[:1].expand(8, 64)),                        # rows on top of each other
        lambda: lo.rms_norm(x, torch.ones(63, device="cuda")),
        lambda: lo.rms_norm(x, residual=x[:7]),
        lambda: lo.rms_norm(x, eps=-1.0),
        lambda: lo.rms_norm(x, out_dtype=torch.int8),
        lambda: lo.rms_norm_8bit(x, dtype=torch.uint8),
        lambda: lo.quantize_rows(x, torch.bfloat16),
        lambda: lo.rms_norm_grad(x, x[:, :32]),
        lambda: lo.rms_norm_grad(x, x, dh=x.float()),
        lambda: lo.linear(x, w.float()),
        lambda: lo.linear(x, w[:, :32]),
        lambda: lo.linear(x, w.t()),
        lambda: lo.linear(x, w, activation="tanh"),
        lambda: lo.linear(x, w, bias=x[0]),
        lambda: lo.linear(x, w, residual=x),
        lambda: lo.linear(x, w, out_dtype=torch.float64),
        lambda: lo.linear_8bit(x, None, w, None),
        lambda: lo.linear_8bit(*lo.quantize_rows(x), *lo.quantize_rows(w, torch.int8)),
        lambda: lo.linear_8bit(lo.quantize_rows(x)[0], torch.ones(7, device="cuda"), *lo.quantize_rows(w)),
        lambda: lo.linear_grad(x, x, w),
        lambda: lo.linear_grad(x[:, :32], x, w, activation="relu"),      # no z
        lambda: lo.linear_grad(x[:, :32].float(), x, w),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError, match="at most 16777216"):
        lo.rms_norm(torch.ones((1, (1 << 24) + 1), device="cuda"))
    long = torch.ones((1, 1 << 17), device="cuda", dtype=I8)
    one = torch.ones(1, device="cuda")
    with pytest.raises(NotImplementedError, match="32 bits"):
        lo.linear_8bit(long, one, long, one)


def test_refusals_of_the_library(lo):
    """Through the C entry points: null pointers, small workspaces, missing scales - an answer, no launch."""
    import ctypes as C
    from liteform_ae_amd import _lib
    lib = _lib.load()
    x = torch.ones((40, 20_000), device="cuda")
    a = _lib.LinearArgs()
    a.x = a.w = x.data_ptr()
    a.ld_x = a.ld_w = 20_000
    a.m = a.n = 40
    a.k = 20_000
    y = torch.empty((40, 40), device="cuda")
    a.y, a.ld_y = y.data_ptr(), 40
    need = lib.lf_linear_work_bytes(40, 40, 20_000, _lib.LF_DTYPE_F32)
    assert need > 0
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert lib.lf_linear(C.addressof(a), None, 0, None) == _lib.LF_ERR_INVALID
    assert lib.lf_linear(C.addressof(a), work.data_ptr(), need - 1, None) == _lib.LF_ERR_WORKSPACE
    assert lib.lf_linear(None, None, 0, None) == _lib.LF_ERR_INVALID
    a.ld_x = 19_999
    assert lib.lf_linear(C.addressof(a), work.data_ptr(), need, None) == _lib.LF_ERR_INVALID
    a.ld_x, a.dtype = 20_000, _lib.LF_DTYPE_I8
    assert lib.lf_linear(C.addressof(a), work.data_ptr(), need, None) == _lib.LF_ERR_INVALID and "scales" in _lib.last_error()
    a.dtype = 9
    assert lib.lf_linear(C.addressof(a), work.data_ptr(), need, None) == _lib.LF_ERR_UNSUPPORTED
    assert lib.lf_rms_norm(None, 64, 0, None, 0, 0, None, 0, 1, 64, 1e-6, y.data_ptr(), 64, 0, None, None, 0, None) == _lib.LF_ERR_INVALID
    assert lib.lf_rms_norm(x.data_ptr(), 64, 0, None, 0, 0, None, 0, 1, 64, 1e-6, y.data_ptr(), 64, _lib.LF_DTYPE_I8, None, None, 0, None) == _lib.LF_ERR_INVALID
    assert lib.lf_rms_norm(x.data_ptr(), 64, 0, None, 0, 0, None, 0, -1, 64, 1e-6, y.data_ptr(), 64, 0, None, None, 0, None) == _lib.LF_ERR_INVALID
    need = lib.lf_rms_norm_grad_work_bytes(40, 64)
    assert lib.lf_rms_norm_grad(x.data_ptr(), 64, 0, x.data_ptr(), 64, 0, x.data_ptr(), 0, None, 0, 40, 64, 1e-6, y.data_ptr(), 64, y.data_ptr(), work.data_ptr(),
                                need - 4, None) == _lib.LF_ERR_WORKSPACE
    torch.cuda.synchronize()


# --------------------------------------------------------------------------- activations over their range


def phi64(z):
    """Phi(z); torch.special.ndtr is 1 + erf below -1, with none of the digits of what it leaves."""
    return 0.5 * torch.special.erfc(-z * math.sqrt(0.5))


def gelu64(z, act):
    return z * phi64(z) if act == "gelu" else act64(z, act)


def act_off(z, act, fine):
    """How far act(z) may be off in 32 bits, roundings counted in E = 2^-24 (a device function's last place: 2).  gelu: the tail 1 - Phi(|z|) is
    a quotient of polynomials of positive terms (4 and 5 products with sums, each coefficient rounded, a reciprocal, a product) and exp(-z^2 / 2),
    with the rounding of z^2 made up for: 20 in all.  For 16 bits: fitted to 4e-7, and two roundings of exp's argument, z^2 / 2."""
    z = z.abs()
    if act == "gelu":
        tail = phi64(-z)
        return z * tail * (20 * E if fine else 4.1e-7 + (20 + z * z) * E)
    # exp, 1 + exp, product, quotient; without fine its argument z is rounded twice
    return act64(-z, "silu").abs() * (8 if fine else 10 + 2 * z) * E if act == "silu" else 0.0 * z


def act_grad_off(z, act, fine):
    a = z.abs()
    if act == "gelu":                                       # a phi(a), with exp as above and three roundings, and the tail
        phi = a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
        rest = 0.0 if fine else 4.1e-7 + a * a * E
        return phi * (10 * E + rest) + phi64(-a) * (20 * E + rest)
    if act == "silu":                                       # s (1 + z (1 - s)): s and 1 - s to seven roundings, without fine as a difference
        s, t = torch.sigmoid(z), torch.sigmoid(-z)
        return s * (a * t + (1 + z * t).abs()) * 9 * E if fine else s * (a * t + 1 + a) * (12 + 2 * a) * E
    return 0.0 * a


@pytest.mark.parametrize("act", ["gelu", "silu", "relu"])
@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_activations_and_their_gradients_keep_their_digits(lo, x_type, act):
    """z = x from -10 to 10, as sums of one product: of few rows, of tiles with and without whole pieces of columns, of parts of k."""
    every = torch.linspace(-10, 10, 40_001, device="cuda").to(x_type)
    for rows, n, k in [(40_001, 1, 1), (40_001, 8, 8), (9, 3, 5), (70, 16, 40_000)]:
        z = every[:: 40_001 // rows][:rows]
        x, w = torch.zeros((rows, k), device="cuda", dtype=x_type), torch.ones((n, k), device="cuda", dtype=x_type)
        x[:, 0] = z
        z64 = z.double()[:, None].expand(rows, n)
        for out in (x_type, F32):
            y = lo.linear(x, w, activation=act, out_dtype=out)
            y64 = gelu64(z64, act)
            within(y, y64, y64.abs() * U[out] + act_off(z64, act, out is F32) + TINY[out], f"{act} {rows, n, k} {out}")
    one = torch.ones((1, 1), device="cuda", dtype=x_type)
    z = every[:, None].contiguous()
    dx, _, db = lo.linear_grad(torch.ones_like(z), z, one, z=z, activation=act, bias_dtype=F32)
    d = z.double()
    want = phi64(d) + d * torch.exp(-d * d / 2) / math.sqrt(2 * math.pi) if act == "gelu" else act_grad64(d, act)
    within(dx, want, want.abs() * U[x_type] + act_grad_off(d, act, x_type is F32) + TINY[x_type], act)


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_activations_of_large_products_keep_their_digits(lo, act):
    """Through the large tiles, 16 and 8 bits in, 32 and 16 bits out."""
    m, n = 7001, 4104
    for x_type, k in [(BF16, 1024), (I8, 2048)]:
        x, w = torch.zeros((m, k), device="cuda", dtype=x_type), torch.zeros((n, k), device="cuda", dtype=x_type)
        w[:, 1] = 1
        if x_type is BF16:
            x[:, 1] = torch.linspace(-9, 9, m, device="cuda")
            z64 = x[:, 1:2].double()
        else:
            x[:, 1] = torch.arange(m, device="cuda") % 256 - 128
            z64 = x[:, 1:2].double() / 16
        scales = [torch.full((m,), 0.25, device="cuda"), torch.full((n,), 0.25, device="cuda")]
        y64 = gelu64(z64, act)
        for out in (F32, BF16, F16):
            y = lo.linear(x, w, activation=act, out_dtype=out) if x_type is BF16 else lo.linear_8bit(x, scales[0], w, scales[1], activation=act, out_dtype=out)
            assert bool((y == y[:, :1]).all())
            within(y[:, :1], y64, y64.abs() * U[out] + act_off(z64, act, out is F32) + TINY[out], f"{act} {x_type} {out}")


# --------------------------------------------------------------------------- rows at the ends of the range


@pytest.mark.parametrize("dim", [5, 300, 3000, 20_001])
@pytest.mark.parametrize("x_type", [F32, BF16])
def test_norm_of_rows_whose_squares_leave_the_range(lo, x_type, dim):
    """Squares of 1e20 and more overflow 32 bits, those of 1e-25 vanish (eps = 0): y, the stream, the 8-bit form and the gradients are as of any row,
    and the rows beside them as ever."""
    g = gen(51)
    for eps, factors in ((1e-6, (1.0, 1e20, 1e25, 3e36, 1.0)), (0.0, (1.0, 1e-17, 1e-25, 1e-37, 1e30, 1.0))):
        rows = len(factors)
        x = normal((rows, dim), F32, g)
        x = (x / x.abs().amax(dim=1, keepdim=True) * torch.tensor(factors, device="cuda")[:, None]).to(x_type)
        res = (normal((rows, dim), F32, g).clamp(-3, 3) * torch.tensor(factors, device="cuda")[:, None] * 0.25).to(x_type)
        w, dy = normal((1, dim), x_type, g)[0], normal((rows, dim), x_type, g)
        for r in (None, res):
            h64, _, y64 = norm_reference(x, w, r, eps)
            y = lo.rms_norm(x, w, residual=r, eps=eps, out_dtype=F32)
            if r is not None:
                y, h = y
                within(h, h64, h64.abs() * (U[x_type] + E) + TINY[x_type], "h")
            # (x + r is rounded to 32 bits first: a unit, and one of the smallest step where that is all it has)
            within(y, y64, y64.abs() * (U[F32] + 64 * E) + (TINY[F32] / h64.abs().amax(dim=1, keepdim=True)) * y64.abs().amax(dim=1, keepdim=True), "y")
            for dtype in (E4M3, I8):
                q, scale, *_ = lo.rms_norm_8bit(x, w, residual=r, eps=eps, dtype=dtype)
                eight_within(q, scale, y64, dtype)
        dx, dw = lo.rms_norm_grad(dy, x, w, eps=eps)
        dx64, size, dw64, dw_size = grad_reference(dy, x, w, eps, None)
        fits = dx64.abs() < 3.3e38                                       # (of the smallest rows 16 / 2e-38 does not)
        within(dx[fits], dx64[fits], (dx64.abs() * U[x_type] + size * 128 * E + TINY[x_type])[fits], "dx")
        within(dw, dw64, dw64.abs() * U[x_type] + dw_size * (rows + 70) * E, "dw")


@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_8bit_rows_of_zeros_without_eps(lo, dtype):
    for dim in (7, 300, 20_001):
        x = torch.zeros((3, dim), device="cuda")
        x[1] = torch.arange(dim, device="cuda") + 1.0
        q, scale = lo.rms_norm_8bit(x, eps=0.0, dtype=dtype)
        assert scale[0].item() == scale[2].item() == 0 and bool((q[0::2].float() == 0).all())
        eight_within(q[1:2], scale[1:2], norm_reference(x[1:2], None, None, 0.0)[2], dtype)


def test_tensors_that_require_gradients(lo):
    """Refused where torch would build a graph, as its gradients would end here; taken under no_grad, with the results of any others."""
    g = gen(61)
    x, w, b, v, r = normal((20, 64), F32, g), normal((32, 64), F32, g), normal((1, 32), F32, g)[0], normal((1, 64), F32, g)[0], normal((20, 64), F32, g)
    dy, z, y = normal((20, 32), F32, g), normal((20, 32), F32, g), normal((20, 32), F32, g)
    q, s = lo.quantize_rows(x)
    p, t = lo.quantize_rows(w)
    calls = [(lo.rms_norm, [x, v, r]), (lo.rms_norm_8bit, [x, v, r]), (lo.quantize_rows, [x]), (lo.rms_norm_grad, [r, x, v]),
             (lambda a, d: lo.rms_norm_grad(r, a, v, dh=d), [x, r]), (lambda *a: lo.linear(*a[:3], "gelu", a[3]), [x, w, b, y]),
             (lambda a, c, e, f: lo.linear_8bit(q, a, p, c, e, residual=f), [s, t, b, y]), (lambda *a: lo.linear_grad(*a, activation="gelu"), [dy, x, w, z])]
    for call, args in calls:
        want = call(*args)
        for i in range(len(args)):
            with_graph = [a.clone().requires_grad_() if k == i else a for k, a in enumerate(args)]
            with pytest.raises(ValueError, match="no_grad"):
                call(*with_graph)
            with torch.no_grad():
                got = call(*with_graph)
            for a, c in zip(*((r if isinstance(r, tuple) else (r,)) for r in (got, want))):
                assert a is None and c is None or torch.equal(a.float(), c.float())


@pytest.mark.parametrize("x_type", [F32, BF16])
def test_products_of_sizes_of_zero(lo, x_type):
    """No rows, no features out, none in, in every combination: sums of nothing are 0."""
    g = gen(81)
    for m in (0, 1, 40, 700):
        for n in (0, 1, 24, 300):
            for k in (0, 1, 40, 300):
                if m and n and k:
                    continue
                x, w, dy, z = normal((m, k), x_type, g), normal((n, k), x_type, g), normal((m, n), x_type, g), normal((m, n), x_type, g)
                b = normal((1, n), F32, g)[0]
                y = lo.linear(x, w, b, activation="relu", residual=dy)
                y64 = b.double().clamp_min(0) + dy.double()
                within(y, y64, y64.abs() * (U[x_type] + 4 * E), f"y {(m, n, k)}")
                for act in ACTS:
                    dx, dw, db = lo.linear_grad(dy, x, w, z=z, activation=act, bias_dtype=F32)
                    assert dx.shape == (m, k) and dw.shape == (n, k) and db.shape == (n,)
                    assert bool((dx == 0).all()) and bool((dw == 0).all())
                    dz = dy.double() if act is None else dy.double() * act_grad64(z.double(), act)
                    within(db, dz.sum(dim=0), (dz.abs() + dy.double().abs()).sum(dim=0) * (m + 40) * E, f"db {(m, n, k)}")
