"""The dense products of sizes that reach every kernel (which sizes reach which: test_product_paths.py), against 64 bits."""
import pytest

from test_gpu_layer_ops import (ACTS, BF16, E, E4M3, F16, F32, I8, TINY, U, act64, check_grad, check_linear, gen, lo, normal, within)  # noqa: F401 (lo: the fixture)
from test_product_paths import FORWARD_8, FORWARD_16, GRAD_16

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("x_type", [BF16, F16])
def test_forward(lo, x_type):  # noqa: F811
    g = gen(41)
    for i, shape in enumerate(FORWARD_16):
        check_linear(lo, shape, x_type, ACTS[i % 4], (x_type, F32, None)[i % 3], (x_type, F32, None, F16)[i // 2 % 4], (x_type, F32)[i % 5 == 4], g)


@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_forward_8bit(lo, dtype):  # noqa: F811
    g = gen(42)
    for i, (m, n, k) in enumerate(FORWARD_8):
        x, sx = lo.quantize_rows(normal((m, k), F32, g), dtype)
        w, sw = lo.quantize_rows(normal((n, k), F32, g, k ** -0.5), dtype)
        out, act = (BF16, F16, F32)[i % 3], ACTS[i % 4]
        b = None if i % 4 == 2 else normal((1, n), (F32, BF16)[i % 2], g)[0]
        r = None if i % 3 == 2 else normal((m, n), (BF16, F32)[i % 2], g)
        y = lo.linear_8bit(x, sx, w, sw, b, activation=act, residual=r, out_dtype=out)
        x64, w64 = x.double() * sx.double()[:, None], w.double() * sw.double()[:, None]
        z64 = x64 @ w64.t() + (0.0 if b is None else b.double())
        # int8 sums are exact; e4m3 products are added in groups of eight, cut below 2^-13 of the group's largest: 7 * 2^-13 of it at most
        off = (x64.abs() @ w64.abs().t()) * (8 * E if dtype is I8 else 2.0 ** -10 + (k + 16) * E) + (0.0 if b is None else b.double().abs()) * 4 * E
        y64 = act64(z64, act)
        # |act'| <= 1.13, exp and erf to 16 units
        off = (off if act is None else 1.13 * off + (z64.abs() + 1) * 16 * E) + y64.abs() * 4 * E
        if r is not None:
            y64 = y64 + r.double()
        within(y, y64, y64.abs() * (U[out] + E) + off + TINY[out], f"{(m, n, k)}")


@pytest.mark.parametrize("x_type", [BF16, F16])
def test_gradients(lo, x_type):  # noqa: F811
    g = gen(43)
    for i, shape in enumerate(GRAD_16):
        # (behind an activation the products' first operand is dz, in rows of their own)
        check_grad(lo, shape, x_type, ACTS[i % 4] if i % 2 else None, (x_type, F32, None)[i % 3], g)
