"""The graph layer's operators without a GPU: they raise, and the library's kernels are as their speed needs them."""
import pytest
import torch

from test_kernel_resources import kernels  # noqa: F401  (the fixture)


@pytest.mark.skipif(torch.cuda.is_available(), reason="only meaningful where no GPU is visible")
def test_operators_raise_without_gpu():
    from liteform_ae_amd import layer_ops as lo
    x, w = torch.ones(3, 8), torch.ones(4, 8)
    for call in (lambda: lo.rms_norm(x), lambda: lo.rms_norm_8bit(x), lambda: lo.quantize_rows(x), lambda: lo.rms_norm_grad(x, x),
                 lambda: lo.linear(x, w), lambda: lo.linear_8bit(x.to(torch.int8), torch.ones(3), w.to(torch.int8), torch.ones(4)),
                 lambda: lo.linear_grad(torch.ones(3, 4), x, w)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_work_bytes_need_no_gpu():
    from liteform_ae_amd import _lib
    lib = _lib.load()
    assert lib.lf_linear_work_bytes(16, 4096, 4096, _lib.LF_DTYPE_BF16) == 0              # few rows: one kernel
    assert lib.lf_linear_work_bytes(8192, 8192, 8192, _lib.LF_DTYPE_BF16) == 0            # tiles enough: k in one part
    assert lib.lf_linear_work_bytes(64, 64, 1 << 16, _lib.LF_DTYPE_BF16) >= 2 * 64 * 64 * 4
    assert lib.lf_linear_work_bytes(-1, 8, 8, _lib.LF_DTYPE_F32) == 0 and lib.lf_linear_work_bytes(8, 8, 8, 99) == 0


def test_tiled_products_keep_their_sums_in_registers(kernels):  # noqa: F811
    tiled = {n: v for n, v in kernels.items() if any(k in n for k in ("11wide_kernel", "13direct_kernel", "14product_kernel"))}
    assert len([n for n in tiled if "wide_kernel" in n]) == 8
    # (large tiles: a few words outside the loop over k, whose 256 sums and operands take all 512 registers)
    assert {n: v for n, v in tiled.items() if v[1] > (64 if "wide_kernel" in n else 0)} == {}


def test_work_bytes_of_sizes_of_zero():
    from liteform_ae_amd import _lib
    lib = _lib.load()
    for m in (0, 1, 700):
        for n in (0, 1, 300):
            for k in (0, 1, 300):
                lib.lf_linear_work_bytes(m, n, k, _lib.LF_DTYPE_BF16)
                for act in (_lib.LF_ACT_NONE, _lib.LF_ACT_GELU):
                    need = lib.lf_linear_grad_work_bytes(m, n, k, _lib.LF_DTYPE_BF16, act, 1, 1, 1)
                    assert need == 0 or m * n > 0
    for rows, dim in ((0, 8), (8, 0), (0, 0), (-1, 8), (8, -1)):
        assert lib.lf_rms_norm_grad_work_bytes(rows, dim) == 0
