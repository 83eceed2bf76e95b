"""Sizes of a gated product that cannot be doubled are refused, not wrapped around; no GPU needed."""
import ctypes as C

import pytest

from liteform_ae_amd import _lib

AT = 1 << 40                                                             # an address that nothing reads
BF16, F32 = _lib.LF_DTYPE_BF16, _lib.LF_DTYPE_F32


@pytest.mark.parametrize("n,status", [(-(1 << 63), _lib.LF_ERR_INVALID), (-(1 << 62), _lib.LF_ERR_INVALID), (-1, _lib.LF_ERR_INVALID), ((1 << 23) + 1, _lib.LF_ERR_UNSUPPORTED),
                                      ((1 << 24) + 1, _lib.LF_ERR_UNSUPPORTED), (1 << 62, _lib.LF_ERR_UNSUPPORTED), ((1 << 62) + 8, _lib.LF_ERR_UNSUPPORTED),
                                      ((1 << 63) - 1, _lib.LF_ERR_UNSUPPORTED)])
def test_features_that_cannot_be_doubled(n, status):
    lib = _lib.load()
    a = _lib.LinearArgs(x=AT, w=AT, y=AT * 2, ld_x=64, ld_w=64, ld_y=1 << 30, ld_z=1 << 30, m=100, n=n, k=64, dtype=BF16, y_dtype=BF16, z_dtype=BF16)
    assert lib.lf_gated_linear(C.byref(a), AT, 1 << 40, None) == status, _lib.last_error()
    a = _lib.LinearGradArgs(dy=AT, z=AT, x=AT, w=AT, dx=AT, dw=AT, db=AT, ld_dy=1 << 30, ld_z=1 << 30, ld_x=64, ld_w=64, ld_dx=64, ld_dw=64, m=100, n=n, k=64, dtype=BF16, db_dtype=F32)
    assert lib.lf_gated_linear_grad(C.byref(a), AT, 1 << 40, None) == status, _lib.last_error()
    if abs(n) > 1 << 24:
        assert lib.lf_gated_linear_work_bytes(100, n, 64, BF16) == 0 and lib.lf_gated_linear_grad_work_bytes(100, n, 64, BF16, 1, 1, 1) == 0
