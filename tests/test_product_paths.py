"""Which kernel a dense product takes (csrc/lf_cut.h, compiled for the host), and that the sizes which test_gpu_product_paths.py runs on the GPU
reach each of them: with k whole and with a last step of less than 128 bytes, in one part and in several, with few workgroups and many."""
import ctypes

import pytest

from helpers import host_library

SOURCE = """
#include "lf_cut.h"
extern "C" void path(int bytes, long long m, long long n, long long k, int px, int qx, long long ld_p, long long ld_q, long long offset, int* out) {
    const lf::Path p = lf::path_of(bytes, {(const char*)nullptr + offset, ld_p, m, px != 0}, {nullptr, ld_q, n, qx != 0}, k);
    out[0] = p.kernel;
    out[1] = p.cut.tile;
    out[2] = p.deep;
    out[3] = p.cut.splits;
}
"""
FEW, PRODUCT, DIRECT, WIDE = range(4)

# rows, n, k of x w^T, all with rows of whole 16 bytes
FORWARD_16 = [(24, 72, 40), (24, 72, 64), (24, 72, 2056), (24, 72, 2048), (200, 4101, 40), (200, 4104, 64), (24, 1032, 6120), (25, 1031, 6144), (1541, 2051, 40), (1544, 2056, 64),
              (2056, 3080, 40), (2053, 3077, 64), (1032, 2056, 12_240), (1032, 2056, 12_288), (200, 4104, 12_240), (200, 4104, 12_288), (3083, 4101, 1032), (3080, 4104, 1024),
              (7001, 4099, 1024), (7003, 4097, 1032), (2616, 1541, 6120), (2617, 2392, 6144), (2616, 3080, 12_240), (2613, 3080, 12_288)]
FORWARD_8 = [(24, 72, 32), (24, 72, 512), (24, 72, 6112), (24, 72, 6144), (200, 4101, 32), (200, 4104, 512), (24, 2056, 6112), (24, 2056, 6144), (1541, 2051, 512), (1544, 2056, 32),
             (2056, 3080, 512), (2053, 3077, 32), (3083, 4101, 2048), (2056, 4104, 6112), (2616, 1541, 12_240), (2616, 1544, 12_288), (7001, 4099, 2048), (7003, 4097, 2064)]
# m, n, k of dy [m][n], x [m][k], w [n][k]: dx takes (m, k, n) with w across, dw (n, k, m) with dy and x across
GRAD_16 = [(24, 40, 72), (40, 24, 72), (64, 24, 72), (24, 64, 72), (24, 2056, 72), (2059, 24, 72), (2048, 24, 72), (24, 2048, 72), (200, 40, 4104), (43, 200, 4104), (200, 64, 4104),
           (64, 200, 4104), (24, 6120, 1032), (6121, 24, 1032), (24, 6144, 1032), (6144, 24, 1032), (1541, 40, 2056), (40, 1544, 2056), (1544, 64, 2056), (64, 1544, 2056),
           (2053, 40, 3080), (43, 2056, 3080), (2056, 64, 3080), (64, 2056, 3080), (1032, 12_240, 2056), (12_241, 1032, 2056), (1032, 12_288, 2056), (12_288, 1032, 2056),
           (200, 12_240, 4104), (12_241, 200, 4104), (200, 12_288, 4104), (12_288, 200, 4104), (3083, 1032, 4104), (1033, 3080, 4104), (3080, 1024, 4104), (1024, 3080, 4104),
           (2613, 6120, 1544), (6121, 2616, 1544), (2616, 6144, 1544), (6144, 2616, 1544), (2616, 12_240, 3080), (12_241, 2616, 3080), (2616, 12_288, 3080), (12_288, 2616, 3080), (7001, 1024, 4104), (7003, 1032, 4104), (1024, 7000, 4104), (1033, 7000, 4104)]


@pytest.fixture(scope="module")
def path(tmp_path_factory):
    lib = host_library(tmp_path_factory.mktemp("paths"), SOURCE)

    def of(size, m, n, k, px=False, qx=False, ld_p=None, ld_q=None, offset=0):
        out = (ctypes.c_int * 4)()
        lib.path(size, *map(ctypes.c_longlong, (m, n, k)), int(px), int(qx), *map(ctypes.c_longlong, (ld_p or (m if px else k), ld_q or (n if qx else k), offset)), out)
        return tuple(out)
    return of


def kind(path, size, m, n, k, px=False, qx=False):
    kernel, tile, deep, splits = path(size, m, n, k, px, qx)
    return kernel, tile, bool(deep), splits > 1, k % (128 // size) > 0


def kinds(*kernels):
    return {(kernel, tile, deep, parts, tail) for kernel, tile, deep in kernels for parts in (False, True) for tail in (False, True)}


SMALL = [(DIRECT, 64, False), (DIRECT, 64, True), (DIRECT, 128, False), (DIRECT, 128, True)]
LARGE = kinds((WIDE, 256, False), (WIDE, 256, True))


def test_forward_sizes_reach_each_kernel(path):
    want = kinds(*SMALL) | LARGE
    assert {kind(path, 2, *shape) for shape in FORWARD_16} >= want
    # (128-byte steps hold twice as many elements: the same sizes have half the parts)
    assert {kind(path, 1, *shape) for shape in FORWARD_8} >= kinds((DIRECT, 64, True), (DIRECT, 64, False)) | kinds((WIDE, 256, True)) | {
        (kernel, tile, deep, False, tail) for kernel, tile, deep in [*SMALL, (WIDE, 256, False)] for tail in (False, True)}


def test_gradient_sizes_reach_each_kernel(path):
    want = kinds(*SMALL) | LARGE
    assert {kind(path, 2, m, k, n, False, True) for m, n, k in GRAD_16} >= want
    assert {kind(path, 2, n, k, m, True, True) for m, n, k in GRAD_16} >= want


def test_operands_that_are_not_aligned_go_through_registers(path):
    assert path(2, 5000, 2600, 1032)[:2] == (WIDE, 256)
    for off in ({"offset": 2}, {"offset": 8}, {"ld_p": 1036}, {"ld_q": 1033}, {"ld_p": 1 << 23}):
        assert path(2, 5000, 2600, 1032, **off)[:2] == (PRODUCT, 128)
    assert path(2, 2616, 2392, 6121, True, True)[:2] == (WIDE, 256)               # (k across: any)
    assert path(2, 2617, 2392, 6120, True, True, ld_p=2624)[:2] == (PRODUCT, 128)  # (a last piece that is not whole)
    assert path(4, 5000, 2600, 1032)[:2] == (PRODUCT, 128) and path(4, 24, 72, 64)[0] == PRODUCT
    assert path(2, 16, 72, 64)[0] == FEW and path(2, 17, 72, 64)[0] == DIRECT and path(2, 16, 72, 64, False, True)[0] == DIRECT
