"""Layer norm, gated product, embedding and clipping without a GPU: they raise, and the library refuses what it must before anything is launched."""
import ctypes as C

import pytest
import torch

from liteform_ae_amd import _lib

F32, BF16, E4M3 = _lib.LF_DTYPE_F32, _lib.LF_DTYPE_BF16, _lib.LF_DTYPE_E4M3
AT = 1 << 40                                                             # an address that nothing reads


@pytest.mark.skipif(torch.cuda.is_available(), reason="only meaningful where no GPU is visible")
def test_operators_raise_without_gpu():
    from liteform_ae_amd import layer_ops as lo
    x, w, ids = torch.ones(4, 8), torch.ones(8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: lo.layer_norm(x, w), lambda: lo.layer_norm_8bit(x), lambda: lo.layer_norm_grad(x, x), lambda: lo.gated_linear(x, x),
                 lambda: lo.gated_linear_8bit(x.to(torch.int8), w[:4], x.to(torch.int8), w[:4]), lambda: lo.gated_linear_grad(x[:, :2], x, x, x[:, :4]),
                 lambda: lo.embedding(ids, x), lambda: lo.embedding_grad(x, ids, 5), lambda: lo.clip_gradients([x], 1.0), lambda: lo.gradient_norm([x])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def refused(rc, status=_lib.LF_ERR_INVALID, text=None):
    assert rc == status, (rc, _lib.last_error())
    assert text is None or text in _lib.last_error()


def test_layer_norm_refusals():
    lib = _lib.load()
    good = dict(x=AT, y=AT * 2, ld_x=8, ld_y=8, rows=4, dim=8, eps=1e-5)

    def call(**change):
        return lib.lf_layer_norm(C.byref(_lib.LayerNormArgs(**{**good, **change})), None)

    refused(lib.lf_layer_norm(None, None))
    for change in (dict(x=None), dict(y=None), dict(ld_x=7), dict(ld_y=7), dict(eps=-1.0), dict(dim=0), dict(rows=-1), dict(residual=AT), dict(h=AT), dict(y_dtype=E4M3), dict(scale=AT),
                   dict(x=AT + 2), dict(eps=float("nan")), dict(residual=AT, h=AT, ld_residual=7, ld_h=8)):
        refused(call(**change))
    for change in (dict(x_dtype=9), dict(y_dtype=9), dict(weight=AT, weight_dtype=E4M3), dict(bias=AT, bias_dtype=9), dict(dim=(1 << 24) + 1, ld_x=1 << 25, ld_y=1 << 25)):
        refused(call(**change), _lib.LF_ERR_UNSUPPORTED)
    assert call(rows=0, x=None, y=None) == 0
    good = dict(dy=AT, h=AT, dx=AT * 2, ld_dy=8, ld_h=8, ld_dx=8, rows=4000, dim=8, eps=1e-5)

    def grad(work=None, size=0, **change):
        return lib.lf_layer_norm_grad(C.byref(_lib.LayerNormGradArgs(**{**good, **change})), work, size, None)

    need = lib.lf_layer_norm_grad_work_bytes(4000, 8)
    assert need > 0
    for change in (dict(dy=None), dict(h=None), dict(dx=None), dict(ld_dx=7), dict(dh=AT, ld_dh=7), dict(eps=-1.0), dict(dw=AT), dict(db=AT), dict(dw=AT, work=AT + 8, size=need)):
        refused(grad(**change))
    refused(grad(dw=AT, work=AT, size=need - 1), _lib.LF_ERR_WORKSPACE)
    refused(grad(db=AT, db_dtype=E4M3, work=AT, size=need), _lib.LF_ERR_UNSUPPORTED)
    for rows, dim in ((0, 8), (8, 0), (0, 0), (-1, 8), (8, -1), (1, 8)):
        assert lib.lf_layer_norm_grad_work_bytes(rows, dim) == 0


def test_gated_refusals():
    lib = _lib.load()
    good = dict(x=AT, w=AT, y=AT * 2, ld_x=64, ld_w=64, ld_y=32, ld_z=64, m=100, n=32, k=64, dtype=BF16, y_dtype=BF16, z_dtype=BF16)

    def call(work=AT, size=1 << 40, **change):
        return lib.lf_gated_linear(C.byref(_lib.LinearArgs(**{**good, **change})), work, size, None)

    refused(lib.lf_gated_linear(None, None, 0, None))
    for change in (dict(x=None), dict(w=None), dict(y=None), dict(ld_x=63), dict(ld_w=63), dict(ld_y=31), dict(z=AT, ld_z=63), dict(n=-1), dict(m=-1), dict(residual=AT), dict(x_scale=AT),
                   dict(dtype=E4M3)):
        refused(call(**change))
    for change in (dict(dtype=9), dict(activation=7), dict(y_dtype=E4M3), dict(n=1 << 24), dict(bias=AT, bias_dtype=9)):
        refused(call(**change), _lib.LF_ERR_UNSUPPORTED)
    assert call(m=0) == 0 and call(n=0) == 0
    good = dict(dy=AT, z=AT, x=AT, w=AT, dx=AT, dw=AT, db=AT, ld_dy=32, ld_z=64, ld_x=64, ld_w=64, ld_dx=64, ld_dw=64, m=100, n=32, k=64, dtype=BF16, db_dtype=F32)

    def grad(work=AT, size=1 << 40, **change):
        return lib.lf_gated_linear_grad(C.byref(_lib.LinearGradArgs(**{**good, **change})), work, size, None)

    for change in (dict(dy=None), dict(z=None), dict(x=None), dict(w=None), dict(ld_z=63), dict(ld_dy=31), dict(ld_dx=63), dict(ld_dw=63), dict(work=None, size=0), dict(work=AT + 8)):
        refused(grad(**change))
    refused(grad(size=16), _lib.LF_ERR_WORKSPACE)
    refused(grad(dtype=E4M3), _lib.LF_ERR_UNSUPPORTED)
    for m in (0, 1, 700):
        for n in (0, 1, 300):
            for k in (0, 1, 300):
                lib.lf_gated_linear_work_bytes(m, n, k, BF16)
                assert lib.lf_gated_linear_grad_work_bytes(m, n, k, BF16, 1, 1, 1) == 0 or m * n > 0


def test_embedding_refusals():
    lib = _lib.load()
    good = dict(ids=AT, table=AT, y=AT * 2, ids_stride=1, ld_table=8, ld_y=8, n=4, rows=5, dim=8, ids_bits=64, scale=1.0)

    def call(**change):
        return lib.lf_embedding(C.byref(_lib.EmbeddingArgs(**{**good, **change})), None)

    refused(lib.lf_embedding(None, None))
    for change in (dict(ids=None), dict(table=None), dict(y=None), dict(ids=AT + 4), dict(ids_stride=-1), dict(ld_table=7), dict(ld_y=7), dict(n=-1), dict(rows=-1), dict(dim=0),
                   dict(y=AT + 2)):
        refused(call(**change))
    for change in (dict(ids_bits=16), dict(table_dtype=E4M3), dict(y_dtype=9), dict(n=1 << 31), dict(rows=1 << 31), dict(dim=(1 << 24) + 1, ld_table=1 << 25, ld_y=1 << 25)):
        refused(call(**change), _lib.LF_ERR_UNSUPPORTED)
    assert call(n=0, ids=None, y=None) == 0
    good = dict(dy=AT, ids=AT, grad=AT * 2, ids_stride=1, ld_dy=8, ld_grad=8, n=4, rows=5, dim=8, ids_bits=32, scale=1.0)
    need = lib.lf_embedding_grad_work_bytes(4, 5, 8, F32)

    def grad(work=AT, size=need, **change):
        return lib.lf_embedding_grad(C.byref(_lib.EmbeddingGradArgs(**{**good, **change})), work, size, None)

    for change in (dict(dy=None), dict(ids=None), dict(grad=None), dict(ld_dy=7), dict(ld_grad=7), dict(work=None), dict(work=AT + 8), dict(ids=AT + 2)):
        refused(grad(**change))
    refused(grad(size=need - 1), _lib.LF_ERR_WORKSPACE)
    assert grad(rows=0, grad=None) == 0
    for n, rows in ((0, 5), (4, 0), (-1, 5), (4, -1), (1 << 31, 5), (4, 1 << 31)):
        assert lib.lf_embedding_grad_work_bytes(n, rows, 8, F32) == 0


def descs(*tensors):
    return (_lib.TensorDesc * len(tensors))(*[_lib.TensorDesc(**{**dict(src=AT, dst=AT * 2, rows=1, cols=100), **t}) for t in tensors])


def clip(lib, list_, most=1.0, eps=0.0, norm=AT * 3, work=AT, size=None):
    n = 0 if list_ is None else len(list_)
    return lib.lf_clip_gradients(list_, n, most, eps, norm, work, lib.lf_clip_work_bytes(n) if size is None else size, None)


def test_clip_refusals():
    lib = _lib.load()
    refused(lib.lf_clip_gradients(None, 1, 1.0, 0.0, AT, AT, 1 << 20, None))
    refused(clip(lib, descs({}), norm=None))
    refused(clip(lib, descs({}), most=-1.0))
    refused(clip(lib, descs({}), most=float("nan")))
    refused(clip(lib, descs({}), eps=-1.0))
    refused(clip(lib, descs({}), work=None))
    refused(clip(lib, descs({}), work=AT + 8))
    refused(clip(lib, descs({}), size=15), _lib.LF_ERR_WORKSPACE)
    for bad in (dict(src=None), dict(src=AT + 2), dict(dst=AT + 1), dict(rows=-1), dict(cols=-1), dict(rows=3, ld_src=99, ld_dst=100), dict(rows=3, ld_src=100, ld_dst=99)):
        refused(clip(lib, descs(bad)))
    refused(clip(lib, descs(dict(dtype=E4M3))), _lib.LF_ERR_UNSUPPORTED)
    for huge in (dict(cols=1 << 62), dict(rows=1 << 62, cols=1), dict(rows=1 << 40, cols=1 << 40), dict(rows=2, ld_src=1 << 62, ld_dst=100), dict(rows=2, ld_src=100, ld_dst=1 << 62)):
        refused(clip(lib, descs(huge)), _lib.LF_ERR_UNSUPPORTED)
    refused(clip(lib, descs(*[dict(cols=1 << 39, src=AT, dst=AT + (i << 42)) for i in range(3)])), _lib.LF_ERR_UNSUPPORTED)
    refused(clip(lib, descs({}, dict(src=AT + 4096, dst=None))), text="for all tensors or for none")
    assert lib.lf_clip_work_bytes(0) == 0 and lib.lf_clip_work_bytes(-3) == 0 and lib.lf_clip_work_bytes(100) >= 100 * 8


# (the first without an output: its address would be null)
@pytest.mark.parametrize("nones", [(0,), (1,), (2,), (0, 1), (0, 2), (1, 2)])
def test_clip_refuses_some_outputs_without_the_others(nones):
    lib = _lib.load()
    some = [dict(src=AT + 4096 * i, dst=None if i in nones else AT * 2 + 4096 * i) for i in range(3)]
    refused(clip(lib, descs(*some)), text="for all tensors or for none")
    empty = dict(src=None, dst=None, rows=0)
    refused(clip(lib, descs(empty, *some, empty)), text="for all tensors or for none")


#  float32 elements of 4 bytes: 100 of them take 400
LIES = [
    [dict(src=AT, dst=AT), dict(src=AT, dst=AT)],                                                        # the same one twice
    [dict(src=AT, dst=AT), dict(src=AT + 396, dst=AT + 396)],                                            # one element of both
    [dict(src=AT, dst=AT + 4)],                                                                          # its own elements in other places
    [dict(src=AT, dst=AT * 2), dict(src=AT * 3, dst=AT + 200)],                                          # an output on another one's input
    [dict(src=AT, dst=AT * 2), dict(src=AT * 3, dst=AT * 2)],                                            # one output for two
    [dict(src=AT, dst=AT, rows=5, cols=60, ld_src=100, ld_dst=100), dict(src=AT + 236, dst=AT + 236, rows=5, cols=41, ld_src=100, ld_dst=100)],
    [dict(src=AT, dst=AT, rows=5, cols=60, ld_src=100, ld_dst=100), dict(src=AT + 240, dst=AT + 240, rows=5, cols=41, ld_src=100, ld_dst=100)],     # (reaches into the next row)
    [dict(src=AT, dst=AT, rows=5, cols=60, ld_src=100, ld_dst=100), dict(src=AT + 240, dst=AT + 240, rows=4, cols=40, ld_src=101, ld_dst=101)],
    [dict(src=AT, dst=AT, rows=5, cols=60, ld_src=100, ld_dst=100), dict(src=AT + 640, dst=AT + 640, cols=41)],
    [dict(src=AT, dst=AT, rows=5, cols=10, ld_src=100, ld_dst=50)],
]


@pytest.mark.parametrize("number", range(len(LIES)))
def test_clip_refuses_outputs_on_other_tensors(number):
    lib = _lib.load()
    refused(clip(lib, descs(*LIES[number])), text="lies on another tensor")
    refused(clip(lib, descs(*reversed(LIES[number]))), text="lies on another tensor")
    # among others that are apart
    apart = [dict(src=AT * 8 + 4096 * i, dst=AT * 9 + 4096 * i) for i in range(200)]
    refused(clip(lib, descs(*apart[:100], *LIES[number], *apart[100:])), text="lies on another tensor")
