"""What a graph layer does beside the sparse product: the norm of the aggregated features with the residual stream's
addition, and the dense transform with its epilogue - forward, in 8 bits, and backward.

    C = HybSpMM(...).run(y)                                       # aggregation (format_algos)
    y, h = rms_norm(C, w, residual=h)                             # h += C; y = norm(h) * w
    y = linear(y, W, b, activation="gelu", residual=r)            # act(y W^T + b) + r

    q, s, h = rms_norm_8bit(C, w, residual=h)                     # the same layer served in 8 bits
    y = linear_8bit(q, s, Wq, Ws, b, activation="gelu")           # Wq, Ws = quantize_rows(W), once

The reference ends with the sparse product (format_algos.py:388-605) and has no counterpart.  Everything runs in
``liblfhip.so`` (``lf_rms_norm``, ``lf_linear``, ...) on the current stream of the current device; there is no CPU path.

Matrices are CUDA tensors (rows, features) whose rows are contiguous; the distance from one row to the next is free, so a
slice of a wider buffer's columns needs no copy.  float32, bfloat16 and float16, sums in 32 bits.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .format_algos import _stream, _torch

ACTIVATIONS = {None: _lib.LF_ACT_NONE, "relu": _lib.LF_ACT_RELU, "gelu": _lib.LF_ACT_GELU, "silu": _lib.LF_ACT_SILU}

_FLOATS = {}
_EIGHTS = {}


def _types():
    """(floating types, 8-bit types), torch dtype -> code of the library."""
    if not _FLOATS:
        torch = _torch()
        _EIGHTS.update({torch.float8_e4m3fn: _lib.LF_DTYPE_E4M3, torch.int8: _lib.LF_DTYPE_I8})
        _FLOATS.update({torch.float32: _lib.LF_DTYPE_F32, torch.bfloat16: _lib.LF_DTYPE_BF16, torch.float16: _lib.LF_DTYPE_F16})
    return _FLOATS, _EIGHTS


def _matrix(name, t, types, shape=None):
    """(address, elements from row to row, type) of a matrix operand; ValueError unless it is one."""
    code = types.get(t.dtype)
    if code is None or not t.is_cuda or t.dim() != 2 or (shape is not None and t.shape != shape):
        want = "(rows, features)" if shape is None else tuple(shape)
        raise ValueError(f"{name} must be a CUDA tensor of shape {want} and one of {[str(d) for d in types]}, "
                         f"got {tuple(t.shape)} of {t.dtype} on {t.device}")
    rows, cols = t.shape
    across, along = t.stride()
    if cols > 1 and along != 1 or rows > 1 and across < cols:
        raise ValueError(f"the rows of {name} must be contiguous and must not overlap (strides {t.stride()})")
    return t.data_ptr(), max(across, cols), code


def _vector(name, t, types, size):
    code = types.get(t.dtype)
    if code is None or not t.is_cuda or t.dim() != 1 or t.shape[0] != size or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA tensor of {size} elements and one of {[str(d) for d in types]}, "
                         f"got {tuple(t.shape)} of {t.dtype} on {t.device}")
    return t.data_ptr(), code


def _scales(name, t, size):
    if t.dtype is not _torch().float32:
        raise ValueError(f"{name} must be float32, got {t.dtype}")
    return _vector(name, t, _FLOATS, size)[0]


def _one_device(torch, *tensors):
    here = torch._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.get_device() != here:
            raise ValueError(f"operands must be on the current device, cuda:{here}, got one on {t.device}")


def _activation(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"unknown activation {name!r}: one of {list(ACTIVATIONS)}") from None


def _float_type(name, dtype):
    if dtype not in _FLOATS:
        raise ValueError(f"{name} must be one of {[str(d) for d in _FLOATS]}, got {dtype}")
    return dtype


def _workspace(torch, like, nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


# --------------------------------------------------------------------------- norm


def _norm(x, weight, residual, eps, dtype, code, eight):
    torch, lib = _torch(), _lib.load()
    floats, _ = _types()
    _one_device(torch, x, weight, residual)
    rows, dim = x.shape if x.dim() == 2 else (0, 0)
    xp, ldx, xt = _matrix("x", x, floats)
    wp, wt = (None, 0) if weight is None else _vector("weight", weight, floats, dim)
    h = scale = None
    rp, ldr, rt, hp = None, 0, 0, None
    if residual is not None:
        rp, ldr, rt = _matrix("residual", residual, floats, x.shape)
        h = torch.empty((rows, dim), dtype=residual.dtype, device=x.device)
        hp = h.data_ptr()
    y = torch.empty((rows, dim), dtype=dtype, device=x.device)
    if eight:
        scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    rc = lib.lf_rms_norm(xp, ldx, xt, rp, ldr, rt, wp, wt, rows, dim, eps, y.data_ptr(), dim, code,
                         None if scale is None else scale.data_ptr(), hp, dim, _stream())
    if rc:
        _lib.check(rc)
    return y, scale, h


def rms_norm(x, weight=None, residual=None, eps: float = 1e-6, out_dtype=None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` with ``h = x + residual``, by rows.  Returns ``y``, and with a residual
    ``(y, h)``: h, the stream that the next layer adds to, in the residual's type, y in ``out_dtype`` (default: x's).  The
    norm is of h before that rounding.  x and residual may be of different types (an f32 product, a bf16 stream)."""
    _torch()
    floats, _ = _types()
    dtype = _float_type("out_dtype", x.dtype if out_dtype is None else out_dtype)
    y, _, h = _norm(x, weight, residual, eps, dtype, floats[dtype], False)
    return y if residual is None else (y, h)


def rms_norm_8bit(x, weight=None, residual=None, eps: float = 1e-6, dtype=None):
    """``rms_norm`` with y in 8 bits: ``(q, scale)``, and with a residual ``(q, scale, h)``.  ``q * scale[:, None]`` stands for y;
    ``scale`` (float32) is the row's largest magnitude over 448 for ``torch.float8_e4m3fn`` (the default) or over 127 for
    ``torch.int8``, 0 for a row of zeros and NaN for a row that holds Inf or NaN."""
    dtype, code = _eight(dtype)
    q, scale, h = _norm(x, weight, residual, eps, dtype, code, True)
    return (q, scale) if residual is None else (q, scale, h)


def _eight(dtype):
    torch = _torch()
    eights = _types()[1]
    dtype = torch.float8_e4m3fn if dtype is None else dtype
    if dtype not in eights:
        raise ValueError(f"dtype must be one of {[str(d) for d in eights]}, got {dtype}")
    return dtype, eights[dtype]


def quantize_rows(x, dtype=None):
    """Rows of x in 8 bits with a scale each: ``(q, scale)`` as ``rms_norm_8bit`` gives them.  For the weight of
    ``linear_8bit``, once."""
    torch, lib = _torch(), _lib.load()
    dtype, code = _eight(dtype)
    _one_device(torch, x)
    xp, ldx, xt = _matrix("x", x, _FLOATS)
    rows, dim = x.shape
    q = torch.empty((rows, dim), dtype=dtype, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    rc = lib.lf_quantize_rows(xp, ldx, xt, rows, dim, q.data_ptr(), dim, code, scale.data_ptr(), _stream())
    if rc:
        _lib.check(rc)
    return q, scale


def rms_norm_grad(dy, h, weight=None, eps: float = 1e-6, dh=None):
    """``(dx, dweight)`` of ``rms_norm`` from the gradient ``dy`` of y and the ``h`` that it returned (x where there was no
    residual).  dx, in h's type, is the gradient of x and of the residual alike; ``dh``, the gradient that comes down the
    residual stream, is added to it.  dweight, in the weight's type, is None without a weight."""
    torch, lib = _torch(), _lib.load()
    floats, _ = _types()
    _one_device(torch, dy, h, weight, dh)
    hp, ldh, ht = _matrix("h", h, floats)
    rows, dim = h.shape
    gp, ldg, gt = _matrix("dy", dy, floats, h.shape)
    wp, wt = (None, 0) if weight is None else _vector("weight", weight, floats, dim)
    dp, ldd = None, 0
    if dh is not None:
        dp, ldd, dt = _matrix("dh", dh, floats, h.shape)
        if dt != ht:
            raise ValueError(f"dh must have h's type {h.dtype}, got {dh.dtype}")
    dx = torch.empty((rows, dim), dtype=h.dtype, device=h.device)
    dw = work = None
    nbytes = 0
    if weight is not None:
        dw = torch.empty(dim, dtype=weight.dtype, device=h.device)
        nbytes = lib.lf_rms_norm_grad_work_bytes(rows, dim)
        work = _workspace(torch, h, nbytes)
    rc = lib.lf_rms_norm_grad(gp, ldg, gt, hp, ldh, ht, wp, wt, dp, ldd, rows, dim, eps, dx.data_ptr(), dim,
                              None if dw is None else dw.data_ptr(), None if work is None else work.data_ptr(), nbytes, _stream())
    if rc:
        _lib.check(rc)
    return dx, dw


# --------------------------------------------------------------------------- product


def _linear(torch, lib, x, weight, x_scale, w_scale, bias, activation, residual, types, out_dtype, z_dtype):
    floats, _ = _types()
    act = _activation(activation)
    _one_device(torch, x, weight, x_scale, w_scale, bias, residual)
    a = _lib.LinearArgs()
    a.x, a.ld_x, a.dtype = _matrix("x", x, types)
    a.w, a.ld_w, wt = _matrix("weight", weight, types)
    m, k = x.shape
    n = weight.shape[0]
    if wt != a.dtype or weight.shape[1] != k:
        raise ValueError(f"weight must be (features out, {k}) of {x.dtype}, got {tuple(weight.shape)} of {weight.dtype}")
    a.m, a.n, a.k, a.activation = m, n, k, act
    if x_scale is not None:
        a.x_scale, a.w_scale = _scales("x_scale", x_scale, m), _scales("weight_scale", w_scale, n)
    if bias is not None:
        a.bias, a.bias_dtype = _vector("bias", bias, floats, n)
    if residual is not None:
        a.residual, a.ld_residual, a.residual_dtype = _matrix("residual", residual, floats, (m, n))
    y = torch.empty((m, n), dtype=out_dtype, device=x.device)
    a.y, a.ld_y, a.y_dtype = y.data_ptr(), n, floats[out_dtype]
    z = None
    if z_dtype is not None:
        z = torch.empty((m, n), dtype=z_dtype, device=x.device)
        a.z, a.ld_z, a.z_dtype = z.data_ptr(), n, floats[z_dtype]
    nbytes = lib.lf_linear_work_bytes(m, n, k, a.dtype)
    work = _workspace(torch, x, nbytes)
    rc = lib.lf_linear(C.addressof(a), None if work is None else work.data_ptr(), nbytes, _stream())
    if rc:
        _lib.check(rc)
    return y, z


def linear(x, weight, bias=None, activation=None, residual=None, out_dtype=None, return_preactivation: bool = False):
    """``y = act(x weight^T + bias) + residual`` for x (rows, k) and weight (n, k) of one type; ``activation`` is None, "relu",
    "gelu" (by erf) or "silu".  bias and residual are floating tensors of any type, y is of ``out_dtype`` (default: x's).
    ``return_preactivation=True`` returns ``(y, z)`` with z = x weight^T + bias in x's type, which ``linear_grad`` needs behind an
    activation.  float32 products are as exact as float32 sums of float32 products."""
    torch, lib = _torch(), _lib.load()
    floats, _ = _types()
    out = _float_type("out_dtype", x.dtype if out_dtype is None else out_dtype)
    y, z = _linear(torch, lib, x, weight, None, None, bias, activation, residual, floats, out, x.dtype if return_preactivation else None)
    return (y, z) if return_preactivation else y


def linear_8bit(x, x_scale, weight, weight_scale, bias=None, activation=None, residual=None, out_dtype=None):
    """``linear`` of rows in 8 bits, both ``torch.float8_e4m3fn`` or both ``torch.int8``, each row of x and of weight with its scale
    (``rms_norm_8bit``, ``quantize_rows``).  y is of ``out_dtype`` (default bfloat16).  int8: at most 131071 features in."""
    torch, lib = _torch(), _lib.load()
    _, eights = _types()
    out = _float_type("out_dtype", torch.bfloat16 if out_dtype is None else out_dtype)
    return _linear(torch, lib, x, weight, x_scale, weight_scale, bias, activation, residual, eights, out, None)[0]


def linear_grad(dy, x, weight, z=None, activation=None, bias_dtype=None, want_dx: bool = True, want_dweight: bool = True):
    """``(dx, dweight, dbias)`` of ``linear`` from the gradient ``dy`` of y: dz = dy act'(z), dx = dz weight, dweight = dz^T x, dbias =
    column sums of dz.  All of one type but dbias, which is of ``bias_dtype`` (None: not computed).  ``z`` is what
    ``linear(..., return_preactivation=True)`` returned; without an activation it is not needed.  Gradients that are not
    wanted are None.  The residual's gradient is dy.  Behind an activation dz is rounded to the operands' type before the
    products, as they take it."""
    torch, lib = _torch(), _lib.load()
    floats, _ = _types()
    act = _activation(activation)
    _one_device(torch, dy, x, weight, z)
    a = _lib.LinearGradArgs()
    a.x, a.ld_x, a.dtype = _matrix("x", x, floats)
    a.w, a.ld_w, wt = _matrix("weight", weight, floats)
    m, k = x.shape
    n = weight.shape[0]
    if wt != a.dtype or weight.shape[1] != k:
        raise ValueError(f"weight must be (features out, {k}) of {x.dtype}, got {tuple(weight.shape)} of {weight.dtype}")
    a.dy, a.ld_dy, gt = _matrix("dy", dy, floats, (m, n))
    if gt != a.dtype:
        raise ValueError(f"dy must have x's type {x.dtype}, got {dy.dtype}")
    if act != _lib.LF_ACT_NONE:
        if z is None:
            raise ValueError("the gradient of an activation needs z: linear(..., return_preactivation=True)")
        a.z, a.ld_z, zt = _matrix("z", z, floats, (m, n))
        if zt != a.dtype:
            raise ValueError(f"z must have x's type {x.dtype}, got {z.dtype}")
    a.m, a.n, a.k, a.activation = m, n, k, act
    dx = dw = db = None
    if want_dx:
        dx = torch.empty((m, k), dtype=x.dtype, device=x.device)
        a.dx, a.ld_dx = dx.data_ptr(), k
    if want_dweight:
        dw = torch.empty((n, k), dtype=x.dtype, device=x.device)
        a.dw, a.ld_dw = dw.data_ptr(), k
    if bias_dtype is not None:
        db = torch.empty(n, dtype=_float_type("bias_dtype", bias_dtype), device=x.device)
        a.db, a.db_dtype = db.data_ptr(), floats[bias_dtype]
    nbytes = lib.lf_linear_grad_work_bytes(m, n, k, a.dtype, act, want_dx, want_dweight, db is not None)
    work = _workspace(torch, x, nbytes)
    rc = lib.lf_linear_grad(C.addressof(a), None if work is None else work.data_ptr(), nbytes, _stream())
    if rc:
        _lib.check(rc)
    return dx, dw, db
