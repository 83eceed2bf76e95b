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

What is returned is no part of a torch graph: gradients are those of ``rms_norm_grad`` and ``linear_grad``.  Tensors that require
gradients are taken under ``torch.no_grad()`` only, and refused where torch would expect a graph.
"""
from __future__ import annotations

import struct

from . import _lib
from .format_algos import _stream, _torch

ACTIVATIONS = {None: _lib.LF_ACT_NONE, "relu": _lib.LF_ACT_RELU, "gelu": _lib.LF_ACT_GELU, "silu": _lib.LF_ACT_SILU}

_FLOATS = {}                      # torch dtype -> code of the library
_EIGHTS = {}
# struct lf_linear_args and lf_linear_grad_args in one call each: a field at a time they cost as much as the launch
_LINEAR_ARGS = struct.Struct("8Q8q6i").pack
_LINEAR_GRAD_ARGS = struct.Struct("7Q9q3i4x").pack


def _begin():
    """(torch, library, index of the current device)."""
    torch = _torch()
    if not _FLOATS:
        _EIGHTS.update({torch.float8_e4m3fn: _lib.LF_DTYPE_E4M3, torch.int8: _lib.LF_DTYPE_I8})
        _FLOATS.update({torch.float32: _lib.LF_DTYPE_F32, torch.bfloat16: _lib.LF_DTYPE_BF16, torch.float16: _lib.LF_DTYPE_F16})
    return torch, _lib.load(), torch._C._cuda_getDevice()


def refuse_graph(name, t):
    """ValueError where a gradient that torch is asked for would be lost without a word."""
    if t.requires_grad and _torch().is_grad_enabled():
        raise ValueError(f"{name} requires gradients, and what is returned would not lead back to it: call this under torch.no_grad() (or pass "
                         f"{name}.detach()) and take them from rms_norm_grad and linear_grad")


def _matrix(name, t, types, device, rows=None, cols=None):
    """(address, elements from row to row, type) of a matrix operand; ValueError unless it is one of the current device, and of
    (rows, cols) where they are given."""
    code = types.get(t.dtype)
    shape = t.shape
    if code is None or len(shape) != 2 or t.get_device() != device or (rows is not None and (shape[0] != rows or shape[1] != cols)):
        want = "(rows, features)" if rows is None else (rows, cols)
        raise ValueError(f"{name} must be a tensor of shape {want} on the current device, cuda:{device}, and one of {[str(d) for d in types]}, "
                         f"got {tuple(t.shape)} of {t.dtype} on {t.device}")
    if t.requires_grad:
        refuse_graph(name, t)
    across, along = t.stride()
    cols = shape[1]
    if (along != 1 and cols > 1) or (across < cols and shape[0] > 1):
        raise ValueError(f"the rows of {name} must be contiguous and must not overlap (strides {t.stride()})")
    return t.data_ptr(), across if across > cols else cols, code


def _vector(name, t, types, device, size):
    code = types.get(t.dtype)
    shape = t.shape
    if code is None or len(shape) != 1 or shape[0] != size or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {size} elements on the current device, cuda:{device}, and one of "
                         f"{[str(d) for d in types]}, got {tuple(t.shape)} of {t.dtype} on {t.device}")
    if t.requires_grad:
        refuse_graph(name, t)
    return t.data_ptr(), code


def _scales(torch, name, t, device, size):
    if t is None or t.dtype is not torch.float32:
        raise ValueError(f"{name} must be float32, got {None if t is None else t.dtype}")
    return _vector(name, t, _FLOATS, device, size)[0]


def _new(like, shape, dtype):
    return like.new_empty(shape) if dtype is like.dtype else like.new_empty(shape, dtype=dtype)


def _activation(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"unknown activation {name!r}: one of {list(ACTIVATIONS)}") from None


def _float_type(name, dtype):
    code = _FLOATS.get(dtype)
    if code is None:
        raise ValueError(f"{name} must be one of {[str(d) for d in _FLOATS]}, got {dtype}")
    return code


def _eight(torch, dtype):
    dtype = torch.float8_e4m3fn if dtype is None else dtype
    code = _EIGHTS.get(dtype)
    if code is None:
        raise ValueError(f"dtype must be one of {[str(d) for d in _EIGHTS]}, got {dtype}")
    return dtype, code


# --------------------------------------------------------------------------- norm


def _norm(torch, lib, device, x, weight, residual, eps, dtype, code, eight):
    xp, ldx, xt = _matrix("x", x, _FLOATS, device)
    rows, dim = x.shape
    wp, wt = (None, 0) if weight is None else _vector("weight", weight, _FLOATS, device, dim)
    h = scale = rp = hp = sp = None
    ldr = rt = 0
    if residual is not None:
        rp, ldr, rt = _matrix("residual", residual, _FLOATS, device, rows, dim)
        h = residual.new_empty((rows, dim))
        hp = h.data_ptr()
    y = _new(x, (rows, dim), dtype)
    if eight:
        scale = _new(x, (rows,), torch.float32)
        sp = scale.data_ptr()
    rc = lib.lf_rms_norm(xp, ldx, xt, rp, ldr, rt, wp, wt, rows, dim, eps, y.data_ptr(), dim, code, sp, hp, dim, _stream())
    if rc:
        _lib.check(rc)
    return y, scale, h


def rms_norm(x, weight=None, residual=None, eps: float = 1e-6, out_dtype=None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` with ``h = x + residual``, by rows.  Returns ``y``, and with a residual
    ``(y, h)``: h, the stream that the next layer adds to, in the residual's type, y in ``out_dtype`` (default: x's).  The
    norm is of h before that rounding.  x and residual may be of different types (an f32 product, a bf16 stream).  Rows whose squares
    overflow or vanish in 32 bits come out as any others; ``eps=0`` makes y of a row of zeros NaN."""
    torch, lib, device = _begin()
    dtype = x.dtype if out_dtype is None else out_dtype
    y, _, h = _norm(torch, lib, device, x, weight, residual, eps, dtype, _float_type("out_dtype", dtype), False)
    return y if residual is None else (y, h)


def rms_norm_8bit(x, weight=None, residual=None, eps: float = 1e-6, dtype=None):
    """``rms_norm`` with y in 8 bits: ``(q, scale)``, and with a residual ``(q, scale, h)``.  ``q * scale[:, None]`` stands for y;
    ``scale`` (float32) is the row's largest magnitude over 448 for ``torch.float8_e4m3fn`` (the default) or over 127 for
    ``torch.int8``, 0 for a row of zeros and NaN for a row that holds Inf or NaN."""
    torch, lib, device = _begin()
    dtype, code = _eight(torch, dtype)
    q, scale, h = _norm(torch, lib, device, x, weight, residual, eps, dtype, code, True)
    return (q, scale) if residual is None else (q, scale, h)


def quantize_rows(x, dtype=None):
    """Rows of x in 8 bits with a scale each: ``(q, scale)`` as ``rms_norm_8bit`` gives them.  For the weight of
    ``linear_8bit``, once."""
    torch, lib, device = _begin()
    dtype, code = _eight(torch, dtype)
    xp, ldx, xt = _matrix("x", x, _FLOATS, device)
    rows, dim = x.shape
    q, scale = _new(x, (rows, dim), dtype), _new(x, (rows,), torch.float32)
    rc = lib.lf_quantize_rows(xp, ldx, xt, rows, dim, q.data_ptr(), dim, code, scale.data_ptr(), _stream())
    if rc:
        _lib.check(rc)
    return q, scale


def rms_norm_grad(dy, h, weight=None, eps: float = 1e-6, dh=None):
    """``(dx, dweight)`` of ``rms_norm`` from the gradient ``dy`` of y and the ``h`` that it returned (x where there was no
    residual).  dx, in h's type, is the gradient of x and of the residual alike; ``dh``, the gradient that comes down the
    residual stream, is added to it.  dweight, in the weight's type, is None without a weight."""
    torch, lib, device = _begin()
    hp, ldh, ht = _matrix("h", h, _FLOATS, device)
    rows, dim = h.shape
    gp, ldg, gt = _matrix("dy", dy, _FLOATS, device, rows, dim)
    wp, wt = (None, 0) if weight is None else _vector("weight", weight, _FLOATS, device, dim)
    dp = dwp = kp = None
    ldd = nbytes = 0
    if dh is not None:
        dp, ldd, dt = _matrix("dh", dh, _FLOATS, device, rows, dim)
        if dt != ht:
            raise ValueError(f"dh must have h's type {h.dtype}, got {dh.dtype}")
    dx = h.new_empty((rows, dim))
    dw = None
    if weight is not None:
        dw = weight.new_empty((dim,))
        dwp = dw.data_ptr()
        nbytes = lib.lf_rms_norm_grad_work_bytes(rows, dim)
        if nbytes:
            work = h.new_empty((nbytes,), dtype=torch.uint8)
            kp = work.data_ptr()
    rc = lib.lf_rms_norm_grad(gp, ldg, gt, hp, ldh, ht, wp, wt, dp, ldd, rows, dim, eps, dx.data_ptr(), dim, dwp, kp, nbytes, _stream())
    if rc:
        _lib.check(rc)
    return dx, dw


# --------------------------------------------------------------------------- product


def _linear(torch, lib, device, x, weight, x_scale, w_scale, bias, activation, residual, types, out_dtype, z_dtype):
    act = _activation(activation)
    xp, ldx, xt = _matrix("x", x, types, device)
    wp, ldw, wt = _matrix("weight", weight, types, device)
    m, k = x.shape
    n = weight.shape[0]
    if wt != xt or weight.shape[1] != k:
        raise ValueError(f"weight must be (features out, {k}) of {x.dtype}, got {tuple(weight.shape)} of {weight.dtype}")
    xs = ws = bp = bt = rp = ldr = rt = zp = zt = nbytes = 0
    if types is _EIGHTS:
        xs, ws = _scales(torch, "x_scale", x_scale, device, m), _scales(torch, "weight_scale", w_scale, device, n)
    if bias is not None:
        bp, bt = _vector("bias", bias, _FLOATS, device, n)
    if residual is not None:
        rp, ldr, rt = _matrix("residual", residual, _FLOATS, device, m, n)
    yt = _float_type("out_dtype", out_dtype)
    y, z, kp = _new(x, (m, n), out_dtype), None, None
    if z_dtype is not None:
        z = _new(x, (m, n), z_dtype)
        zp, zt = z.data_ptr(), _FLOATS[z_dtype]
    nbytes = lib.lf_linear_work_bytes(m, n, k, xt)
    if nbytes:
        work = x.new_empty((nbytes,), dtype=torch.uint8)
        kp = work.data_ptr()
    rc = lib.lf_linear(_LINEAR_ARGS(xp, wp, xs, ws, bp, rp, y.data_ptr(), zp, ldx, ldw, ldr, n, n, m, n, k, xt, bt, rt, yt, zt, act), kp, nbytes, _stream())
    if rc:
        _lib.check(rc)
    return y, z


def linear(x, weight, bias=None, activation=None, residual=None, out_dtype=None, return_preactivation: bool = False):
    """``y = act(x weight^T + bias) + residual`` for x (rows, k) and weight (n, k) of one type; ``activation`` is None, "relu",
    "gelu" (by erf) or "silu".  bias and residual are floating tensors of any type, y is of ``out_dtype`` (default: x's).
    ``return_preactivation=True`` returns ``(y, z)`` with z = x weight^T + bias in x's type, which ``linear_grad`` needs behind an
    activation.  float32 products are as exact as float32 sums of float32 products of values from 2^-110 (8e-34) on; what smaller ones
    have below 2^-126 may be lost.  gelu and silu keep their digits at any z (float32 y: some 20 roundings)."""
    torch, lib, device = _begin()
    out = x.dtype if out_dtype is None else out_dtype
    y, z = _linear(torch, lib, device, x, weight, None, None, bias, activation, residual, _FLOATS, out, x.dtype if return_preactivation else None)
    return (y, z) if return_preactivation else y


def linear_8bit(x, x_scale, weight, weight_scale, bias=None, activation=None, residual=None, out_dtype=None):
    """``linear`` of rows in 8 bits, both ``torch.float8_e4m3fn`` or both ``torch.int8``, each row of x and of weight with its scale
    (``rms_norm_8bit``, ``quantize_rows``).  y is of ``out_dtype`` (default bfloat16).  int8: at most 131071 features in, and exact sums.
    e4m3: the matrix instruction adds its products in groups of eight and cuts them below 2^-13 of the group's largest."""
    torch, lib, device = _begin()
    out = torch.bfloat16 if out_dtype is None else out_dtype
    return _linear(torch, lib, device, x, weight, x_scale, weight_scale, bias, activation, residual, _EIGHTS, out, None)[0]


def linear_grad(dy, x, weight, z=None, activation=None, bias_dtype=None, want_dx: bool = True, want_dweight: bool = True):
    """``(dx, dweight, dbias)`` of ``linear`` from the gradient ``dy`` of y: dz = dy act'(z), dx = dz weight, dweight = dz^T x, dbias =
    column sums of dz.  All of one type but dbias, which is of ``bias_dtype`` (None: not computed).  ``z`` is what
    ``linear(..., return_preactivation=True)`` returned; without an activation it is not needed.  Gradients that are not
    wanted are None.  The residual's gradient is dy.  Behind an activation dz is rounded to the operands' type before the
    products, as they take it."""
    torch, lib, device = _begin()
    act = _activation(activation)
    xp, ldx, xt = _matrix("x", x, _FLOATS, device)
    wp, ldw, wt = _matrix("weight", weight, _FLOATS, device)
    m, k = x.shape
    n = weight.shape[0]
    if wt != xt or weight.shape[1] != k:
        raise ValueError(f"weight must be (features out, {k}) of {x.dtype}, got {tuple(weight.shape)} of {weight.dtype}")
    gp, ldg, gt = _matrix("dy", dy, _FLOATS, device, m, n)
    if gt != xt:
        raise ValueError(f"dy must have x's type {x.dtype}, got {dy.dtype}")
    zp = ldz = dxp = dwp = dbp = bt = 0
    if act != _lib.LF_ACT_NONE:
        if z is None:
            raise ValueError("the gradient of an activation needs z: linear(..., return_preactivation=True)")
        zp, ldz, zt = _matrix("z", z, _FLOATS, device, m, n)
        if zt != xt:
            raise ValueError(f"z must have x's type {x.dtype}, got {z.dtype}")
    dx = dw = db = kp = None
    if want_dx:
        dx = x.new_empty((m, k))
        dxp = dx.data_ptr()
    if want_dweight:
        dw = x.new_empty((n, k))
        dwp = dw.data_ptr()
    if bias_dtype is not None:
        bt = _float_type("bias_dtype", bias_dtype)
        db = _new(x, (n,), bias_dtype)
        dbp = db.data_ptr()
    nbytes = lib.lf_linear_grad_work_bytes(m, n, k, xt, act, want_dx, want_dweight, db is not None)
    if nbytes:
        work = x.new_empty((nbytes,), dtype=torch.uint8)
        kp = work.data_ptr()
    rc = lib.lf_linear_grad(_LINEAR_GRAD_ARGS(gp, zp, xp, wp, dxp, dwp, dbp, ldg, ldz, ldx, ldw, k, k, m, n, k, xt, bt, act), kp, nbytes, _stream())
    if rc:
        _lib.check(rc)
    return dx, dw, db
