"""Matrix products of a layer, forward and backward, on the HIP kernels of ``csrc/gdn2_linear.hip``.

``linear`` computes y = act(x W + bias) + residual in one pass behind the product: float32, bfloat16 or float16 rows,
one (a token) or thousands (a batch).  W is (in, out), as ``e2e_lm.Dense`` holds it, or a transposed view of an
(out, in) matrix (a tied embedding), read as it lies.  Sums are float32 and y is rounded once.  float32 operands of
larger products enter as three bfloat16 pieces each (entries below 1e-33 lose their bits below 2^-133): what the six
products of pieces leave out is below 2^-21 of |x| |W|, towards zero, at the rate of the 16-bit matrix cores.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .w4 import _rows

__all__ = ["linear"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # GDN2_F32, GDN2_BF16, GDN2_F16
_ACTS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}                  # GDN2_ACT_*
_XW, _XWT, _XTW = 0, 1, 2
_HALVES, _Z_F32, _DZ_LOW = 4, 16, 32                                     # GDN2_*
_FINE, _FINE_X, _FINE_Z = 2 ** 30, 2 ** 21, 2 ** 21                      # GDN2_LINEAR_FINE, _X, _Z


def _addr(t):
    return None if t is None else t.data_ptr()


def _turned(w):
    """Whether w is the transposed view of a matrix with whole rows."""
    return w.stride(0) == 1 and w.stride(1) >= w.shape[0] and not (w.stride(1) == 1 and w.shape[1] > 1)


def _ld(t):
    return t.shape[1] if t.shape[0] == 1 else t.stride(0)


def _product(form, a, b, M, K, N, out, bias=None, residual=None, act=0, z=None):
    """out (M, N) = act(A B + bias) + residual; a, b rows of whole elements (include/gdn2.h, gdn2_product)."""
    if z is not None and z.dtype == torch.float32:
        act |= _Z_F32
    p = _lib.Gdn2Product(M, K, N, form, _DTYPES[a.dtype], _DTYPES[out.dtype], 0 if bias is None else _DTYPES[bias.dtype], act,
                         _ld(a), _ld(b), 0 if residual is None else _ld(residual), a.data_ptr(), b.data_ptr(), _addr(bias),
                         _addr(residual), out.data_ptr(), _addr(z))
    L = _lib.lib()
    with torch.cuda.device(out.device):         # (its CUs say how a product is split)
        ws = torch.empty(L.gdn2_linear_workspace_bytes(ctypes.byref(p)), dtype=torch.uint8, device=out.device)
        _lib.check(L.gdn2_linear(ctypes.byref(p), _lib.ptr(ws), _lib.stream_handle(out.device)), "gdn2_linear")
    return out


def _fine(M, K, N, dtype):
    """Whether the gradients of a product of 16 bits are formed from dz and what its rounding leaves out.  Rounded alone, dz makes
    their error 1.42 times that of rounding them, in products of 32 to 100 rows or columns up to twice.  (With silu, us on the GPU,
    rounded and both: 1 x 5412 x 127 27, 32; 2 x 1793 x 4407 66, 82; 300 x 677 x 811 51, 63; 2048 x 768 x 512 39, 57.
    x is copied for it, so that a long one is left out: 16384 x 4096 x 1 118, 547.)"""
    return dtype != torch.float32 and 2 * M * K * N <= _FINE and M * K <= _FINE_X


def _z_dtype(M, K, N, dtype):
    """What z is kept in: rounded to 16 bits it makes that 1.46 times.  (Two bytes more a result.)"""
    return torch.float32 if _fine(M, K, N, dtype) or M * N <= _FINE_Z else dtype


def _forward(x, weight, bias, residual, act, out_dtype, keep):
    """y, and z = x W + bias where keep; x (M, K), residual (M, N) rows."""
    M, (K, N) = x.shape[0], weight.shape
    y = torch.empty((M, N), dtype=out_dtype, device=x.device)
    z = torch.empty((M, N), dtype=_z_dtype(M, K, N, x.dtype), device=x.device) if keep else None
    if M:
        turned = _turned(weight)
        _product(_XWT if turned else _XW, x, weight.t() if turned else weight, M, K, N, y, bias, residual, act, z)
    return y, z


def _slope(dy, z, dtype, act, bias_dtype, need_dz, fine=False):
    """dz = dy act'(z) (None: dy itself; fine: 2 M rows, the second M what rounding leaves out) and the bias' gradient (None: not
    asked for)."""
    M, N = dy.shape
    dz = torch.empty((2 * M if fine else M, N), dtype=dtype, device=dy.device) if need_dz else None
    act |= (_Z_F32 if z is not None and z.dtype == torch.float32 else 0) | (_DZ_LOW if fine and need_dz else 0)
    db = None if bias_dtype is None else torch.empty(N, dtype=bias_dtype, device=dy.device)
    p = _lib.Gdn2Slope(M, N, _DTYPES[dtype], _DTYPES[dy.dtype], 0 if db is None else _DTYPES[bias_dtype], act, dy.data_ptr(), _addr(z),
                       _addr(dz), _addr(db))
    L = _lib.lib()
    with torch.cuda.device(dy.device):
        ws = torch.empty(L.gdn2_linear_slope_workspace_bytes(ctypes.byref(p)), dtype=torch.uint8, device=dy.device)
        _lib.check(L.gdn2_linear_slope(ctypes.byref(p), _lib.ptr(ws), _lib.stream_handle(dy.device)), "gdn2_linear_slope")
    return dz, db


def _saved(ctx):
    """x of whole rows, the weight of whole rows or turned, z as one array; hooks may have changed strides, types or devices."""
    x, weight, z = (t if t is None or (t.shape, t.dtype, t.device) == like else _lib.restored(t, *like)
                    for t, like in zip(ctx.saved_tensors, ctx.likes))
    return _rows(x, x.shape[1]), weight if _turned(weight) else _rows(weight, weight.shape[1]), None if z is None else z.contiguous()


class _Linear(torch.autograd.Function):
    """(x rows, weight, bias, residual rows) -> y rows.  Once differentiable: a second derivative raises."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_dtype):
        y, z = _forward(x, weight, bias, residual, act, out_dtype, act != 0)
        ctx.act, ctx.bias_dtype = act, None if bias is None else bias.dtype
        ctx.save_for_backward(x, weight, z)
        ctx.likes = [None if t is None else (t.shape, t.dtype, t.device) for t in (x, weight, z)]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = _saved(ctx)
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        (M, K), N, dev = x.shape, weight.shape[1], x.device
        if M == 0:
            return (torch.zeros_like(x) if need_x else None, torch.zeros_like(weight) if need_w else None,
                    torch.zeros(N, dtype=ctx.bias_dtype, device=dev) if need_b else None, dy if need_r else None, None, None)
        dres, dy = dy if need_r else None, dy.contiguous()
        own = (ctx.act != 0 or dy.dtype != x.dtype) and (need_x or need_w)
        fine = own and _fine(M, K, N, x.dtype)
        dz, db = dy, None
        if own or need_b:
            dz, db = _slope(dy, z, x.dtype, ctx.act, ctx.bias_dtype if need_b else None, own, fine)
            dz = dy if dz is None else dz
        turned, dx, dw = _turned(weight), None, None
        if need_x:
            dx = _product((_XW if turned else _XWT) | (_HALVES if fine else 0), dz, weight.t() if turned else weight, M, N, K,
                          torch.empty((M, K), dtype=x.dtype, device=dev))
        if need_w and fine:             # (x^T dz is a sum over the rows: over those of both)
            x, M = torch.cat((x, x)), 2 * M
        if need_w and turned:
            dw = _product(_XTW, dz, x, N, M, K, torch.empty((N, K), dtype=x.dtype, device=dev)).t()
        elif need_w:
            dw = _product(_XTW, x, dz, K, M, N, torch.empty((K, N), dtype=x.dtype, device=dev))
        return dx, dw, db, dres, None, None


def linear(x, weight, bias=None, residual=None, activation=None, out_dtype=None):
    """y = act(x W + bias) + residual: x (..., in), weight (in, out), y (..., out).

    x and weight share a dtype: float32, bfloat16 or float16.  y has out_dtype, theirs (default) or float32 (a
    float32 residual stream over 16-bit products).  bias (out,): their dtype or float32; residual (..., out) is cast
    to out_dtype.  activation: None, "silu", "gelu" (z Phi(z)) or "gelu_tanh".  x and residual may be rows of wider
    matrices.  Gradients of all four, each summed in float32 and in its tensor's dtype; with an activation
    z = x W + bias is kept for them in x's dtype, and the gradient of z has x's dtype; a product of up to 2^30
    operations over an x of up to 2^21 elements keeps z in float32 and rounds no gradient on its way, and results of up to
    2^21 elements keep z in float32.  Once differentiable.  A row
    of x with an infinity or NaN gives nothing finite in float32 (an infinity may come out as NaN: larger float32 products
    take it in pieces), and touches no other row."""
    if activation in _ACTS and isinstance(x, torch.Tensor) and x.is_cuda and out_dtype in (None, x.dtype, torch.float32):
        # plain calls (csrc/bind.cpp) go native; None = not one, and what follows handles it
        y = _lib.bind().linear(x, weight, bias, residual, _ACTS[activation], out_dtype is torch.float32)
        if y is not None:
            return y
    if activation not in _ACTS:
        raise ValueError(f"activation must be one of {', '.join(map(repr, _ACTS))}, got {activation!r}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if weight.dtype != x.dtype:
        raise TypeError(f"weight must be {x.dtype} as x, got {weight.dtype}")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in (x.dtype, torch.float32):
        raise TypeError(f"out_dtype must be {x.dtype} or float32, got {out_dtype}")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be (in, out), got {tuple(weight.shape)}")
    K, N = weight.shape
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x must be (..., {K}), got {tuple(x.shape)}")
    if max(x.numel() // K, K, N) > 2 ** 27:
        raise ValueError(f"a product of {x.numel() // K} x {K} x {N}: up to 2^27 each are supported")
    shape = (*x.shape[:-1], N)
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"bias must be ({N},), got {tuple(bias.shape)}")
    if bias is not None and bias.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"bias must be {x.dtype} or float32, got {bias.dtype}")
    if residual is not None and tuple(residual.shape) != shape:
        raise ValueError(f"residual must be {shape}, got {tuple(residual.shape)}")
    dev = x.device
    for t, n in ((weight, "weight"), (bias, "bias"), (residual, "residual")):
        if t is not None and t.device != dev:
            raise ValueError(f"{n} is on {t.device}, x on {dev}")
    if not x.is_cuda:
        raise ValueError(f"linear needs tensors on a ROCm device, got {dev}")
    x = _rows(x, K)
    weight = weight if _turned(weight) else _rows(weight, N)
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else _rows(residual.to(out_dtype), N)
    return _Linear.apply(x, weight, bias, residual, _ACTS[activation], out_dtype).view(shape)
