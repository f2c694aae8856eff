"""The next-token loss of a language model and its gradient, on the HIP kernels of ``csrc/gdn2_loss.hip``.

``cross_entropy`` reads each row of logits for its loss and, where a gradient will be asked for, writes the gradient in
the same call: the backward pass then only scales it (and leaves it as it is where the loss itself is differentiated).
"""
from __future__ import annotations

import ctypes

import torch
import torch.autograd.forward_ad as fwd
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["cross_entropy"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # GDN2_F32, GDN2_BF16, GDN2_F16
_INDEX = {torch.int32: 1, torch.int64: 2}                                # GDN2_FLAG_INT32, GDN2_FLAG_INT64
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _run(x, targets, how, loss, dlogits, upstream=None, upstream_ld=0):
    """Losses and gradient of rows x (N, V) where they are given; how: (ignore_index, smoothing, z_loss, reduction)."""
    (N, V), dev = x.shape, x.device
    addr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    a = _lib.Gdn2Loss(N, V, _DTYPES[x.dtype], _INDEX[targets.dtype], how[3], upstream_ld, how[1], how[2], V if N == 1 else x.stride(0),
                      how[0], x.data_ptr(), targets.data_ptr(), addr(upstream), addr(loss), addr(dlogits))
    L = _lib.lib()
    ws = torch.empty(L.gdn2_loss_workspace_bytes(N), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(L.gdn2_cross_entropy(ctypes.byref(a), _lib.ptr(ws), _lib.stream_handle(dev)), "gdn2_cross_entropy")


def _saved(t, like):
    """A saved tensor as it was saved: the kernels take its address, and hooks may have changed its strides, type or device."""
    rows = t.is_contiguous() or (t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1])
    return t if rows and (t.shape, t.dtype, t.device) == like else _lib.restored(t, *like)


class _CrossEntropy(torch.autograd.Function):
    """(rows of logits, targets) -> loss.  Once differentiable: a second derivative raises."""

    @staticmethod
    def forward(ctx, x, targets, how):
        loss = torch.empty(x.shape[0] if how[3] == 0 else (), dtype=torch.float32, device=x.device)
        # float16 gradients are formed when the factor of a scaled loss is known: without it they would underflow
        d = torch.empty(x.shape, dtype=x.dtype, device=x.device) if x.dtype != torch.float16 and ctx.needs_input_grad[0] else None
        _run(x, targets, how, loss, d)
        ctx.how, ctx.grad, ctx.likes = how, d, [(t.shape, t.dtype, t.device) for t in (x, targets)]
        ctx.save_for_backward(x, targets)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, targets = (_saved(t, like) for t, like in zip(ctx.saved_tensors, ctx.likes))
        g = g.contiguous()
        ld = 1 if ctx.how[3] == 0 else 0
        d = ctx.grad
        if d is not None:
            # (multiplied where it lies: a graph of the backward pass alone would do so at every replay)
            with torch.cuda.device(x.device):
                captured = torch.cuda.is_current_stream_capturing()
            d, ctx.grad = (None, d) if captured else (d, None)
        if d is None:           # float16, a second pass over a kept graph, or a captured one
            d = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            _run(x, targets, ctx.how, None, d, g, ld)
            return d, None, None
        with torch.cuda.device(x.device):
            _lib.check(_lib.lib().gdn2_scale_rows(_lib.ptr(d), _DTYPES[x.dtype], *x.shape, _lib.ptr(g), ld,
                                                  _lib.stream_handle(x.device)), "gdn2_scale_rows")
        return d, None, None


def cross_entropy(logits, targets, ignore_index: int = -100, label_smoothing: float = 0.0, z_loss: float = 0.0,
                  reduction: str = "mean"):
    """Cross-entropy of logits (..., V) with targets (...), whole numbers: float32.

    Of a row x with target t: lse - (1 - label_smoothing) x[t] - label_smoothing mean(x) + z_loss lse^2, with
    lse = log sum exp x.  Rows with t = ignore_index have no loss and no gradient.  reduction: "mean" over the others
    (0 where there are none), "sum", or "none" (...,).  logits float32, bfloat16 or float16, rows of any stride;
    statistics are float32, the sum over the rows 64 bits, the gradient has the logits' dtype (scaled by what the loss
    is multiplied with before it is rounded in float16, after it in the others).  A target outside 0 .. V-1 makes its
    row's loss and gradient NaN (the host does not wait to look at them).  -inf is a banned token.  Once
    differentiable."""
    how = _REDUCTIONS.get(reduction)
    if (isinstance(logits, torch.Tensor) and logits.is_cuda and how is not None and type(label_smoothing) is float and 0.0 <= label_smoothing <= 1.0
            and type(z_loss) is float and z_loss >= 0.0):
        # plain calls (csrc/bind.cpp) go native; None = not one, and what follows handles it
        loss = _lib.bind().cross_entropy(logits, targets, ignore_index, label_smoothing, z_loss, how)
        if loss is not None:
            return loss
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise TypeError(f"targets must be whole numbers, got {targets.dtype}")
    if logits.dim() < 1 or logits.numel() == 0 or tuple(targets.shape) != tuple(logits.shape[:-1]):
        raise ValueError(f"logits must be (..., V), not empty, and targets (...), got {tuple(logits.shape)} and {tuple(targets.shape)}")
    if max(targets.numel(), logits.shape[-1]) > 2 ** 30:
        raise ValueError(f"{targets.numel()} rows of {logits.shape[-1]}: up to 2^30 each are supported")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(map(repr, _REDUCTIONS))}, got {reduction!r}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing={label_smoothing}: between 0 and 1")
    if not z_loss >= 0.0:
        raise ValueError(f"z_loss={z_loss}: not negative")
    if targets.device != logits.device:
        raise ValueError(f"targets are on {targets.device}, logits on {logits.device}")
    if not logits.is_cuda:
        raise ValueError(f"cross_entropy needs tensors on a ROCm device, got {logits.device}")
    V = logits.shape[-1]
    x = logits.reshape(-1, V)
    if (x.stride(1) != 1 and V > 1) or (x.stride(0) < V and x.shape[0] > 1):
        x = x.clone(memory_format=torch.contiguous_format)
    t = targets.reshape(-1)
    t = t.contiguous() if t.dtype in _INDEX else t.to(torch.int64)
    how = (int(ignore_index), float(label_smoothing), float(z_loss), how)
    if (torch.is_grad_enabled() and x.requires_grad) or (fwd._current_level >= 0 and fwd.unpack_dual(x).tangent is not None):
        loss = _CrossEntropy.apply(x, t, how)
    else:
        loss = torch.empty(x.shape[0] if reduction == "none" else (), dtype=torch.float32, device=x.device)
        _run(x, t, how, loss, None)
    return loss.view(targets.shape) if reduction == "none" else loss
