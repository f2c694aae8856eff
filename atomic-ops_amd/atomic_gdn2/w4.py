"""Matrix products with 4-bit weights for serving, on the HIP kernels of ``csrc/gdn2_w4.hip``.

A matrix W (in, out), as ``e2e_lm.Dense`` holds it, is kept as whole codes q of 0 .. 15 with a scale
and a zero for each column and group of ``group_size`` (32, 64 or 128) rows:

    W[k, n] = scale[g, n] (q[k, n] - zero[g, n]),  g = k // group_size.

``quantize_w4`` forms them from a matrix, ``pack_w4`` takes codes that a program has, and both lay them
out once, when a model is loaded, in the order in which the kernels read them (``W4Weight``).
``w4_linear`` multiplies: float32, bfloat16 or float16 rows, one (a token) or thousands (a prompt).
Codes enter the products as they are and sums are float32, so a result differs from the definition's
by float32 rounding (of entries below 1e-33 of a float32 row, by their bits below 2^-133) and one
rounding to its own type.  For inference: no gradients, and asking for one
raises.
"""
from __future__ import annotations

import ctypes
import operator

import torch
import torch.autograd.forward_ad as fwd

from . import _lib

__all__ = ["W4Weight", "pack_w4", "quantize_w4", "w4_linear"]

GROUP_SIZES = (32, 64, 128)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # GDN2_F32, GDN2_BF16, GDN2_F16
_KB, _NB = 128, 16          # rows and columns of a block of the layout
_NIBBLE = (0, 2, 4, 6, 1, 3, 5, 7)


def _int(x):
    """x as an int where it is a whole number of another type."""
    return operator.index(x) if hasattr(x, "__index__") else x


class _Inference(torch.autograd.Function):
    """fn(*ts) as a node whose gradients raise.  (It has no forward mode either: a tangent raises.)"""

    @staticmethod
    def forward(ctx, name, fn, *ts):
        ctx.name = name
        return fn(*ts)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} is for inference and has no gradients: call it under torch.no_grad(), or detach its inputs")


def for_inference(name, fn, *ts):
    """fn(*ts) where a gradient or tangent of one of ts is not to be lost in silence, else None."""
    if (torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in ts)) \
            or fwd._current_level >= 0 and any(
                isinstance(t, torch.Tensor) and fwd.unpack_dual(t).tangent is not None for t in ts):
        return _Inference.apply(name, fn, *ts)
    return None


class W4Weight:
    """A matrix (in_features, out_features) of 4-bit codes with group scales, laid out for the kernels
    (include/gdn2.h, ``gdn2_w4``): q (out / 16, in / 128, 64, 4) and meta (out / 16, in / group_size, 16),
    int32, sizes rounded up to whole blocks of 128 rows and 16 columns."""
    __slots__ = ("q", "meta", "in_features", "out_features", "group_size")

    def __init__(self, q, meta, in_features, out_features, group_size):
        self.q, self.meta = q, meta
        self.in_features, self.out_features, self.group_size = _int(in_features), _int(out_features), _int(group_size)
        self._check()

    def _check(self):
        """Raise unless q and meta are what the sizes say: the kernels read by the sizes."""
        _check_group(self.group_size)
        for n in ("in_features", "out_features"):
            if type(getattr(self, n)) is not int or getattr(self, n) < 1:
                raise ValueError(f"{n} must be a positive int, got {getattr(self, n)!r}")
        nkb, nnb = -(-self.in_features // _KB), -(-self.out_features // _NB)
        for t, n, shape in ((self.q, "q", (nnb, nkb, 64, 4)), (self.meta, "meta", (nnb, nkb * _KB // self.group_size, _NB))):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
                raise TypeError(f"{n} must be an int32 tensor, got {getattr(t, 'dtype', type(t).__name__)}")
            if tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{n} must be contiguous {shape} for a weight of {self.in_features} x {self.out_features} in "
                                 f"groups of {self.group_size}, got {tuple(t.shape)}")
        if self.q.device != self.meta.device:
            raise ValueError(f"meta is on {self.meta.device}, q on {self.q.device}")

    @property
    def shape(self):
        return (self.in_features, self.out_features)

    @property
    def device(self):
        return self.q.device

    @property
    def nbytes(self):
        return 4 * (self.q.numel() + self.meta.numel())

    def to(self, device):
        return W4Weight(self.q.to(device), self.meta.to(device), self.in_features, self.out_features, self.group_size)

    def unpack(self):
        """(codes uint8 (in, out), scales bfloat16 (groups, out), zeros bfloat16 (groups, out))."""
        nnb, nkb = self.q.shape[:2]
        w = self.q.reshape(nnb, nkb, 4, 16, 4)                                       # c, r, j
        e = torch.stack([(w >> (4 * p)) & 15 for p in _NIBBLE], dim=-1).to(torch.uint8)
        codes = e.permute(1, 4, 2, 5, 0, 3).reshape(nkb * _KB, nnb * _NB)            # k = (nkb, j, c, e), n = (nnb, r)
        per = lambda bits: bits.to(torch.int16).view(torch.bfloat16).permute(1, 0, 2).reshape(-1, nnb * _NB)  # noqa: E731
        groups = -(-self.in_features // self.group_size)
        low = ((self.meta & 0xffff) ^ 0x8000) - 0x8000                               # (sign extended: fits an int16)
        return (codes[:self.in_features, :self.out_features].contiguous(),
                per(low)[:groups, :self.out_features].contiguous(),
                per(self.meta >> 16)[:groups, :self.out_features].contiguous())

    def dequantize(self):
        """The matrix in float32."""
        codes, scales, zeros = self.unpack()
        spread = lambda t: t.float().repeat_interleave(self.group_size, 0)[:self.in_features]  # noqa: E731
        return (codes.float() - spread(zeros)) * spread(scales)


def _check_group(group_size):
    if type(group_size) is not int or group_size not in GROUP_SIZES:
        raise ValueError(f"group_size={group_size}: the kernels support groups of {', '.join(map(str, GROUP_SIZES))} rows")
    return group_size


def pack_w4(codes, scales, zeros=None, group_size: int = 128) -> W4Weight:
    """The matrix of given codes as the kernels read it.

    codes (in, out): whole numbers 0 .. 15; scales (groups, out), groups = ceil(in / group_size), kept
    as bfloat16; zeros (groups, out), kept as bfloat16, or None: 8 everywhere."""
    group_size = _check_group(_int(group_size))
    if codes.dim() != 2 or codes.numel() == 0:
        raise ValueError(f"codes must be (in, out), got {tuple(codes.shape)}")
    if codes.is_floating_point() or codes.is_complex() or codes.dtype == torch.bool:
        raise TypeError(f"codes must be whole numbers, got {codes.dtype}")
    K, N = codes.shape
    groups = -(-K // group_size)
    for t, name in ((scales, "scales"), (zeros, "zeros")):
        if t is not None and tuple(t.shape) != (groups, N):
            raise ValueError(f"{name} must be (groups, out) = {(groups, N)}, got {tuple(t.shape)}")
        if t is not None and t.device != codes.device:
            raise ValueError(f"{name} is on {t.device}, codes on {codes.device}")
    lo, hi = (int(v) for v in torch.aminmax(codes))
    if lo < 0 or hi > 15:
        raise ValueError(f"codes must lie in 0 .. 15, got {lo} .. {hi}")
    dev, nkb, nnb = codes.device, -(-K // _KB), -(-N // _NB)
    full = torch.zeros((nkb * _KB, nnb * _NB), dtype=torch.uint8, device=dev)
    full[:K, :N] = codes
    e = full.view(nkb, 4, 4, 8, nnb, 16).permute(4, 0, 2, 5, 1, 3)                   # nnb, nkb, c, r, j, e
    q = torch.zeros(e.shape[:-1], dtype=torch.int32, device=dev)
    for i, p in enumerate(_NIBBLE):
        q |= e[..., i].to(torch.int32) << (4 * p)
    bits = lambda t: t.to(torch.bfloat16).view(torch.int16).to(torch.int32)  # noqa: E731
    zeros = torch.full_like(scales, 8) if zeros is None else zeros
    word = (bits(scales) & 0xffff) | (bits(zeros) << 16)
    meta = torch.zeros((nkb * _KB // group_size, nnb * _NB), dtype=torch.int32, device=dev)
    meta[:groups, :N] = word
    meta = meta.view(-1, nnb, _NB).permute(1, 0, 2).contiguous()
    return W4Weight(q.reshape(nnb, nkb, 64, 4), meta, K, N, group_size)


def quantize_w4(weight, group_size: int = 128, symmetric: bool = False) -> W4Weight:
    """The matrix ``weight`` (in, out) rounded to 4-bit codes, each to the nearest of its group's grid:
    16 levels from the group's least to its largest entry (and 0, which stays exactly 0), or with
    ``symmetric`` 15 levels around 0 and no zeros to choose."""
    group_size = _check_group(_int(group_size))
    if weight.dim() != 2 or weight.numel() == 0 or not weight.is_floating_point():
        raise ValueError(f"weight must be a floating-point (in, out) matrix, got {weight.dtype} {tuple(weight.shape)}")
    K, N = weight.shape
    groups = -(-K // group_size)
    w = torch.zeros((groups * group_size, N), dtype=torch.float32, device=weight.device)
    w[:K] = weight.detach()
    if not bool(torch.isfinite(w).all()):
        raise ValueError("weight must be finite in float32")
    w = w.view(groups, group_size, N)
    if symmetric:
        scales, zeros = w.abs().amax(1) / 7, None
    else:
        lo, hi = w.amin(1).clamp(max=0), w.amax(1).clamp(min=0)
        scales = (hi - lo) / 15
        scales = torch.where(torch.isinf(scales), hi / 15 - lo / 15, scales)         # (hi - lo above float32)
    # codes are chosen for the scale as it is kept; a group of zeros, or below bfloat16's least scale, has any
    scales = scales.to(torch.bfloat16)
    scales = torch.where(scales > 0, scales, torch.ones_like(scales))
    s = scales.float()
    if symmetric:
        offset = torch.full_like(s, 8.0)
    else:
        zeros = offset = torch.round(-lo / s).clamp(0, 15)
    codes = (torch.round(w / s[:, None]) + offset[:, None]).clamp(0, 15).to(torch.uint8)
    return pack_w4(codes.view(-1, N)[:K], scales, zeros, group_size)


def _rows(t, K):
    """t (..., K) as rows with a stride of at least K, without a copy where its layout allows one."""
    r = t.reshape(-1, K)
    plain = (r.stride(1) == 1 or K == 1) and (r.stride(0) >= K or r.shape[0] == 1)
    return r if plain else r.clone(memory_format=torch.contiguous_format)


def w4_linear(x, weight: W4Weight, bias=None, residual=None):
    """y = x W (+ bias) (+ residual): x (..., in) float32, bfloat16 or float16, y (..., out) in x's dtype.

    bias (out,) and residual (..., out) are cast to x's dtype.  Rows may be strided (a slice of wider
    rows); sums are float32 (16 K max |x| has to fit).  A row of x that holds an infinity or NaN gives
    nothing finite, and touches no other row."""
    if type(weight) is W4Weight and isinstance(x, torch.Tensor) and x.is_cuda:
        # plain calls (csrc/bind.cpp) go native; None = not one, and what follows handles it
        y = _lib.bind().w4(x, weight.q, weight.meta, weight.in_features, weight.out_features, weight.group_size, bias, residual)
        if y is not None:
            return y
    y = for_inference("w4_linear", lambda *ts: w4_linear(ts[0], weight, *ts[1:]), x, bias, residual)
    if y is not None:
        return y
    if not isinstance(weight, W4Weight):
        raise TypeError(f"weight must be a W4Weight (pack_w4, quantize_w4), got {type(weight).__name__}")
    weight._check()
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    K, N = weight.shape
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x must be (..., {K}), got {tuple(x.shape)}")
    if x.numel() // K >= 2 ** 31:
        raise ValueError(f"x has {x.numel() // K} rows: fewer than 2^31 are supported")
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"bias must be ({N},), got {tuple(bias.shape)}")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], N):
        raise ValueError(f"residual must be {(*x.shape[:-1], N)}, got {tuple(residual.shape)}")
    dev = x.device
    for t, n in ((weight, "weight"), (bias, "bias"), (residual, "residual")):
        if t is not None and t.device != dev:
            raise ValueError(f"{n} is on {t.device}, x on {dev}")
    if not x.is_cuda:
        raise ValueError(f"w4_linear needs tensors on a ROCm device, got {dev}")
    y = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=dev)
    if x.numel() == 0:
        return y
    x = _rows(x, K)
    bias = None if bias is None else bias.to(x.dtype).contiguous()
    residual = None if residual is None else _rows(residual.to(x.dtype), N)
    M = x.shape[0]
    a = _lib.Gdn2W4(M, K, N, weight.group_size, _DTYPES[x.dtype], K if M == 1 else x.stride(0),
                    0 if residual is None else N if M == 1 else residual.stride(0), x.data_ptr(), weight.q.data_ptr(),
                    weight.meta.data_ptr(), None if bias is None else bias.data_ptr(),
                    None if residual is None else residual.data_ptr(), y.data_ptr())
    ws = torch.empty(_lib.lib().gdn2_w4_workspace_bytes(ctypes.byref(a)), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().gdn2_w4_linear(ctypes.byref(a), _lib.ptr(ws), _lib.stream_handle(dev)), "gdn2_w4_linear")
    return y
