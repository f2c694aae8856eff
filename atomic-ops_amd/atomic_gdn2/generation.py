"""Token generation from the benchmark LM: the steps of beam search on the HIP kernels.

* ``beam_step``    of all continuations of a group's beams, the best n (``csrc/gdn2_beam.hip``);
* ``premix_step``  one token of a block's convolutions, gates and norms from the cached projections of
                   the three tokens before it (``csrc/gdn2_lm.hip``).

A beam that is kept continues the sequence of its parent, so its caches are its parent's.  Both caches
of a block are taken from the parent's row where a step reads them anyway (``parents`` here and in
``inference.decode_step``): nothing is copied to reorder them.  For inference: no gradients.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib

__all__ = ["BeamStep", "PremixStep", "beam_step", "premix_step"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # GDN2_F32, GDN2_BF16, GDN2_F16
_INDEX = {torch.int32: 1, torch.int64: 2}                                # GDN2_FLAG_INT32, GDN2_FLAG_INT64


class BeamStep(NamedTuple):
    """The kept continuations of each group, the best first, all (B, n): the new tokens (int64), the
    rows b K + k of the beams that they continue (int64: ``parents`` of the next steps), their scores
    (float32), and whether they are finished (None without an end token)."""
    tokens: torch.Tensor
    rows: torch.Tensor
    scores: torch.Tensor
    finished: Optional[torch.Tensor]


class PremixStep(NamedTuple):
    """What the recurrence takes for one token, q, k, v, w, b, g (R, H, D); the output gate's logits
    (R, H D); the history of the next token (R, 3, 3 H D)."""
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    w: torch.Tensor
    b: torch.Tensor
    g: torch.Tensor
    gate: torch.Tensor
    history: torch.Tensor


def _on(dev, **ts):
    for n, t in ts.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{n} is on {t.device}, expected {dev}")


def beam_step(logits, scores, n: Optional[int] = None, finished=None, eos_id: Optional[int] = None) -> BeamStep:
    """The n best continuations (default K) of each group of K beams over the vocabulary.

    logits (B K, V) or (B, K, V), float32, bfloat16 or float16, rows of any stride; scores (B, K): the
    beams' log-probabilities so far.  A continuation's score is scores[b, k] +
    log_softmax(logits[b, k])[v] in float32; equal scores go to the lower k V + v.  NaN counts as -inf
    (a banned token, a beam that is not in use), and with fewer than n continuations above -inf the
    lowest of the others follow, at -inf.  finished (B, K) bool, with eos_id: a finished beam has one
    continuation, eos_id at its own score; a beam that takes eos_id is finished.  Each group's
    result does not depend on the others, and equal inputs give equal bits."""
    if isinstance(logits, torch.Tensor) and logits.is_cuda and (finished is None or eos_id is not None) \
            and (eos_id is None or type(eos_id) is int and eos_id >= 0) and (n is None or type(n) is int):
        # plain calls (csrc/bind.cpp) go native; None = not one, and what follows handles it
        out = _lib.bind().beam(logits, scores, scores.shape[-1] if n is None else n, finished, -1 if eos_id is None else eos_id)
        if out is not None:
            return BeamStep(*out, None) if eos_id is None else BeamStep(*out)
    if scores.dim() != 2 or scores.numel() == 0:
        raise ValueError(f"scores must be (B, K), got {tuple(scores.shape)}")
    B, K = scores.shape
    if logits.dim() not in (2, 3) or tuple(logits.shape[:-1]) not in ((B * K,), (B, K)) or logits.shape[-1] == 0:
        raise ValueError(f"logits must be {(B * K, 'V')} or {(B, K, 'V')}, got {tuple(logits.shape)}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    V = logits.shape[-1]
    n = K if n is None else int(n)
    if not 1 <= n <= min(128, K * V):
        raise ValueError(f"n={n}: between 1 and min(128, K V) = {min(128, K * V)} continuations can be kept")
    if finished is not None and eos_id is None:
        raise ValueError("finished beams need an eos_id")
    if eos_id is not None and not 0 <= eos_id < V:
        raise ValueError(f"eos_id={eos_id} lies outside the vocabulary of {V}")
    if finished is not None and tuple(finished.shape) != (B, K):
        raise ValueError(f"finished must be {(B, K)}, got {tuple(finished.shape)}")
    dev = logits.device
    _on(dev, scores=scores, finished=finished)
    if not logits.is_cuda:
        raise ValueError(f"beam_step needs tensors on a ROCm device, got {dev}")
    rows = logits.reshape(B * K, V)
    if (rows.stride(1) != 1 and V > 1) or (rows.stride(0) < V and B * K > 1):
        rows = rows.clone(memory_format=torch.contiguous_format)
    scores = scores.to(torch.float32).contiguous()
    done = None if finished is None else (finished != 0).contiguous()
    out = [torch.empty((B, n), dtype=dt, device=dev) for dt in (torch.int64, torch.int64, torch.float32)]
    new = None if eos_id is None else torch.empty((B, n), dtype=torch.bool, device=dev)
    L_ = _lib.lib()
    a = _lib.Gdn2Beam(B, K, V, n, -1 if eos_id is None else int(eos_id), _DTYPES[logits.dtype],
                      V if B * K == 1 else rows.stride(0), rows.data_ptr(), scores.data_ptr(),
                      None if done is None else done.data_ptr(), *(t.data_ptr() for t in out),
                      None if new is None else new.data_ptr())
    ws = torch.empty(L_.gdn2_beam_workspace_bytes(B, K, V, n), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(L_.gdn2_beam_step(ctypes.byref(a), _lib.ptr(ws), _lib.stream_handle(dev)), "gdn2_beam_step")
    return BeamStep(*out, new)


def premix_step(y, history, conv_w, conv_b, gate_b, decay_b, decay_a, n_heads: int, g_max: float,
                parents=None) -> PremixStep:
    """One token of a block between its input projections and the recurrence.

    y (R, >= 6 C + H), C = H D: the token's projections [q | k | v | erase | write | output gate |
    decay], rows of any stride; history (S, 3, 3 C): the q | k | v projections of the three tokens
    before, oldest first (zeros before the first token).  conv_w three (C, 4) and conv_b three (C,):
    the convolutions' taps and biases for q, k, v; gate_b two (C,): the erase and write gates' biases;
    decay_b, decay_a (H,).  parents (R,) int32 or int64: the history row that each row continues (one
    outside 0 .. S-1 has none: zeros); None: its own.  All float32 but parents."""
    if isinstance(y, torch.Tensor) and y.is_cuda and type(n_heads) is int and type(g_max) is float:
        out = _lib.bind().premix_step(y, history, (*conv_w, *conv_b, *gate_b, decay_b, decay_a), n_heads, g_max, parents)
        if out is not None:
            return PremixStep(*out)
    H = int(n_heads)
    if y.dim() != 2 or history.dim() != 3 or H < 1 or history.shape[1] != 3 or history.shape[2] % (3 * H) or history.shape[2] == 0:
        raise ValueError(f"y must be (R, columns) and history (S, 3, 3 H D), got {tuple(y.shape)} and {tuple(history.shape)}")
    R, S, C = y.shape[0], history.shape[0], history.shape[2] // 3
    D = C // H
    if D not in (64, 128):
        raise ValueError(f"D={D}: the HIP kernels support head dimensions 64 and 128")
    if y.shape[1] < 6 * C + H:
        raise ValueError(f"y has {y.shape[1]} columns, 6 H D + H = {6 * C + H} are needed")
    if R == 0 or S == 0:
        raise ValueError("empty input")
    ps = {f"conv_w[{i}]": (t, (C, 4)) for i, t in enumerate(conv_w)}
    ps.update({f"conv_b[{i}]": (t, (C,)) for i, t in enumerate(conv_b)})
    ps.update({f"gate_b[{i}]": (t, (C,)) for i, t in enumerate(gate_b)})
    ps.update(decay_b=(decay_b, (H,)), decay_a=(decay_a, (H,)))
    if len(ps) != 10:
        raise ValueError("three convolutions (taps and biases) and two gates are needed")
    for n, (t, shape) in ps.items():
        if tuple(t.shape) != shape:
            raise ValueError(f"{n} must be {shape}, got {tuple(t.shape)}")
    dev = y.device
    _on(dev, history=history, parents=parents, **{n: t for n, (t, _) in ps.items()})
    for n, t in dict(y=y, history=history, **{n: t for n, (t, _) in ps.items()}).items():
        if t.dtype != torch.float32:
            raise TypeError(f"{n} must be float32, got {t.dtype}")
    if parents is None and S != R:
        raise ValueError(f"without parents, history must have a row for each of the {R} rows of y, got {S}")
    parents = _parent_rows(parents, R)
    if not y.is_cuda:
        raise ValueError(f"premix_step needs tensors on a ROCm device, got {dev}")
    if y.stride(1) != 1 or (y.stride(0) < 6 * C + H and R > 1):
        y = y.clone(memory_format=torch.contiguous_format)
    history = history.contiguous()
    cw, cb, gb = ([t.contiguous() for t in ts] for ts in (conv_w, conv_b, gate_b))
    cw = [t if t.data_ptr() % 16 == 0 else t.clone() for t in cw]
    decay_b, decay_a = decay_b.contiguous(), decay_a.contiguous()
    outs = [torch.empty((R, H, D), dtype=torch.float32, device=dev) for _ in range(6)]
    gate = torch.empty((R, C), dtype=torch.float32, device=dev)
    new = torch.empty((R, 3, 3 * C), dtype=torch.float32, device=dev)
    at = lambda ts: (_lib._vp * len(ts))(*(t.data_ptr() for t in ts))  # noqa: E731
    a = _lib.Gdn2LmPremixStep(R, S, H, D, 6 * C + H if R == 1 else y.stride(0),
                              0 if parents is None else _INDEX[parents.dtype], float(g_max), y.data_ptr(),
                              history.data_ptr(), None if parents is None else parents.data_ptr(), at(cw), at(cb),
                              at(gb), decay_b.data_ptr(), decay_a.data_ptr(), at(outs), gate.data_ptr(), new.data_ptr())
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().gdn2_lm_premix_step_fwd(ctypes.byref(a), _lib.stream_handle(dev)), "gdn2_lm_premix_step_fwd")
    return PremixStep(*outs, gate, new)


def _parent_rows(parents, R):
    """parents as the kernels take them: (R,) int32 or int64."""
    if parents is None:
        return None
    if tuple(parents.shape) != (R,):
        raise ValueError(f"parents must be ({R},), got {tuple(parents.shape)}")
    if parents.is_floating_point() or parents.is_complex() or parents.dtype == torch.bool:
        raise TypeError(f"parents must be whole numbers, got {parents.dtype}")
    return parents.contiguous() if parents.dtype in _INDEX else parents.to(torch.int64)
