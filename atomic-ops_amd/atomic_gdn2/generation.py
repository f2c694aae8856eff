"""Token generation from the benchmark LM: beam search on the HIP kernels.

* ``Generator``    the LM with 4-bit weights (``w4``): prefill of a prompt, one token for a batch of
                   sequences, and ``beam_search`` over them;
* ``beam_step``      of all continuations of a group's beams, the best n (``csrc/gdn2_beam.hip``);
* ``premix_step``  one token of a block's convolutions, gates and norms from the cached projections of
                   the three tokens before it (``csrc/gdn2_lm.hip``).

A beam that is kept continues the sequence of its parent, so its caches are its parent's.  Both caches
of a block are taken from the parent's row where a step reads them anyway (``parents`` here and in
``inference.decode_step``): nothing is copied to reorder them.  For inference: no gradients; asking
``beam_step`` or ``premix_step`` for one raises.
"""
from __future__ import annotations

import ctypes
from typing import List, NamedTuple, Optional

import torch

from . import _lib, lm_kernels
from .inference import chunk_forward_inference, decode_step
from .w4 import for_inference, quantize_w4, w4_linear

__all__ = ["BeamStep", "PremixStep", "beam_step", "premix_step", "Cache", "BeamResult", "Generator"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # GDN2_F32, GDN2_BF16, GDN2_F16
_INDEX = {torch.int32: 1, torch.int64: 2}                                # GDN2_FLAG_INT32, GDN2_FLAG_INT64


class BeamStep(NamedTuple):
    """The kept continuations of each group, the best first, all (B, n): the new tokens (int64), the
    rows b K + k of the beams that they continue (int64: ``parents`` of the next steps), their scores
    (float32), and whether they are finished (None without an end token).  They may share one storage."""
    tokens: torch.Tensor
    rows: torch.Tensor
    scores: torch.Tensor
    finished: Optional[torch.Tensor]


class PremixStep(NamedTuple):
    """What the recurrence takes for one token, q, k, v, w, b, g (R, H, D); the output gate's logits
    (R, H D); the history of the next token (R, 3, 3 H D).  All but the history may share one storage."""
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
    continuation, eos_id at its own score; a beam that takes eos_id is finished.  A group's result
    does not depend on what the others hold (on their number its scores' last bits do), and equal inputs
    give equal bits."""
    if isinstance(logits, torch.Tensor) and logits.is_cuda and (finished is None or eos_id is not None) \
            and (eos_id is None or type(eos_id) is int and eos_id >= 0) and (n is None or type(n) is int) and scores.dim() == 2:
        # plain calls (csrc/bind.cpp) go native; None = not one, and what follows handles it
        out = _lib.bind().beam(logits, scores, scores.shape[-1] if n is None else n, finished, -1 if eos_id is None else eos_id)
        if out is not None:
            return BeamStep(*out, None) if eos_id is None else BeamStep(*out)
    out = for_inference("beam_step", lambda *ts: beam_step(*ts, n=n, finished=finished, eos_id=eos_id), logits, scores)
    if out is not None:
        return BeamStep(*out)
    if scores.dim() != 2 or scores.numel() == 0:
        raise ValueError(f"scores must be (B, K), got {tuple(scores.shape)}")
    B, K = scores.shape
    if logits.dim() not in (2, 3) or tuple(logits.shape[:-1]) not in ((B * K,), (B, K)) or logits.shape[-1] == 0:
        raise ValueError(f"logits must be {(B * K, 'V')} or {(B, K, 'V')}, got {tuple(logits.shape)}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    V = logits.shape[-1]
    if max(B * K, K * V) >= 2 ** 31:
        raise ValueError(f"{B} groups of {K} beams over {V} tokens: B K and K V must be below 2^31")
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
    conv_w, conv_b, gate_b = tuple(conv_w), tuple(conv_b), tuple(gate_b)
    if (len(conv_w), len(conv_b), len(gate_b)) != (3, 3, 2):
        raise ValueError("three convolutions (taps and biases) and two gates are needed")
    if isinstance(y, torch.Tensor) and y.is_cuda and type(n_heads) is int and type(g_max) is float:
        out = _lib.bind().premix_step(y, history, (*conv_w, *conv_b, *gate_b, decay_b, decay_a), n_heads, g_max, parents)
        if out is not None:
            return PremixStep(*out)
    out = for_inference("premix_step", lambda y, history, *ws: premix_step(
        y, history, ws[:3], ws[3:6], ws[6:8], *ws[8:], n_heads=n_heads, g_max=g_max, parents=parents),
        y, history, *conv_w, *conv_b, *gate_b, decay_b, decay_a)
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
    if y.stride(1) != 1 or (not 6 * C + H <= y.stride(0) < 2 ** 31 and R > 1):      # (a stride has 32 bits)
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


# ------------------------------------------------------------------------------------------
# the LM
# ------------------------------------------------------------------------------------------

class Cache(NamedTuple):
    """What a batch of R sequences carries to its next token, per block: the recurrence's state
    (R, H, D, D) and the last three tokens' q | k | v projections (R, 3, 3 H D)."""
    states: List[torch.Tensor]
    history: List[torch.Tensor]


class BeamResult(NamedTuple):
    """tokens (B, n_beams, T): the new tokens, the best beam first, eos_id after a beam's end; scores
    (B, n_beams): their log-probabilities."""
    tokens: torch.Tensor
    scores: torch.Tensor


class _Block(NamedTuple):
    w_in: object            # [Wq | Wk | Wv | We | Ww | Wo | Wd], columns to a multiple of 4
    conv_w: tuple
    conv_b: tuple
    gate_b: tuple
    decay_b: torch.Tensor
    decay_a: torch.Tensor
    mix_norm: torch.Tensor
    w_out: object
    mlp_norm: torch.Tensor
    w_gate_up: object
    w_down: object


class Generator:
    """An ``e2e_lm.LM`` with its matrices in 4 bits, for generation: float32 activations, every product
    through ``w4_linear``.  The model itself is not changed or kept."""

    def __init__(self, model, group_size: int = 64, op_cfg=None):
        from . import e2e_lm
        c = model.cfg
        dev = model.embed.device
        if not model.embed.is_cuda:
            raise ValueError(f"Generator needs a model on a ROCm device, got {dev}")
        if c.d_head not in (64, 128) or c.d_conv != 4:
            raise ValueError(f"d_head={c.d_head}, d_conv={c.d_conv}: the HIP kernels support heads of 64 and 128 and 4 taps")
        if max(c.proj_dim, c.d_model) > lm_kernels._MAX_C or c.d_model % 4 or (c.mlp_mult * c.d_model) % 4:
            raise ValueError(f"widths up to {lm_kernels._MAX_C}, multiples of 4")
        self.cfg, self.device = c, dev
        self.op_cfg = e2e_lm.operator_cfg() if op_cfg is None else op_cfg
        self.scale = float(c.d_head) ** -0.5
        f32 = lambda t: t.detach().to(torch.float32).clone()  # noqa: E731
        q4 = lambda *ws: quantize_w4(torch.cat([w.detach() for w in ws], 1), group_size)  # noqa: E731
        pad = torch.zeros((c.d_model, -(6 * c.proj_dim + c.n_heads) % 4), device=dev)
        self.blocks = [_Block(
            w_in=q4(*(m.weight for m in (b.q_proj, b.k_proj, b.v_proj, b.erase_gate, b.write_gate, b.out_gate, b.decay_proj)), pad),
            conv_w=tuple(f32(m.weight) for m in (b.q_conv, b.k_conv, b.v_conv)),
            conv_b=tuple(f32(m.bias) for m in (b.q_conv, b.k_conv, b.v_conv)),
            gate_b=(f32(b.erase_gate.bias), f32(b.write_gate.bias)),
            decay_b=f32(b.decay_proj.bias), decay_a=f32(b.decay_a),
            mix_norm=f32(b.mixer_out_norm.scale), w_out=q4(b.out_proj.weight), mlp_norm=f32(b.mlp_norm.scale),
            w_gate_up=q4(b.gate_proj.weight, b.up_proj.weight), w_down=q4(b.down_proj.weight)) for b in model.blocks]
        self.embed, self.final_norm = f32(model.embed), f32(model.final_norm.scale)
        self.head = q4(model.embed.t())

    def _rest(self, blk, o, gate, x, L):
        """The block behind the recurrence; o (B, H, L, D), gate and x rows (B L, ...)."""
        z = lm_kernels._rms(o, blk.mix_norm, gate, (L, self.cfg.d_head))
        x = w4_linear(z, blk.w_out, residual=x)
        act = lm_kernels._swiglu(w4_linear(lm_kernels._rms(x, blk.mlp_norm), blk.w_gate_up))
        return w4_linear(act, blk.w_down, residual=x)

    def _logits(self, x):
        return w4_linear(lm_kernels._rms(x, self.final_norm), self.head)

    def _ids(self, ids, dim):
        if ids.dim() != dim or ids.numel() == 0 or ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
            raise ValueError(f"token ids must be whole numbers of {dim} dimensions, not empty, got {ids.dtype} {tuple(ids.shape)}")
        if ids.device != self.device:
            raise ValueError(f"token ids are on {ids.device}, the model on {self.device}")

    @torch.no_grad()
    def prefill(self, ids):
        """Prompts ids (B, L) from an empty cache: the logits (B, V) behind the last token, the cache."""
        self._ids(ids, 2)
        ids = ids.long()
        lo, hi = (int(v) for v in torch.aminmax(ids))
        if lo < 0 or hi >= self.cfg.vocab_size:
            raise ValueError(f"token ids must lie in 0 .. {self.cfg.vocab_size - 1}, got {lo} .. {hi}")
        (B, L), c, cache = ids.shape, self.cfg, Cache([], [])
        H, D, C = c.n_heads, c.d_head, c.proj_dim
        x = self.embed[ids].reshape(B * L, -1)
        for blk in self.blocks:
            y = w4_linear(x, blk.w_in)
            ops = [torch.empty((B, H, L, D), device=self.device) for _ in range(6)]
            gate = torch.empty((B * L, C), device=self.device)
            at = lambda ts: (lm_kernels._vp * len(ts))(*(t.data_ptr() for t in ts))  # noqa: E731
            a = lm_kernels._PremixArgs(B, L, H, D, y.shape[1], float(c.g_max), y.data_ptr(), at(blk.conv_w), at(blk.conv_b),
                                       at(blk.gate_b), blk.decay_b.data_ptr(), blk.decay_a.data_ptr(), at(ops), gate.data_ptr())
            lm_kernels._call("gdn2_lm_premix_fwd", self.device, ctypes.byref(a))
            o, state = chunk_forward_inference(*ops, scale=self.scale, cfg=self.op_cfg)
            past = y.view(B, L, -1)[:, max(L - 3, 0):, :3 * C]
            history = torch.zeros((B, 3, 3 * C), device=self.device)
            history[:, 3 - past.shape[1]:] = past
            cache.states.append(state)
            cache.history.append(history)
            x = self._rest(blk, o, gate, x, L)
        return self._logits(x.view(B, L, -1)[:, -1].contiguous()), cache

    @torch.no_grad()
    def step(self, tokens, cache: Cache, rows=None):
        """One token for each of R sequences: tokens (R,), one outside the vocabulary counting as the nearest
        within (the host does not wait for the tokens to look at them); rows (R,): the row of the cache that each
        sequence continues (None: its own).  The logits (R, V) and the sequences' cache."""
        self._ids(tokens, 1)
        return self._step(tokens.long().clamp(0, self.cfg.vocab_size - 1), cache, rows)

    def _step(self, tokens, cache, rows):
        R, c, new = tokens.shape[0], self.cfg, Cache([], [])
        x = self.embed[tokens]
        for blk, state, history in zip(self.blocks, cache.states, cache.history):
            m = premix_step(w4_linear(x, blk.w_in), history, blk.conv_w, blk.conv_b, blk.gate_b, blk.decay_b, blk.decay_a,
                            n_heads=c.n_heads, g_max=float(c.g_max), parents=rows)
            o, state = decode_step(m.q, m.k, m.v, m.w, m.b, m.g, state, self.scale, parents=rows)
            new.states.append(state)
            new.history.append(m.history)
            x = self._rest(blk, o.view(R, c.n_heads, 1, c.d_head), m.gate, x, 1)
        return self._logits(x), new

    def _captured(self, r, cache, n_beams, eos_id):
        """One step and its selection as a HIP graph that works in place on r and cache: its replay.  A step
        of the benchmark LM is 75 launches, bound by the host: 0.66 ms, as a graph 0.33 (8 rows).  The
        caches are copied back inside the graph.  The capture is on a stream of the model's device (torch's own
        one belongs to the device that was current at the process's first capture), and other threads may
        use the GPU meanwhile."""
        keep = [r.tokens, r.rows, r.scores, *([] if r.finished is None else [r.finished]), *cache.states, *cache.history]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.device(self.device), torch.cuda.graph(graph, stream=torch.cuda.Stream(self.device),
                                                              capture_error_mode="thread_local"):
            logits, new = self._step(r.tokens.view(-1), cache, r.rows.view(-1))
            s = beam_step(logits, r.scores, n=n_beams, finished=r.finished, eos_id=eos_id)
            for old, t in zip(keep, [s.tokens, s.rows, s.scores, *([] if s.finished is None else [s.finished]),
                                     *new.states, *new.history]):
                old.copy_(t)
        return graph.replay

    @torch.no_grad()
    def beam_search(self, ids, n_beams: int, max_new_tokens: int, eos_id: Optional[int] = None,
                    graph: Optional[bool] = None) -> BeamResult:
        """The n_beams continuations of each prompt ids (B, L) that beam search keeps, up to
        max_new_tokens tokens.  With eos_id a beam ends when it takes that token, keeping its score, and the
        search ends when all have (looked at every 16 tokens: it costs a synchronisation).  graph: replay
        the steps as a HIP graph; None: from 48 tokens on, where that repays its capture."""
        if max_new_tokens < 1:
            raise ValueError(f"max_new_tokens={max_new_tokens}: at least one is needed")
        graph = max_new_tokens >= 48 if graph is None else graph
        # (the graph is dropped as _search returns, which makes its device the current one)
        with torch.cuda.device(self.device):
            return self._search(ids, n_beams, max_new_tokens, eos_id, graph)

    def _search(self, ids, n_beams, max_new_tokens, eos_id, graph):
        logits, cache = self.prefill(ids)
        B = ids.shape[0]
        # the first token's beams all continue the prompt's one row
        r = beam_step(logits, torch.zeros((B, 1), device=self.device), n=n_beams, eos_id=eos_id)
        steps = [(r.tokens, torch.zeros_like(r.rows))]
        base = torch.arange(B, device=self.device)[:, None] * n_beams
        replay = None
        for t in range(1, max_new_tokens):
            if eos_id is not None and t % 16 == 0 and bool(r.finished.all()):
                break
            if t == 2 and graph:
                replay = self._captured(r, cache, n_beams, eos_id)
            if replay is not None:
                replay()
                steps.append((r.tokens.clone(), r.rows - base))
                continue
            logits, cache = self._step(r.tokens.view(-1), cache, r.rows.view(-1))
            r = beam_step(logits, r.scores, n=n_beams, finished=r.finished, eos_id=eos_id)
            # (copies: a graph that is captured next works in place on r)
            steps.append((r.tokens.clone(), r.rows - base) if graph else (r.tokens, r.rows - base))
        # back from the last token along the parents
        out, at = [], torch.arange(n_beams, device=self.device).expand(B, n_beams)
        for tokens, parent in reversed(steps):
            out.append(tokens.gather(1, at))
            at = parent.gather(1, at)
        return BeamResult(torch.stack(out[::-1], -1), r.scores)


def main():
    """Beam search from the benchmark LM with random weights: tokens and time per token."""
    import time

    from . import e2e_lm
    cfg = e2e_lm.LMConfig()
    gen = Generator(e2e_lm.make_lm(cfg))
    ids = e2e_lm.synthetic_tokens(cfg, batch=2, length=100)
    for n, graph in ((64, False), (64, True), (256, True)):
        gen.beam_search(ids, 4, n, graph=graph)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        r = gen.beam_search(ids, 4, n, graph=graph)
        torch.cuda.synchronize()
        print(f"2 prompts of 100 tokens, 4 beams, {n} new tokens{', graph' if graph else ''}: "
              f"{(time.perf_counter() - t0) * 1e3:.1f} ms, best scores {[round(x, 3) for x in r.scores[:, 0].tolist()]}", flush=True)


if __name__ == "__main__":
    main()
