"""AdamW over many tensors in few launches, on the HIP kernels of ``csrc/gdn2_optim.hip``.

``AdamW`` is a ``torch.optim.Optimizer``: parameter groups, state_dict and schedulers as there.  A step forms the
gradients' global norm, clips by it and updates every tensor, without waiting for the GPU, so it can be captured into
a graph once every parameter has taken a step (the step counts live on the GPU; lr and the others are those of the capture).
"""
from __future__ import annotations

import ctypes
from itertools import chain

import torch

from . import _lib

__all__ = ["AdamW"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # GDN2_F32, GDN2_BF16, GDN2_F16
_BLOCK = 256                                                             # GDN2_ADAMW_BLOCK


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, clipped by the global norm of all gradients.

    params: tensors or groups, float32, bfloat16 or float16 in any mixture, contiguous, on one ROCm device; 16-bit ones
    are updated as a float32 ``master`` in their state and rounded (values written into one between steps count, and
    its master starts anew from them).  max_norm: every gradient times max_norm /
    max(norm, max_norm) (None, or infinite: as it is); ``norm`` is then the last step's norm, a float32 scalar on the GPU (0 where
    there was no gradient).
    state_bits: 32, or 8: ``exp_avg`` and ``exp_avg_sq`` as codes of one byte, with a scale for each 256 elements
    (include/gdn2.h, gdn2_adamw); ``unpack_states`` gives the values that they stand for.  A NaN or infinity in a
    gradient goes into what is formed from it (in 8 bits its block); with a finite max_norm a NaN goes into everything, and an
    infinity makes the factor 0: NaN where it is, a step of no gradient elsewhere."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 max_norm=None, state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits={state_bits}: 8 or 32")
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError(f"max_norm={max_norm}: positive, or None")
        self.max_norm, self.state_bits, self.norm = None if max_norm is None else float(max_norm), state_bits, None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm, "state_bits": self.state_bits, "norm": None}

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._minimises(group)
            self._hyper(group)
            for p in group["params"]:
                self._check(p)
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    @staticmethod
    def _minimises(group):
        """torch.optim's groups may ask for steps that are not formed here."""
        for key in ("maximize", "amsgrad"):
            if group.get(key):
                raise ValueError(f"a group with {key}={group[key]}: AdamW has no {key}")
        if not group.get("decoupled_weight_decay", True) and group["weight_decay"]:
            raise ValueError("a group of Adam's weight decay: AdamW's is decoupled from the gradient")

    @staticmethod
    def _hyper(group):
        """(lr, beta1, beta2, eps, weight_decay) of a group."""
        h = (group["lr"], *group["betas"], group["eps"], group["weight_decay"])
        if any(isinstance(x, torch.Tensor) and x.is_cuda for x in h):
            raise TypeError("lr and the others must be numbers: reading a tensor on the GPU would wait for it")
        lr, b1, b2, eps, wd = h = tuple(float(x) for x in h)
        if not (lr >= 0.0 and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0 and wd >= 0.0):
            raise ValueError(f"lr={lr}, betas={(b1, b2)}, eps={eps}, weight_decay={wd}: not negative, betas below 1")
        return h

    def _check(self, p):
        if p.dtype not in _DTYPES:
            raise TypeError(f"parameters must be float32, bfloat16 or float16, got {p.dtype}")
        if not p.is_cuda or p.layout != torch.strided:
            raise ValueError(f"AdamW needs dense tensors on a ROCm device, got {p.layout} on {p.device}")
        if not p.is_contiguous():
            raise ValueError(f"parameters must be contiguous, got strides {p.stride()} for {tuple(p.shape)}")
        dev = next(q.device for group in self.param_groups for q in group["params"])       # (a group may be empty)
        if p.device != dev:
            raise ValueError(f"parameters must be on one device, got {p.device} and {dev}")

    def _state(self, p):
        """p's state, made at its first step."""
        s = self.state[p]
        if not s:
            if torch.cuda.is_current_stream_capturing():        # (each replay would begin with the states anew)
                raise RuntimeError("a parameter's first step makes its state: take one before a step is captured")
            f32 = lambda n: torch.zeros(n, dtype=torch.float32, device=p.device)  # noqa: E731
            s["step"] = f32(())
            if self.state_bits == 32:
                s["exp_avg"], s["exp_avg_sq"] = f32(p.shape), f32(p.shape)
            else:
                s["exp_avg"] = torch.zeros(p.shape, dtype=torch.int8, device=p.device)
                s["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
                blocks = -(-p.numel() // _BLOCK)
                s["exp_avg_scale"], s["exp_avg_sq_scale"] = f32(blocks), f32(blocks)
            if p.dtype != torch.float32:
                s["master"] = p.detach().to(torch.float32)
        return s

    def _tensors(self, p, s):
        """The state's tensors in the order of gdn2_adamw_tensor, looked over: the kernels read by p's size."""
        n, byte = p.numel(), self.state_bits == 8
        want = [("exp_avg", torch.int8 if byte else torch.float32, n), ("exp_avg_sq", torch.uint8 if byte else torch.float32, n),
                ("exp_avg_scale", torch.float32, -(-n // _BLOCK) if byte else None),
                ("exp_avg_sq_scale", torch.float32, -(-n // _BLOCK) if byte else None),
                ("master", torch.float32, None if p.dtype == torch.float32 else n), ("step", torch.float32, 1)]
        out = []
        for key, dtype, size in want:
            t = s.get(key) if size is not None else None
            if size is not None and not (isinstance(t, torch.Tensor) and t.dtype == dtype and t.numel() == size and t.device == p.device
                                         and t.is_contiguous()):
                raise ValueError(f"state {key!r} must be contiguous {dtype} of {size} elements on {p.device}")
            out.append(t)
        return out

    def _entry(self, a, p, g, s, ordinal, hyper):
        m, v, ms, vs, master, step = (None if t is None else t.data_ptr() for t in self._tensors(p, s))
        a.p, a.g, a.m, a.v, a.m_scale, a.v_scale, a.master, a.step = p.data_ptr(), None if g is None else g.data_ptr(), m, v, ms, vs, master, step
        a.numel, a.ordinal, a.dtype = p.numel(), ordinal, _DTYPES[p.dtype]
        a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = hyper

    @torch.no_grad()
    def step(self, closure=None):
        """One update of every parameter that has a gradient.  closure: as in torch.optim."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # plain steps (csrc/bind.cpp) go native; None = not one, and what follows handles it
        done = _lib.bind().adamw(self.param_groups, self.state, self.state_bits, self.max_norm or 0.0)
        if done is not None:
            self.norm = None if done is True else done
            return loss
        todo, ordinal = [], 0
        for group in self.param_groups:
            hyper = self._hyper(group)
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    if p.grad.is_sparse:
                        raise RuntimeError("AdamW takes no sparse gradients")
                    self._check(p)
                    todo.append((p, p.grad.to(p.dtype).contiguous(), self._state(p), ordinal, hyper))
                ordinal += 1
        if not todo:
            dev = next((p.device for group in self.param_groups for p in group["params"]), None)
            self.norm = None if self.max_norm is None or dev is None else torch.zeros((), dtype=torch.float32, device=dev)
            return loss
        dev = todo[0][0].device
        ts = (_lib.Gdn2AdamwTensor * len(todo))()
        for a, one in zip(ts, todo):
            self._entry(a, *one)
        L = _lib.lib()
        self.norm = None if self.max_norm is None else torch.empty((), dtype=torch.float32, device=dev)
        ws = torch.empty(L.gdn2_adamw_workspace_bytes(ts, len(todo)), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            _lib.check(L.gdn2_adamw(ts, len(todo), self.state_bits, self.max_norm or 0.0, _lib.ptr(self.norm), _lib.ptr(ws),
                                    _lib.stream_handle(dev)), "gdn2_adamw")
        torch.autograd.graph.increment_version([p for p, *_ in todo])
        return loss

    @torch.no_grad()
    def unpack_states(self, exp_avg=None, exp_avg_sq=None):
        """The float32 values of 8-bit states, (exp_avg, exp_avg_sq): lists with a tensor for each parameter, in the
        groups' order, written into the given tensors or new ones (a parameter without a state has zeros)."""
        if self.state_bits != 8:
            raise ValueError("states of 32 bits are values already")
        if type(exp_avg) is list and type(exp_avg_sq) is list and _lib.bind().adamw_unpack(self.param_groups, self.state, exp_avg, exp_avg_sq):
            return exp_avg, exp_avg_sq
        ps = [p for group in self.param_groups for p in group["params"]]
        outs = []
        for given in (exp_avg, exp_avg_sq):
            outs.append([torch.empty(p.shape, dtype=torch.float32, device=p.device) for p in ps] if given is None else list(given))
            if len(outs[-1]) != len(ps) or not all(t.dtype == torch.float32 and t.numel() == p.numel() and t.device == p.device
                                                   and t.is_contiguous() for t, p in zip(outs[-1], ps)):
                raise ValueError("a contiguous float32 tensor of its size is needed for each parameter")
        at = []
        for i, p in enumerate(ps):
            if p.numel() and self.state.get(p):
                at.append(i)
            else:
                outs[0][i].zero_()
                outs[1][i].zero_()
        if at:
            ts = (_lib.Gdn2AdamwTensor * len(at))()
            for a, i in zip(ts, at):
                self._entry(a, ps[i], None, self.state[ps[i]], i, (0.0,) * 5)
            ptrs = [(ctypes.c_void_p * len(at))(*(out[i].data_ptr() for i in at)) for out in outs]
            dev = ps[0].device
            with torch.cuda.device(dev):
                _lib.check(_lib.lib().gdn2_adamw_unpack(ts, len(at), *ptrs, _lib.stream_handle(dev)), "gdn2_adamw_unpack")
            torch.autograd.graph.increment_version([out[i] for out in outs for i in at])
        return tuple(outs)

    def load_state_dict(self, state_dict):
        """As in torch.optim, but states keep their own dtypes (there they take the parameter's); states of
        torch.optim.AdamW are taken over with state_bits 32, but for those of one that maximises or is amsgrad (or of
        Adam's weight decay), which are refused.  The states must fit state_bits."""
        for group in state_dict["param_groups"]:
            self._minimises(group)
        ps = [p for group in self.param_groups for p in group["params"]]
        ids = list(chain.from_iterable(g["params"] for g in state_dict["param_groups"]))
        new = {}
        if len(ids) == len(ps):
            for i, p in zip(ids, ps):
                old = state_dict["state"].get(i)
                if not old:
                    continue
                s = {}
                for key, t in old.items():
                    if not isinstance(t, torch.Tensor):
                        t = torch.tensor(float(t)) if key == "step" else t
                    if isinstance(t, torch.Tensor):
                        t = t.detach().to(device=p.device, dtype=torch.float32 if t.is_floating_point() else t.dtype, copy=True).contiguous()
                    s[key] = t
                if p.dtype != torch.float32 and "master" not in s:
                    s["master"] = p.detach().to(torch.float32)
                self._tensors(p, s)
                new[p] = s
        super().load_state_dict(state_dict)
        self.state.update(new)
