"""Token generation with beams, as measured cases: the operators that a program serving the language
model calls for each new token.

* ``w4``      ``w4.w4_linear``: rows of activations times a matrix of 4-bit weights with group scales;
* ``beam``    ``generation.beam_step``: the best n continuations over all beams and the vocabulary;
* ``decode``  ``inference.decode_step(parents=...)``: the recurrence of every beam from its parent's state;
* ``premix``  ``generation.premix_step``: convolutions, gates and norms of one token from the cached
              projections of its beam's parent.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one sequence's token through the LM's input projections (512 -> 6 x 768 and 6 decays): all latency
        {"name": "w4_m1_512x4614_fp32", "kind": "w4", "M": 1, "K": 512, "N": 4614, "group": 64, "dtype": "fp32",
         "zeros": True, "residual": False},
        # five beams through a layer of odd sizes: a last group that ends early, columns past a tile
        {"name": "w4_m5_1000x777_fp16", "kind": "w4", "M": 5, "K": 1000, "N": 777, "group": 32, "dtype": "fp16",
         "zeros": False, "residual": True},
        # one token of a single user through a wide layer: every weight read for one row
        {"name": "w4_m1_8192x28672_bf16", "kind": "w4", "M": 1, "K": 8192, "N": 28672, "group": 128, "dtype": "bf16",
         "zeros": True, "residual": False},
        # a serving batch: eight sequences of four beams into the residual stream
        {"name": "w4_m32_14336x4096_bf16", "kind": "w4", "M": 32, "K": 14336, "N": 4096, "group": 128, "dtype": "bf16",
         "zeros": True, "residual": True},
        # a prompt of 2048 tokens through the same weights
        {"name": "w4_m2048_4096x4096_bf16", "kind": "w4", "M": 2048, "K": 4096, "N": 4096, "group": 128, "dtype": "bf16",
         "zeros": True, "residual": False},
        # four beams over the LM's own byte vocabulary: all latency
        {"name": "beam_b1k4_v256_fp32", "kind": "beam", "B": 1, "K": 4, "V": 256, "n": 4, "dtype": "fp32",
         "eos": False},
        # a serving batch over an ordinary vocabulary, some beams finished, twice the beams kept
        {"name": "beam_b16k4_v32000_bf16", "kind": "beam", "B": 16, "K": 4, "V": 32000, "n": 8, "dtype": "bf16",
         "eos": True},
        # a large batch over a large vocabulary
        {"name": "beam_b64k8_v131072_fp32", "kind": "beam", "B": 64, "K": 8, "V": 131072, "n": 8, "dtype": "fp32",
         "eos": True},
        # one layer of the LM for four beams of one sequence
        {"name": "decode_b1k4h6_fp32", "kind": "decode", "B": 1, "K": 4, "H": 6, "D": 128, "dtype": "fp32"},
        # one layer of the serving benchmark's width for 64 sequences of four beams
        {"name": "decode_b64k4h16_bf16", "kind": "decode", "B": 64, "K": 4, "H": 16, "D": 128, "dtype": "bf16"},
        # the LM's convolutions and gates for four beams of one sequence, and of 256 sequences
        {"name": "premix_b1k4h6", "kind": "premix", "B": 1, "K": 4, "H": 6, "D": 128},
        {"name": "premix_b256k4h6", "kind": "premix", "B": 256, "K": 4, "H": 6, "D": 128},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["w4", "w4", "w4", "beam", "beam", "decode", "premix"])
    if kind == "w4":
        M, K, N = _spread(rng, 1, 2048), _spread(rng, 256, 14336), _spread(rng, 256, 28672)
        while K * N > 8192 * 28672 or M * K * N > 2048 * 4096 * 4096:
            K, N = max(256, K * 3 // 4), max(256, N * 3 // 4)
            M = max(1, M * 7 // 8)
        return {"kind": kind, "M": M, "K": K, "N": N, "group": rng.choice([32, 64, 128]),
                "dtype": rng.choice(["fp32", "bf16", "fp16"]), "zeros": rng.random() < 0.7, "residual": rng.random() < 0.5}
    if kind == "beam":
        B, K, V = _spread(rng, 1, 64), rng.randint(1, 8), _spread(rng, 256, 131072)
        return {"kind": kind, "B": B, "K": K, "V": V, "n": rng.choice([K, 2 * K]),
                "dtype": rng.choice(["fp32", "bf16", "fp16"]), "eos": rng.random() < 0.7}
    B, K = _spread(rng, 1, 64), rng.randint(1, 4)
    if kind == "decode":
        return {"kind": kind, "B": B, "K": K, "H": _spread(rng, 1, 16), "D": rng.choice([64, 128]),
                "dtype": rng.choice(["fp32", "bf16"])}
    return {"kind": kind, "B": _spread(rng, 1, 256), "K": K, "H": _spread(rng, 1, 6), "D": rng.choice([64, 128])}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _framework():
    at = os.path.join(os.getcwd(), "atomic-ops_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from atomic_gdn2 import generation, inference, w4
    return generation, inference, w4


def _parents(gen, B, K):
    """Beams of the rows' own sequences; most go back to one or two of the K, as they do in a search."""
    k = (torch.rand((B, K), device=DEV, generator=gen) ** 2 * K).long().clamp_(max=K - 1)
    return (torch.arange(B, device=DEV)[:, None] * K + k).reshape(-1)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    randn = lambda *s: torch.randn(s, device=DEV, generator=gen)  # noqa: E731
    rand = lambda *s: torch.rand(s, device=DEV, generator=gen)  # noqa: E731
    s = {"case": case}
    if case["kind"] == "w4":
        M, K, N, dt = case["M"], case["K"], case["N"], DTYPES[case["dtype"]]
        groups = -(-K // case["group"])
        # activations as norms leave them, a few channels twenty times the others
        s["x"] = (randn(M, K) * torch.where(rand(K) < 0.005, 20.0, 1.0)).to(dt)
        s["residual"] = randn(M, N).to(dt) if case["residual"] else None
        # codes of roughly normal weights; each group's scale and zero are its own
        s["codes"] = (randn(K, N) * 2.8 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
        s["scales"] = (torch.exp(randn(groups, N) * 0.3) * (0.4 / math.sqrt(K))).to(torch.bfloat16)
        s["zeros"] = (randn(groups, N) * 1.2 + 7.5).round_().clamp_(0, 15).to(torch.uint8) if case["zeros"] else None
        if own:
            # the weights as a serving program keeps them, laid out once when the model is loaded
            s["weight"] = _framework()[2].pack_w4(s["codes"], s["scales"], s["zeros"], group_size=case["group"])
    elif case["kind"] == "beam":
        B, K, V = case["B"], case["K"], case["V"]
        # logits of a model that is fairly sure: a wide bulk, some banned tokens
        x = randn(B * K, V) * 3.0
        x.masked_fill_(rand(V) < 0.01, -math.inf)
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["scores"] = -10.0 - 4.0 * rand(B, K)
        s["eos_id"] = V // 3 if case["eos"] else None
        s["finished"] = rand(B, K) < 0.2 if case["eos"] else None
    elif case["kind"] == "decode":
        B, K, H, D, dt = case["B"], case["K"], case["H"], case["D"], DTYPES[case["dtype"]]
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
        R = B * K
        xs = (unit(randn(R, H, D)), unit(randn(R, H, D)), randn(R, H, D), torch.sigmoid(randn(R, H, D)),
              torch.sigmoid(randn(R, H, D)), -0.1 * torch.nn.functional.softplus(randn(R, H, D)))
        s["xs"] = tuple(x.to(dt) for x in xs)
        s["state"] = (randn(R, H, D, D) * 0.2).to(dt)
        s["parents"] = _parents(gen, B, K)
    else:
        B, K, H, D = case["B"], case["K"], case["H"], case["D"]
        C, R = H * D, B * K
        s["y"], s["history"], s["parents"] = randn(R, 6 * C + H), randn(R, 3, 3 * C), _parents(gen, B, K)
        s["conv_w"] = tuple(randn(C, 4) * 0.5 for _ in range(3))
        s["conv_b"] = tuple(randn(C) * 0.1 for _ in range(3))
        s["gate_b"] = tuple(randn(C) * 0.1 for _ in range(2))
        s["decay_b"], s["decay_a"] = randn(H) * 0.1, randn(H) * 0.3 - 3.0
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

G_MAX = 1.25            # the LM's bound on a token's decay


def _plain_w4(s):
    group = s["case"]["group"]
    K = s["codes"].shape[0]
    spread = lambda t: t.float().repeat_interleave(group, 0)[:K]  # noqa: E731
    zeros = 8.0 if s["zeros"] is None else spread(s["zeros"])
    y = s["x"].float() @ ((s["codes"].float() - zeros) * spread(s["scales"]))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(s["x"].dtype)}


def _plain_beam(s):
    B, K = s["scores"].shape
    x = s["logits"].float().view(B, K, -1)
    V, n, eos, finished = x.shape[-1], s["case"]["n"], s["eos_id"], s["finished"]
    d = x - x.amax(-1, keepdim=True)
    c = s["scores"][:, :, None] + (d - d.exp().sum(-1, keepdim=True).log())
    if finished is not None:
        is_eos = torch.arange(V, device=x.device) == eos
        c = torch.where(finished[:, :, None], torch.where(is_eos, s["scores"][:, :, None], -math.inf), c)
    best, at = torch.sort(c.view(B, K * V), dim=-1, descending=True, stable=True)
    at = at[:, :n]
    k, tokens = at // V, at % V
    out = {"tokens": tokens, "rows": k + torch.arange(B, device=x.device)[:, None] * K, "scores": best[:, :n].clone()}
    if finished is not None:
        out["finished"] = finished.gather(1, k) | (tokens == eos)
    return out


def _plain_decode(s):
    q, k, v, w, b, g = (x.float() for x in s["xs"])
    h = s["state"].float()[s["parents"]] * torch.exp(g.clamp(max=0.0))[..., None]
    erase = ((b * k)[..., None] * h).sum(-2)
    h = h + k[..., None] * (w * v - erase)[..., None, :]
    o = (h * (q * (1.0 / math.sqrt(q.shape[-1])))[..., None]).sum(-2)
    finite = lambda x: torch.where(torch.isfinite(x), x, 0.0)  # noqa: E731
    return {"o": finite(o).to(s["xs"][0].dtype), "state": finite(h).to(s["state"].dtype)}


def _plain_premix(s):
    H, D = s["case"]["H"], s["case"]["D"]
    C, y = H * D, s["y"]
    R = y.shape[0]
    past = s["history"][s["parents"]]
    window = torch.cat([past, y[:, None, :3 * C]], 1)
    sigmoid = lambda x: 1.0 / (1.0 + torch.exp(-x))  # noqa: E731
    heads = lambda x: x.reshape(R, H, D)  # noqa: E731
    u = (window * torch.cat(s["conv_w"]).t()).sum(1) + torch.cat(s["conv_b"])
    u = u * sigmoid(u)
    q, k, v = (heads(u[:, i * C:(i + 1) * C]) for i in range(3))
    q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    b, w = (heads(sigmoid(y[:, (3 + i) * C:(4 + i) * C] + s["gate_b"][i])) for i in range(2))
    z = y[:, 6 * C:] + s["decay_b"]
    decay = torch.exp(s["decay_a"]) * (z.clamp(min=0.0) + torch.log1p(torch.exp(-z.abs())))
    g = -decay.clamp(max=G_MAX)[..., None].expand(R, H, D)
    return {"q": q, "k": k, "v": v.clamp(-50.0, 50.0), "w": w, "b": b, "g": g.contiguous(),
            "gate": y[:, 5 * C:6 * C].contiguous(), "history": window[:, 1:].contiguous()}


PLAIN = {"w4": _plain_w4, "beam": _plain_beam, "decode": _plain_decode, "premix": _plain_premix}


def run(s):
    if not own:
        return PLAIN[s["case"]["kind"]](s)
    generation, inference, w4 = _framework()
    kind = s["case"]["kind"]
    if kind == "w4":
        return {"y": w4.w4_linear(s["x"], s["weight"], residual=s["residual"])}
    if kind == "beam":
        r = generation.beam_step(s["logits"], s["scores"], n=s["case"]["n"], finished=s["finished"], eos_id=s["eos_id"])
        out = {"tokens": r.tokens, "rows": r.rows, "scores": r.scores}
        return out if r.finished is None else {**out, "finished": r.finished}
    if kind == "decode":
        o, state = inference.decode_step(*s["xs"], s["state"], 1.0 / math.sqrt(s["case"]["D"]),
                                         state_dtype=s["state"].dtype, parents=s["parents"])
        return {"o": o, "state": state}
    r = generation.premix_step(s["y"], s["history"], s["conv_w"], s["conv_b"], s["gate_b"], s["decay_b"], s["decay_a"],
                               n_heads=s["case"]["H"], g_max=G_MAX, parents=s["parents"])
    return {"q": r.q, "k": r.k, "v": r.v, "w": r.w, "b": r.b, "g": r.g, "gate": r.gate, "history": r.history}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and the definitions in 64 bits
# ---------------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "w4":
        M, K, N = case["M"], case["K"], case["N"]
        e = 4 if case["dtype"] == "fp32" else 2
        rows = M * (K + N * (2 if case["residual"] else 1)) * e
        # half a byte a weight, a scale of two bytes and a zero of one a group
        return {"bytes": K * N // 2 + -(-K // case["group"]) * N * (3 if case["zeros"] else 2) + rows, "flops": 2 * M * K * N}
    if case["kind"] == "beam":
        n = case["B"] * case["K"] * case["V"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2), "flops": 4 * n}
    R = case["B"] * case["K"]
    if case["kind"] == "decode":
        e, h = 4 if case["dtype"] == "fp32" else 2, R * case["H"] * case["D"] ** 2
        # every row's new state, and the states read: of a sequence's K, about the share that
        # _parents' distribution leaves with a child
        K = case["K"]
        read = sum(1 - (1 - (math.sqrt((k + 1) / K) - math.sqrt(k / K))) ** K for k in range(K)) / K
        return {"bytes": int(h * e * (1 + read)) + 7 * R * case["H"] * case["D"] * e, "flops": 7 * h}
    C = case["H"] * case["D"]
    return {"bytes": 4 * R * (6 * C + case["H"] + 9 * C + 9 * C + 7 * C), "flops": 60 * R * C}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "w4":
        K, group = case["K"], case["group"]
        y = torch.zeros((case["M"], case["N"]), dtype=torch.float64, device=DEV)
        for g in range(s["scales"].shape[0]):
            rows = slice(g * group, min(K, (g + 1) * group))
            x = s["x"][:, rows].double()
            q = x @ s["codes"][rows].double()
            z = 8.0 if s["zeros"] is None else s["zeros"][g].double()
            y += s["scales"][g].double() * (q - z * x.sum(1, keepdim=True))
        return {"y": y if s["residual"] is None else y + s["residual"].double()}
    if case["kind"] == "beam":
        B, K, V = case["B"], case["K"], case["V"]
        best = []
        for i in range(B):
            p = torch.log_softmax(s["logits"][i * K:(i + 1) * K].double(), -1) + s["scores"][i].double()[:, None]
            if s["finished"] is not None:
                done = s["finished"][i]
                p[done] = -math.inf
                p[done, s["eos_id"]] = s["scores"][i, done].double()
            best.append(torch.topk(p.reshape(-1), case["n"]).values)
        out = {"tokens": None, "rows": None, "scores": torch.stack(best)}
        return out if s["finished"] is None else {**out, "finished": None}
    if case["kind"] == "decode":
        os_, hs = [], []
        for i in range(0, s["parents"].numel(), 32):
            r = slice(i, i + 32)
            q, k, v, w, b, g = (x[r].double() for x in s["xs"])
            h = torch.exp(g).unsqueeze(-1) * s["state"][s["parents"][r]].double()
            new = w * v - torch.matmul((b * k).unsqueeze(-2), h).squeeze(-2)
            h = h + torch.matmul(k.unsqueeze(-1), new.unsqueeze(-2))
            os_.append(torch.matmul(q.unsqueeze(-2), h).squeeze(-2) / math.sqrt(case["D"]))
            hs.append(h)
        return {"o": torch.cat(os_), "state": torch.cat(hs)}
    H, D = case["H"], case["D"]
    C, y = H * D, s["y"].double()
    past = s["history"].double()[s["parents"]]
    out = {}
    for i, n in enumerate("qkv"):
        c = slice(i * C, (i + 1) * C)
        w = s["conv_w"][i].double()
        u = past[:, 0, c] * w[:, 0] + past[:, 1, c] * w[:, 1] + past[:, 2, c] * w[:, 2] + y[:, c] * w[:, 3] + s["conv_b"][i].double()
        u = torch.nn.functional.silu(u).view(-1, H, D)
        out[n] = u.clamp(-50, 50) if n == "v" else u * torch.rsqrt(u.square().sum(-1, keepdim=True) + 1e-6)
    for i, n in enumerate("bw"):
        out[n] = torch.sigmoid(y[:, (3 + i) * C:(4 + i) * C] + s["gate_b"][i].double()).view(-1, H, D)
    d = torch.exp(s["decay_a"].double()) * torch.nn.functional.softplus(y[:, 6 * C:] + s["decay_b"].double())
    out["g"] = -d.clamp(max=G_MAX)[..., None].expand(-1, H, D)
    out["gate"] = y[:, 5 * C:6 * C]
    out["history"] = torch.cat([past[:, 1:], y[:, None, :3 * C]], 1)
    return out
