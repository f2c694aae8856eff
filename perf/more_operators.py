"""A training step of the language model around its blocks, as measured cases: the operators that a
program calls for products, loss and update.

* ``linear``  ``linear.linear``: rows times a matrix, with bias, activation and residual behind the product;
              alone (serving) or with all its gradients (training);
* ``loss``    ``losses.cross_entropy``: next-token cross-entropy with the gradient of the logits;
* ``adamw``   ``optim.AdamW``: one update of many tensors, clipped by their global norm, states of 32 or 8 bits.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token of a single user through a wide layer: every weight read for one row
        {"name": "linear_m1_4096x14336_bf16", "kind": "linear", "M": 1, "K": 4096, "N": 14336, "dtype": "bf16", "act": "silu",
         "bias": False, "residual": False, "grad": False},
        # seven sequences through a layer of odd sizes: all latency
        {"name": "linear_m7_1000x777_fp16", "kind": "linear", "M": 7, "K": 1000, "N": 777, "dtype": "fp16", "act": "gelu",
         "bias": True, "residual": True, "grad": False},
        # a prompt of 2048 tokens into a wide layer
        {"name": "linear_m2048_4096x14336_bf16", "kind": "linear", "M": 2048, "K": 4096, "N": 14336, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": False, "grad": False},
        # training: the benchmark LM's product from the mixer back to the residual stream, one sequence, float32
        {"name": "linear_grad_m2048_768x512_fp32", "kind": "linear", "M": 2048, "K": 768, "N": 512, "dtype": "fp32",
         "act": "none", "bias": False, "residual": True, "grad": True},
        # training: the benchmark LM's MLP input over its whole batch (8 sequences of 2048)
        {"name": "linear_grad_m16384_512x1024_bf16", "kind": "linear", "M": 16384, "K": 512, "N": 1024, "dtype": "bf16",
         "act": "silu", "bias": False, "residual": False, "grad": True},
        # training: a large layer
        {"name": "linear_grad_m8192_4096x4096_bf16", "kind": "linear", "M": 8192, "K": 4096, "N": 4096, "dtype": "bf16",
         "act": "gelu_tanh", "bias": True, "residual": True, "grad": True},
        # a few tokens over an ordinary vocabulary, odd, smoothed, some of them padding: all latency
        {"name": "loss_n5_v50257_fp16", "kind": "loss", "rows": 5, "V": 50257, "dtype": "fp16", "smoothing": 0.1, "z": 0.0,
         "ignored": 0.4, "reduction": "sum", "grad": True},
        # the benchmark LM's batch over its byte vocabulary
        {"name": "loss_n16384_v256_fp32", "kind": "loss", "rows": 16384, "V": 256, "dtype": "fp32", "smoothing": 0.0, "z": 0.0,
         "ignored": 0.0005, "reduction": "mean", "grad": True},
        # a training batch over a large vocabulary
        {"name": "loss_n8192_v131072_bf16", "kind": "loss", "rows": 8192, "V": 131072, "dtype": "bf16", "smoothing": 0.0,
         "z": 1e-4, "ignored": 0.1, "reduction": "mean", "grad": True},
        # one layer of the benchmark LM, states of 8 bits: all latency
        {"name": "adamw_layer_8bit", "kind": "adamw", "layers": 1, "tensors": 0, "numel": 0, "mix": 0, "dtype": "fp32", "bits": 8,
         "clip": False},
        # the benchmark LM's 186 tensors as its training step updates them
        {"name": "adamw_lm_fp32", "kind": "adamw", "layers": 8, "tensors": 0, "numel": 0, "mix": 0, "dtype": "fp32", "bits": 32,
         "clip": True},
        # a shard of a large model: bfloat16 parameters with float32 masters
        {"name": "adamw_200m_bf16", "kind": "adamw", "layers": 0, "tensors": 24, "numel": 200000000, "mix": 1, "dtype": "bf16",
         "bits": 32, "clip": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "loss", "loss", "adamw", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "linear":
        M, K, N, grad = _spread(rng, 1, 16384), _spread(rng, 32, 14336), _spread(rng, 32, 14336), rng.random() < 0.5
        while M * K * N * (3 if grad else 1) > 3 * 8192 * 4096 * 4096:
            M, K, N = max(1, M * 3 // 4), max(32, K * 7 // 8), max(32, N * 7 // 8)
        return {"kind": kind, "M": M, "K": K, "N": N, "dtype": dtype, "act": rng.choice(["none", "silu", "gelu", "gelu_tanh"]),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "grad": grad}
    if kind == "loss":
        rows, V = _spread(rng, 1, 16384), _spread(rng, 32, 131072)
        while rows * V > 8192 * 131072:
            rows, V = max(1, rows * 3 // 4), max(32, V * 7 // 8)
        return {"kind": kind, "rows": rows, "V": V, "dtype": dtype, "smoothing": rng.choice([0.0, 0.0, 0.1]),
                "z": rng.choice([0.0, 1e-4]), "ignored": rng.choice([0.0, 0.1, 0.5]), "reduction": rng.choice(["mean", "sum"]),
                "grad": rng.random() < 0.8}
    tensors = _spread(rng, 1, 200)
    return {"kind": kind, "layers": 0, "tensors": tensors, "numel": _spread(rng, 1000 * tensors, 200000000),
            "mix": rng.randrange(1 << 30), "dtype": dtype, "bits": rng.choice([8, 32]), "clip": rng.random() < 0.6}


def _sizes(case):
    """The tensors' sizes: the benchmark LM's of so many layers, or large and small ones, the first the largest."""
    if case["layers"]:
        d, p, h, mlp = 512, 768, 6, 1024
        layer = 6 * [d * p] + [d * h] + 3 * [p * 4, p] + 2 * [p] + [h, h, p, p * d, d, d * mlp, d * mlp, mlp * d]
        return [256 * d] + case["layers"] * layer + [d]
    rng = random.Random(case["mix"])
    share = sorted((math.exp(rng.uniform(-8.0, 0.0)) for _ in range(case["tensors"])), reverse=True)
    return [max(1, int(case["numel"] * s / sum(share))) for s in share]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

LR, BETAS, EPS, DECAY, STEP, MAX_NORM = 1e-3, (0.9, 0.999), 1e-8, 0.01, 200, 1.0
BLOCK = 256             # elements that share a scale of 8-bit states
IGNORE = -100


def _framework():
    at = os.path.join(os.getcwd(), "atomic-ops_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from atomic_gdn2 import linear, losses, optim
    return linear, losses, optim


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    randn = lambda *s: torch.randn(s, device=DEV, generator=gen)  # noqa: E731
    rand = lambda *s: torch.rand(s, device=DEV, generator=gen)  # noqa: E731
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        leaf = lambda t: t.to(dt).requires_grad_(case["grad"])  # noqa: E731
        # activations as norms leave them, a few channels ten times the others
        s["x"] = leaf(randn(M, K) * torch.where(rand(K) < 0.005, 10.0, 1.0))
        s["w"] = leaf(randn(K, N) / math.sqrt(K))
        s["bias"] = leaf(randn(N) * 0.2) if case["bias"] else None
        s["residual"] = leaf(randn(M, N)) if case["residual"] else None
        s["dy"] = randn(M, N).to(dt) if case["grad"] else None
    elif case["kind"] == "loss":
        rows, V = case["rows"], case["V"]
        # logits of a model that is fairly sure of its targets; some tokens banned in some rows
        x = randn(rows, V) * 2.5
        s["targets"] = torch.randint(0, V, (rows,), device=DEV, generator=gen)
        at = s["targets"][:, None]
        x.scatter_add_(1, at, 4.0 * rand(rows, 1) * math.log(V))
        if not case["smoothing"]:
            keep = x.gather(1, at)
            x[: rows // 4].masked_fill_(rand(V) < 0.02, -math.inf)
            x.scatter_(1, at, keep)
        s["logits"] = x.to(dt).requires_grad_(case["grad"])
        s["targets"] = torch.where(rand(rows) < case["ignored"], IGNORE, s["targets"])
    else:
        sizes = _sizes(case)
        # one buffer each for all parameters, gradients and states, every tensor from a whole block on
        starts, total = [], 0
        for n in sizes:
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        views = lambda t: [t[a:a + n] for a, n in zip(starts, sizes)]  # noqa: E731
        blocks = torch.tensor([-(-n // BLOCK) for n in sizes], device=DEV)
        last = (torch.tensor(starts, device=DEV) + torch.tensor(sizes, device=DEV)).repeat_interleave(blocks)
        used = torch.arange(total, device=DEV).view(-1, BLOCK) < last[:, None]
        # gradients of tensors, blocks and elements of different size, as embeddings and norms give them
        size = torch.exp(randn(len(sizes)).repeat_interleave(blocks) + 0.5 * randn(total // BLOCK))[:, None] * 2e-4
        draw_ = lambda: torch.where(used, randn(total // BLOCK, BLOCK) * size, 0.0)  # noqa: E731
        g, m = draw_(), draw_() * 0.3
        v = torch.where(used, (size * torch.exp(0.5 * randn(total // BLOCK, BLOCK))) ** 2, 0.0)
        master = torch.where(used, randn(total // BLOCK, BLOCK) * 0.05, 0.0).view(-1)
        s["p"], s["g"], s["step"] = master.to(dt), g.view(-1).to(dt), STEP
        s["master"] = None if dt == torch.float32 else master
        if case["bits"] == 32:
            s["m"], s["v"] = m.view(-1), v.view(-1)
        else:
            s["m"], s["m_scale"] = _nearest(m, 127, torch.int8)
            s["v"], s["v_scale"] = _nearest(v.sqrt(), 255, torch.uint8)
            s["m_out"], s["v_out"] = torch.empty(total, device=DEV), torch.empty(total, device=DEV)
            s["tensor"] = torch.arange(len(sizes), device=DEV).repeat_interleave(blocks)
            s["element"] = (torch.arange(total, device=DEV).view(-1, BLOCK)
                            - torch.tensor(starts, device=DEV).repeat_interleave(blocks)[:, None])
        if own:
            s["views"] = {k: views(s[k]) for k in ("p", "g", "m", "v", "master", "m_out", "v_out") if s.get(k) is not None}
            params = [torch.nn.Parameter(t) for t in s["views"]["p"]]
            s["opt"] = _framework()[2].AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                                             max_norm=MAX_NORM if case["clip"] else None)
            for i, (p, t) in enumerate(zip(params, s["views"]["g"])):
                p.grad = t
                state = {"step": torch.tensor(float(STEP), device=DEV), "exp_avg": s["views"]["m"][i], "exp_avg_sq": s["views"]["v"][i]}
                if dt != torch.float32:
                    state["master"] = s["views"]["master"][i]
                if case["bits"] == 8:
                    at = slice(starts[i] // BLOCK, starts[i] // BLOCK + -(-sizes[i] // BLOCK))
                    state["exp_avg_scale"], state["exp_avg_sq_scale"] = s["m_scale"][at], s["v_scale"][at]
                s["opt"].state[p] = state
    return s


def _nearest(x, top, dtype):
    """Codes c whose squares, signed, are nearest to the blocks of x in units of the blocks' largest."""
    scale = x.abs().amax(1) * (1.0 / top ** 2)
    c = torch.sqrt(x.abs() / torch.where(scale > 0, scale, 1.0)[:, None]).round().clamp(max=top)
    return (torch.sign(x) * c).to(dtype).view(-1), scale


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

SQRT_HALF, SQRT_2_PI = math.sqrt(0.5), math.sqrt(2.0 / math.pi)


def _activation(z, act):
    """The activation of z and its derivative, in z's type."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * SQRT_HALF))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (0.5 * SQRT_2_PI)
    t = torch.tanh(SQRT_2_PI * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * SQRT_2_PI * (1.0 + 3.0 * 0.044715 * z * z)


def _plain_linear(s):
    x, w, case = s["x"].detach().float(), s["w"].detach().float(), s["case"]
    z = x @ w
    if case["bias"]:
        z = z + s["bias"].detach().float()
    a, slope = _activation(z, case["act"])
    y = a + s["residual"].detach().float() if case["residual"] else a
    dt = s["x"].dtype
    out = {"y": y.to(dt)}
    if case["grad"]:
        dz = s["dy"].float() * slope
        out["dx"], out["dw"] = (dz @ w.t()).to(dt), (x.t() @ dz).to(dt)
        if case["bias"]:
            out["dbias"] = dz.sum(0).to(dt)
        if case["residual"]:
            out["dresidual"] = s["dy"]
    return out


def _plain_loss(s):
    case, t = s["case"], s["targets"]
    x = s["logits"].detach().float()
    V, e, z = case["V"], case["smoothing"], case["z"]
    kept = t != IGNORE
    at = torch.where(kept, t, 0)[:, None]
    top = x.amax(1, keepdim=True)
    lse = top + (x - top).exp().sum(1, keepdim=True).log()
    rows = lse - (1.0 - e) * x.gather(1, at) + z * lse * lse
    if e:
        rows = rows - e * x.mean(1, keepdim=True)
    rows = torch.where(kept, rows[:, 0], 0.0)
    scale = kept.float()
    if case["reduction"] == "mean":
        scale = scale / kept.sum().clamp(min=1)
    loss = (rows.double() * scale.double()).sum().float()
    if not case["grad"]:
        return {"loss": loss}
    d = (x - lse).exp() * (1.0 + 2.0 * z * lse)
    if e:
        d = d - e / V
    d = d.scatter_add(1, at, torch.full_like(lse, e - 1.0))
    return {"loss": loss, "dlogits": (d * scale[:, None]).to(s["logits"].dtype)}


def _dither(element, tensor, step):
    """Two numbers of (0, 1), of 16 bits each, for every element of every tensor in this step: a hash in 32 bits."""
    low = 0xFFFFFFFF
    x = (element * 0x9E3779B1 + tensor[:, None] * 0x7F4A7C15 + step * 0x6C62272F) & low
    x = ((x ^ (x >> 16)) * 0x5D8AF3B5) & low
    x = ((x ^ (x >> 15)) * 0x2F6B4E1D) & low
    x = x ^ (x >> 16)
    return ((x & 0xFFFF).float() + 0.5) * (1.0 / 65536), ((x >> 16).float() + 0.5) * (1.0 / 65536)


def _codes(x, root, scale, top, value, dither):
    """The code below root / scale's square root or the one above it, in proportion to where x lies between their values."""
    unit = scale > 0
    c = torch.sqrt(root / torch.where(unit, scale, 1.0)).floor().clamp(max=top - 1)
    low, high = value(c), value(c + 1.0)
    return torch.where(unit, torch.where(x - low > dither * (high - low), c + 1.0, c), 0.0)


def _plain_adamw(s):
    case = s["case"]
    b1, b2 = BETAS
    s["step"] += 1
    g = s["g"].float()
    out = {}
    if case["clip"]:
        norm = g.double().square().sum().sqrt()
        g = g * (MAX_NORM / norm.clamp(min=MAX_NORM)).float()
        out["norm"] = norm.float()
    if case["bits"] == 8:
        c, u = s["m"].float(), s["v"].float()
        s_m, s_v = s["m_scale"][:, None], s["v_scale"][:, None]
        m = ((c * c.abs()).view(-1, BLOCK) * s_m).view(-1)
        v = ((u * u).view(-1, BLOCK) * s_v).square().view(-1)
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    # (products and sums rounded one by one: what is then held in 8 bits turns on the last bit)
    p = s["p"] if s["master"] is None else s["master"]
    size, root = LR / (1.0 - b1 ** s["step"]), 1.0 / math.sqrt(1.0 - b2 ** s["step"])
    p = p * (1.0 - LR * DECAY) - (m / (torch.sqrt(v) * root + EPS)) * size
    if s["master"] is not None:
        out["master"] = s["master"].copy_(p)
    out["p"] = s["p"].copy_(p)
    if case["bits"] == 32:
        out["m"], out["v"] = s["m"].copy_(m), s["v"].copy_(v)
        return out
    m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
    r_m, r_v = _dither(s["element"], s["tensor"], s["step"])
    root = torch.sqrt(v)
    s_m, s_v = m.abs().amax(1, keepdim=True) * (1.0 / 127 ** 2), root.amax(1, keepdim=True) * (1.0 / 255 ** 2)
    c = torch.sign(m) * _codes(m.abs(), m.abs(), s_m, 127, lambda c: c * c * s_m, r_m)
    u = _codes(v, root, s_v, 255, lambda u: (u * u * s_v).square(), r_v)
    u = torch.where((v > 0) & (s_v > 0), u.clamp(min=1.0), u)
    s["m"].copy_(c.view(-1))
    s["v"].copy_(u.view(-1))
    s["m_scale"].copy_(s_m.view(-1))
    s["v_scale"].copy_(s_v.view(-1))
    out["m"] = (c * c.abs() * s_m).view(-1)
    out["v"] = (u * u * s_v).square().view(-1)
    return out


PLAIN = {"linear": _plain_linear, "loss": _plain_loss, "adamw": _plain_adamw}


def run(s):
    case = s["case"]
    if not own:
        return PLAIN[case["kind"]](s)
    linear, losses, optim = _framework()
    if case["kind"] == "linear":
        act = None if case["act"] == "none" else case["act"]
        if not case["grad"]:
            return {"y": linear.linear(s["x"], s["w"], bias=s["bias"], residual=s["residual"], activation=act)}
        names = ["x", "w"] + [n for n in ("bias", "residual") if case[n]]
        y = linear.linear(s["x"], s["w"], bias=s["bias"], residual=s["residual"], activation=act)
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        return {"y": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
    if case["kind"] == "loss":
        loss = losses.cross_entropy(s["logits"], s["targets"], ignore_index=IGNORE, label_smoothing=case["smoothing"],
                                    z_loss=case["z"], reduction=case["reduction"])
        if not case["grad"]:
            return {"loss": loss}
        return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, s["logits"])[0]}
    opt = s["opt"]
    opt.step()
    out = {"norm": opt.norm} if case["clip"] else {}
    if s["master"] is not None:
        out["master"] = s["master"]
    out["p"] = s["p"]
    if case["bits"] == 32:
        return {**out, "m": s["m"], "v": s["v"]}
    opt.unpack_states(s["views"]["m_out"], s["views"]["v_out"])
    return {**out, "m": s["m_out"], "v": s["v_out"]}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and the definitions in 64 bits
# ---------------------------------------------------------------------------------------------

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        n = M * K + K * N + M * N + (N if case["bias"] else 0) + (M * N if case["residual"] else 0)
        if case["grad"]:        # dy read; dx, dw and the bias' gradient written
            n += M * N + M * K + K * N + (N if case["bias"] else 0)
        return {"bytes": n * e, "flops": (6 if case["grad"] else 2) * M * K * N}
    if case["kind"] == "loss":
        n = case["rows"] * case["V"]
        return {"bytes": n * e * (2 if case["grad"] else 1) + 8 * case["rows"], "flops": 6 * n}
    # gradient read, parameter (16 bits: and its master) read and written, both states read and written; 8-bit states
    # are also given as the float32 values that they stand for
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
    return {"bytes": int(sum(_sizes(case)) * (e + (8 if e == 4 else 2 + 8) + states)), "flops": 16 * sum(_sizes(case))}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        x, w = s["x"].detach().double(), s["w"].detach().double()
        z = torch.mm(x, w)
        if case["bias"]:
            z += s["bias"].detach().double()
        z.requires_grad_(True)
        y = {"none": lambda t: t * 1.0, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]](z)
        out = {"y": y.detach() + s["residual"].detach().double() if case["residual"] else y.detach()}
        if case["grad"]:
            dz, = torch.autograd.grad(y, z, s["dy"].double())
            out["dx"], out["dw"] = torch.mm(dz, w.t()), torch.mm(x.t(), dz)
            if case["bias"]:
                out["dbias"] = dz.sum(0)
            if case["residual"]:
                out["dresidual"] = s["dy"].double()
        return out
    if case["kind"] == "loss":
        t, total, n = s["targets"], 0.0, max(1, int((s["targets"] != IGNORE).sum()))
        grads = torch.empty(s["logits"].shape, dtype=torch.float64, device=DEV) if case["grad"] else None
        for i in range(0, case["rows"], 1024):
            r = slice(i, i + 1024)
            x = s["logits"][r].detach().double().requires_grad_(case["grad"])
            loss = torch.nn.functional.cross_entropy(x, t[r], ignore_index=IGNORE, label_smoothing=case["smoothing"], reduction="sum")
            loss = loss + case["z"] * (torch.logsumexp(x, 1) * (t[r] != IGNORE)).square().sum()
            if case["reduction"] == "mean":
                loss = loss / n
            total = total + loss.detach()
            if case["grad"]:
                grads[r] = torch.autograd.grad(loss, x)[0]
        return {"loss": total, "dlogits": grads} if case["grad"] else {"loss": total}
    g, out = s["g"].double(), {}
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, MAX_NORM / float(out["norm"]))
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        spread = lambda t: t.double().repeat_interleave(BLOCK)  # noqa: E731
        m = s["m"].double() * s["m"].double().abs() * spread(s["m_scale"])
        v = (s["v"].double() ** 2 * spread(s["v_scale"])) ** 2
    m, v = torch.lerp(g, m, BETAS[0]), torch.lerp(g * g, v, BETAS[1])
    t = STEP + 1
    p = (s["p"] if s["master"] is None else s["master"]).double()
    p = p - LR * (DECAY * p + m / (1 - BETAS[0] ** t) / (torch.sqrt(v / (1 - BETAS[1] ** t)) + EPS))
    if s["master"] is not None:
        out["master"] = p
    out["p"] = p
    # (8-bit states are one of two neighbours, by the dither: no value in 64 bits)
    return {**out, "m": m, "v": v} if case["bits"] == 32 else {**out, "m": None, "v": None}
