"""The steps of token generation on the GPU: beam selection against the definition in 64 bits, the
recurrence from parents' states and one token of the block's convolutions and gates.

Beam scores are score + ((x - m) - ln sum): three float32 roundings of at most |score| + 2 |x - m| +
ln V, an exponential within 2e-6 of its value and its sum, so 4 2^-24 (|score| + 2 |x - m| + ln V) +
4e-6 bounds a score's error; where two continuations differ by less than both bounds, either order
is right."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def _scores64(logits, scores, finished, eos):
    """(B, K V) in 64 bits."""
    B, K = scores.shape
    x = torch.nan_to_num(logits.double().reshape(B, K, -1), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    s = torch.nan_to_num(scores.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    m = x.amax(-1, keepdim=True)
    d = torch.where(x == m, 0.0, x - m)
    lp = torch.where((x == -math.inf) | (m == -math.inf), -math.inf, d - d.exp().sum(-1, keepdim=True).log())
    c = torch.where(s[..., None] == -math.inf, -math.inf, lp + s[..., None])
    if finished is not None:
        only = torch.arange(x.shape[-1], device=x.device) == eos
        c = torch.where(finished[..., None], torch.where(only, s[..., None], -math.inf), c)
    return c.reshape(B, -1)


def _check_beam(r, logits, scores, n, finished=None, eos=None):
    B, K = scores.shape
    V = logits.shape[-1]
    c = _scores64(logits, scores, finished, eos)
    assert r.tokens.shape == r.rows.shape == r.scores.shape == (B, n)
    assert r.tokens.dtype == r.rows.dtype == torch.int64 and r.scores.dtype == torch.float32
    k = r.rows - torch.arange(B, device=c.device)[:, None] * K
    assert bool(((k >= 0) & (k < K) & (r.tokens >= 0) & (r.tokens < V)).all())
    flat = k * V + r.tokens
    got, ref = r.scores.double(), c.gather(1, flat)
    x = logits.double().reshape(B, K * V).gather(1, flat)
    top = torch.nan_to_num(logits.double().reshape(B, K, V), nan=-math.inf).amax(-1).gather(1, k)
    fin = torch.isfinite(ref)
    size = scores.double().gather(1, k).abs() + 2 * (top - x).abs() + math.log(V)
    tol = torch.where(fin, 4 * 2.0 ** -24 * size.nan_to_num(0, 0, 0) + 4e-6, 0.0)
    assert bool((torch.where(fin, (got - ref).abs(), 0.0) <= tol).all())
    assert torch.equal(got[~fin], ref[~fin])
    assert bool((r.scores[:, 1:] <= r.scores[:, :-1]).all())
    assert all(len(set(row.tolist())) == n for row in flat)
    # nothing that was left out beats what was kept, and equal scores keep the order of their indices
    left = c.scatter(1, flat, -math.inf)
    assert bool((left.amax(1) <= ref.amin(1) + 2 * tol.amax(1)).all())
    same = (r.scores[:, 1:] == r.scores[:, :-1])
    assert bool((~same | (flat[:, 1:] > flat[:, :-1])).all())
    if eos is None:
        assert r.finished is None
    else:
        was = torch.zeros((B, K), dtype=torch.bool, device=c.device) if finished is None else finished
        assert torch.equal(r.finished, was.gather(1, k) | (r.tokens == eos))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 4, 256, 4), (2, 3, 7, 21), (3, 5, 1001, 5), (4, 4, 2049, 8),
                                     (2, 8, 50257, 16), (1, 2, 131072, 2), (1, 1, 300, 128), (130, 2, 9000, 3),
                                     (2, 128, 40, 128), (1, 16, 20011, 64)])
def test_beam_step_matches_the_definition(B, K, V, n, dtype):
    from atomic_gdn2.generation import beam_step
    print(f"[gpu-test] beam B {B} K {K} V {V} n {n} {dtype}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(B + K + V + n)
    logits = (torch.randn((B * K, V), device="cuda", generator=gen) * 3).to(dtype)
    scores = -5 * torch.rand((B, K), device="cuda", generator=gen)
    r = beam_step(logits, scores, n=n)
    _check_beam(r, logits, scores, n)
    again = beam_step(logits.view(B, K, V), scores, n=n)
    assert all(torch.equal(a, b) for a, b in zip(r[:3], again[:3]))
    eos = V // 2
    fin = torch.rand((B, K), device="cuda", generator=gen) < 0.4
    logits[torch.rand(logits.shape, device="cuda", generator=gen) < 0.3] = -math.inf
    r = beam_step(logits, scores, n=n, finished=fin, eos_id=eos)
    _check_beam(r, logits, scores, n, fin, eos)


def _stable(c, n):
    v, at = torch.sort(c, dim=-1, descending=True, stable=True)
    return v[:, :n], at[:, :n]


def test_beam_ties_go_to_the_lowest_index():
    from atomic_gdn2.generation import beam_step
    V, K = 5000, 3
    # the same few values everywhere, the same rows and scores: ties within rows, pieces and across beams
    row = torch.tensor([1.0, 0.5, 1.0, -0.0, 0.0, 0.5, 1.0], device="cuda").repeat(V // 7 + 1)[:V]
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits = row.to(dtype).expand(2 * K, V).contiguous()
        scores = torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -1.0, -2.0]], device="cuda")
        r = beam_step(logits, scores, n=100)
        c = _scores64(logits, scores, None, None)
        _, at = _stable(c, 100)
        assert torch.equal((r.rows - torch.tensor([[0], [K]], device="cuda")) * V + r.tokens, at)
    flat = beam_step(torch.zeros((1, 70000), device="cuda"), torch.zeros((1, 1), device="cuda"), n=128)
    assert torch.equal(flat.tokens[0], torch.arange(128, device="cuda"))


def test_beam_rows_with_nothing_left():
    """Masked rows, NaN, infinities, dead beams: -inf by the lowest index, never NaN."""
    from atomic_gdn2.generation import beam_step
    inf = math.inf
    V, K = 3000, 4
    gen = torch.Generator(device="cuda").manual_seed(1)
    lowest = torch.finfo(torch.float32).min
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.randn((2 * K, V), device="cuda", generator=gen)
        x[0] = -inf                                    # nothing allowed
        x[1, 5:] = -inf                                # five tokens allowed
        x[2, ::2] = float("nan")
        x[3] = -inf
        x[3, 2500] = 2.0                               # one token, in a later piece
        x[4:] = -inf                                   # a group with nothing at all
        x = x.to(dtype)
        scores = torch.tensor([[-1.0, -2.0, -3.0, -0.5], [-1.0, -inf, float("nan"), 0.0]], device="cuda")
        r = beam_step(x, scores, n=12)
        _check_beam(r, x, scores, 12)
        assert torch.equal(r.scores[1], torch.full((12,), -inf, device="cuda"))
        assert torch.equal(r.tokens[1], torch.arange(12, device="cuda")) and bool((r.rows[1] == K).all())
        assert not r.scores.isnan().any()
        x[:, 7] = inf                                  # certain tokens
        x[:, 2999] = inf
        r = beam_step(x, scores, n=4)
        _check_beam(r, x, scores, 4)
        assert torch.equal(r.tokens[0, :2], torch.tensor([7, 2999], device="cuda"))
    x = torch.full((2, V), lowest, device="cuda")      # masks of the type's lowest value: all alike
    r = beam_step(x, torch.zeros((1, 2), device="cuda"), n=3)
    assert torch.allclose(r.scores, torch.full((1, 3), -math.log(V), device="cuda"), atol=4e-6)
    assert torch.equal(r.tokens[0], torch.arange(3, device="cuda"))
    # everything dead, everything finished
    r = beam_step(torch.randn((3, 9), device="cuda"), torch.full((1, 3), -inf, device="cuda"), n=5)
    assert torch.equal(r.tokens[0], torch.arange(5, device="cuda")) and bool((r.scores == -inf).all())
    fin = torch.ones((1, 3), dtype=torch.bool, device="cuda")
    r = beam_step(torch.randn((3, 9), device="cuda"), torch.tensor([[-3.0, -1.0, -2.0]], device="cuda"), n=4, finished=fin, eos_id=6)
    assert r.tokens[0, :3].tolist() == [6, 6, 6] and r.rows[0].tolist() == [1, 2, 0, 0]
    assert r.scores[0].tolist() == [-1.0, -2.0, -3.0, -inf] and r.tokens[0, 3] == 0 and bool(r.finished.all())


def test_beam_strides_and_streams():
    from atomic_gdn2.generation import beam_step
    gen = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.randn((6, 5003), device="cuda", generator=gen)
    scores = -torch.rand((2, 3), device="cuda", generator=gen)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        w = wide.to(dtype)
        for x in (w[:, :4000], w[:, 1:4002], w[:, 8:], w.t().contiguous().t(), w[:1].expand(6, 5003), w[:, ::2]):
            want = beam_step(x.contiguous().clone(), scores, n=7)
            got = beam_step(x, scores, n=7)
            assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))
            _check_beam(got, x, scores, 7)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = beam_step(wide, scores, n=7)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got[:3], beam_step(wide, scores, n=7)[:3]))


def test_beam_graph_replay():
    from atomic_gdn2.generation import beam_step
    gen = torch.Generator(device="cuda").manual_seed(3)
    xs = [torch.randn((8, 9001), device="cuda", generator=gen) * 2 for _ in range(4)]
    scores = -torch.rand((2, 4), device="cuda", generator=gen)
    buf = xs[0].clone()
    beam_step(buf, scores, n=8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam_step(buf, scores, n=8)
    for x in xs:
        buf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = beam_step(x, scores, n=8)
        assert all(torch.equal(a, b) for a, b in zip(out[:3], want[:3]))


def test_beam_refusals():
    from atomic_gdn2.generation import beam_step
    x, s = torch.randn((4, 10), device="cuda"), torch.zeros((1, 4), device="cuda")
    for kw, err in ((dict(n=0), "n=0"), (dict(n=41), "n=41"), (dict(n=129), "n=129"), (dict(eos_id=10), "eos_id"),
                    (dict(finished=torch.zeros((1, 4), device="cuda")), "eos_id"),
                    (dict(finished=torch.zeros((4,), device="cuda"), eos_id=1), "finished must be")):
        with pytest.raises(ValueError, match=err):
            beam_step(x, s, **kw)
    with pytest.raises(ValueError, match="logits must be"):
        beam_step(x[:3], s)
    with pytest.raises(ValueError, match="scores must be"):
        beam_step(x, s[0])
    with pytest.raises(TypeError, match="logits"):
        beam_step(x.double(), s)
    with pytest.raises(ValueError, match="is on cpu"):
        beam_step(x, s.cpu())


# ---------------------------------------------------------------- decode_step(parents=...)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mode", ["fp32", "bf16", "bf16_state", "cap", "fused", "reset"])
def test_decode_from_parents_is_decode_of_gathered_states(D, mode):
    from atomic_gdn2.inference import decode_step
    print(f"[gpu-test] decode parents D {D} {mode}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(D)
    R, S, H = 7, 5, 3
    xs = [torch.randn((R, H, D), device="cuda", generator=gen) * 0.3 for _ in range(6)]
    st = torch.randn((S, H, D, D), device="cuda", generator=gen) * 0.2
    kw = {}
    if mode == "bf16":
        xs, st = [x.bfloat16() for x in xs], st
    if mode in ("bf16", "bf16_state"):
        kw["state_dtype"], st = torch.bfloat16, st.bfloat16()
    if mode == "cap":
        kw["stability_tau"] = 1.5
    if mode == "fused":
        kw.update(fuse_prologue=True, a_log=torch.randn(H, device="cuda", generator=gen) * 0.3,
                  dt_bias=torch.randn(D, device="cuda", generator=gen) * 0.3)
    if mode == "reset":
        kw["reset"] = torch.tensor([0, 1, 0, 0, 0, 1, 0], device="cuda")
    par = torch.tensor([4, 0, 0, 2, 2, 1, 4], device="cuda")
    o, h = decode_step(*xs, st, 0.1, parents=par, **kw)
    ro, rh = decode_step(*xs, st[par].contiguous(), 0.1, **kw)
    assert torch.equal(o, ro) and torch.equal(h, rh)
    twice = torch.stack([par, par], 1)
    for p in (par.int(), par.to(torch.int16), twice[:, 0]):      # other types and strides
        o2, h2 = decode_step(*xs, st, 0.1, parents=p, **kw)
        assert torch.equal(o, o2) and torch.equal(h, h2)
    # rows outside the states start from zero
    par2 = torch.tensor([4, -1, 0, 5, 2, 2 ** 40, 4], device="cuda")
    o, h = decode_step(*xs, st, 0.1, parents=par2, **kw)
    full = torch.cat([st, torch.zeros_like(st[:1])])
    ro, rh = decode_step(*xs, full[torch.tensor([4, 5, 0, 5, 2, 5, 4], device="cuda")].contiguous(), 0.1, **kw)
    assert torch.equal(o, ro) and torch.equal(h, rh)


def test_decode_parents_refusals():
    from atomic_gdn2 import _lib
    from atomic_gdn2.inference import decode_step
    xs = [torch.randn((2, 1, 64), device="cuda") for _ in range(6)]
    st = torch.zeros((3, 1, 64, 64), device="cuda")
    with pytest.raises(ValueError, match="state must be"):
        decode_step(*xs, st)
    with pytest.raises(ValueError, match="parents must be"):
        decode_step(*xs, st, parents=torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError, match="whole numbers"):
        decode_step(*xs, st, parents=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError, match="is on cpu"):
        decode_step(*xs, st, parents=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="state to start from"):
        decode_step(*xs, st[:0], parents=torch.zeros(2, dtype=torch.int64, device="cuda"))
    # the C entry refuses a state that would be read after another row has written it
    import ctypes
    dd = _lib.Gdn2DecodeDesc(2, 1, 64, 1, 1, 0, 0, 0, 0, 0, 1.0, 0.0)
    par, o = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.empty((2, 1, 64), device="cuda")
    rc = _lib.lib().gdn2_decode_from(ctypes.byref(dd), 0, *(x.data_ptr() for x in xs), None, None, None, 2, par.data_ptr(), 3,
                                     st.data_ptr(), o.data_ptr(), st[1:].data_ptr(), None)
    assert rc == 1 and b"overlap" in _lib.lib().gdn2_last_error()


# ---------------------------------------------------------------- premix_step
def _premix_inputs(R, S, H, D, seed, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    C = H * D
    return (randn(R, 6 * C + H + pad), randn(S, 3, 3 * C), tuple(randn(C, 4) * 0.5 for _ in range(3)),
            tuple(randn(C) * 0.1 for _ in range(3)), tuple(randn(C) * 0.1 for _ in range(2)), randn(H) * 0.1, randn(H) * 0.5 - 1)


def _premix64(y, history, cw, cb, gb, db, da, H, g_max, parents):
    R, C = y.shape[0], history.shape[2] // 3
    y = y.double()
    S = history.shape[0]
    ok = (parents >= 0) & (parents < S)
    past = torch.where(ok[:, None, None], history.double()[parents.clamp(0, S - 1)], 0.0)
    win = torch.cat([past, y[:, None, :3 * C]], 1)
    out = {}
    for i, n in enumerate("qkv"):
        w = win[:, :, i * C:(i + 1) * C]
        u = torch.nn.functional.silu((w * cw[i].double().t()).sum(1) + cb[i].double()).reshape(R, H, -1)
        out[n] = u.clamp(-50, 50) if n == "v" else u * torch.rsqrt((u * u).sum(-1, keepdim=True) + 1e-6)
    for i, n in enumerate("bw"):
        out[n] = torch.sigmoid(y[:, (3 + i) * C:(4 + i) * C] + gb[i].double()).reshape(R, H, -1)
    d = torch.exp(da.double().clamp(-20, 20)) * torch.nn.functional.softplus(y[:, 6 * C:6 * C + H] + db.double())
    out["g"] = -d.clamp(max=g_max)[..., None].expand(R, H, C // H)
    out["gate"], out["history"] = y[:, 5 * C:6 * C], win[:, 1:]
    return out


@pytest.mark.parametrize("R,S,H,D", [(1, 1, 1, 64), (4, 4, 6, 128), (5, 2, 3, 64), (64, 70, 2, 128)])
def test_premix_step_matches_the_definition(R, S, H, D):
    """Bound: chains of about ten float32 operations on values of order one, 2e-6 of the largest entry of
    a head; the logits and the history are copies."""
    from atomic_gdn2.generation import premix_step
    print(f"[gpu-test] premix step {R} {S} {H} {D}", flush=True)
    y, hist, *ps = _premix_inputs(R, S, H, D, R + S, pad=R % 3)
    gen = torch.Generator(device="cuda").manual_seed(9)
    par = torch.randint(-1, S + 1, (R,), device="cuda", generator=gen)
    r = premix_step(y, hist, *ps, n_heads=H, g_max=1.25, parents=par)
    want = _premix64(y, hist, *ps, H, 1.25, par)
    for n in want:
        got, ref = getattr(r, n).double(), want[n]
        assert got.shape == ref.shape
        if n in ("gate", "history"):
            assert torch.equal(got, ref)
        else:
            assert bool(((got - ref).abs() <= 2e-6 * ref.abs().amax(-1, keepdim=True)).all()), n
    again = premix_step(y, hist, *ps, n_heads=H, g_max=1.25, parents=par.int())
    assert all(torch.equal(a, b) for a, b in zip(r, again))
    if R == S:
        own = premix_step(y, hist, *ps, n_heads=H, g_max=1.25)
        idx = premix_step(y, hist, *ps, n_heads=H, g_max=1.25, parents=torch.arange(R, device="cuda"))
        assert all(torch.equal(a, b) for a, b in zip(own, idx))


def test_premix_steps_are_the_blocks_premix():
    """Token by token from an empty history: the outputs of the block's own pass over the sequence."""
    import ctypes

    from atomic_gdn2 import _lib, lm_kernels
    from atomic_gdn2.generation import premix_step
    B, L, H, D = 2, 9, 2, 64
    C = H * D
    y, _, cw, cb, gb, db, da = _premix_inputs(B * L, 1, H, D, 4, pad=2)
    outs = [torch.empty((B, H, L, D), device="cuda") for _ in range(6)]
    og = torch.empty((B * L, C), device="cuda")
    at = lambda ts: (lm_kernels._vp * len(ts))(*(t.data_ptr() for t in ts))  # noqa: E731
    a = lm_kernels._PremixArgs(B, L, H, D, y.shape[1], 1.25, y.data_ptr(), at(cw), at(cb), at(gb), db.data_ptr(),
                               da.data_ptr(), at(outs), og.data_ptr())
    _lib.check(_lib.lib().gdn2_lm_premix_fwd(ctypes.byref(a), _lib.stream_handle()), "premix")
    hist = torch.zeros((B, 3, 3 * C), device="cuda")
    y3 = y.view(B, L, -1)
    for t in range(L):
        r = premix_step(y3[:, t], hist, cw, cb, gb, db, da, n_heads=H, g_max=1.25)
        hist = r.history
        for n, o in zip("qkvwbg", outs):
            assert torch.allclose(getattr(r, n), o[:, :, t], rtol=2e-6, atol=1e-6), (n, t)
        assert torch.equal(r.gate, og.view(B, L, C)[:, t])
    assert torch.equal(hist, y3[:, L - 3:, :3 * C])


def test_premix_step_refusals():
    from atomic_gdn2.generation import premix_step
    y, hist, *ps = _premix_inputs(3, 2, 1, 64, 0)
    go = lambda y=y, hist=hist, ps=ps, **kw: premix_step(y, hist, *ps, **{"n_heads": 1, "g_max": 1.0, **kw})  # noqa: E731
    par = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="without parents"):
        go()
    with pytest.raises(ValueError, match="parents must be"):
        go(parents=par[:2])
    with pytest.raises(TypeError, match="whole numbers"):
        go(parents=par.float())
    with pytest.raises(ValueError, match="D=32"):
        go(n_heads=2, parents=par)
    with pytest.raises(ValueError, match="columns"):
        go(y=y[:, :-1], parents=par)
    with pytest.raises(TypeError, match="float32"):
        go(y=y.double(), parents=par)
    with pytest.raises(ValueError, match="decay_b must be"):
        go(ps=ps[:3] + [ps[3][:0]] + ps[4:], parents=par)
    with pytest.raises(ValueError, match="is on cpu"):
        go(parents=par.cpu())


# ---------------------------------------------------------------- the LM
def _small_lm(seed=0, **kw):
    from atomic_gdn2 import e2e_lm
    cfg = e2e_lm.LMConfig(**{**dict(vocab_size=61, d_model=128, n_heads=2, d_head=64, n_layers=2), **kw})
    model = e2e_lm.make_lm(cfg, seed=seed)
    with torch.no_grad():       # logits that are not all alike, gates and biases that are not all zero
        gen = torch.Generator().manual_seed(seed + 1)
        model.embed.mul_(4.0)
        for n, p in model.named_parameters():
            if n.endswith(("bias", "decay_a")) or "conv" in n:
                p.add_(torch.randn(p.shape, generator=gen).to(p) * 0.3)
    return model


def _lm64(model, group):
    """The LM of the rounded weights in float64 on the CPU, its recurrence token by token."""
    from atomic_gdn2 import e2e_lm
    from atomic_gdn2.w4 import quantize_w4

    def rounded(*ws):
        full = quantize_w4(torch.cat([w.detach() for w in ws], 1), group).dequantize().double().cpu()
        return full.split([w.shape[1] for w in ws], 1)

    def mixer(q, k, v, w, b, g):                       # (B, L, H, D)
        B, L, H, D = q.shape
        h, os_ = torch.zeros((B, H, D, D), dtype=q.dtype), []
        for t in range(L):
            h = h * torch.exp(g[:, t])[..., None]
            new = w[:, t] * v[:, t] - ((b[:, t] * k[:, t])[..., None] * h).sum(-2)
            h = h + k[:, t][..., None] * new[..., None, :]
            os_.append((h * q[:, t][..., None]).sum(-2) * D ** -0.5)
        return torch.stack(os_, 1)

    c = model.cfg
    ref = e2e_lm.LM(c, mixer).double()
    ref.load_state_dict({n: p.double().cpu() for n, p in model.state_dict().items()})
    pad = torch.zeros((c.d_model, -(6 * c.proj_dim + c.n_heads) % 4), device="cuda")
    with torch.no_grad():
        for b, r in zip(model.blocks, ref.blocks):
            names = ("q_proj", "k_proj", "v_proj", "erase_gate", "write_gate", "out_gate", "decay_proj")
            for n, w in zip(names, rounded(*(getattr(b, n).weight for n in names), pad)):
                getattr(r, n).weight.copy_(w)
            for names in (("out_proj",), ("gate_proj", "up_proj"), ("down_proj",)):
                for n, w in zip(names, rounded(*(getattr(b, n).weight for n in names))):
                    getattr(r, n).weight.copy_(w)
    head = rounded(model.embed.t())[0]

    def logits(ids):
        x = ref.embed[ids]
        for blk in ref.blocks:
            x = blk(x)
        return (ref.final_norm(x) @ head).detach()
    return logits


@pytest.mark.parametrize("L", [1, 2, 5, 64, 70])
def test_prefill_and_steps_are_the_language_model(L):
    """Logits of a prompt and of the tokens after it, from caches, against the whole sequence at once.
    Bound: float32 through two blocks, 2e-4 of the largest logit (the operator's own gate is 2e-3)."""
    from atomic_gdn2.generation import Generator
    model = _small_lm()
    gen, ref = Generator(model, group_size=32), _lm64(model, 32)
    ids = torch.randint(0, 61, (3, L + 6), generator=torch.Generator().manual_seed(L))
    want = ref(ids)
    logits, cache = gen.prefill(ids[:, :L].cuda())
    tol = 2e-4 * float(want.abs().max())
    assert float((logits.cpu().double() - want[:, L - 1]).abs().max()) <= tol
    order = torch.tensor([0, 1, 2])
    for t in range(L, L + 6):
        perm = torch.randperm(3, generator=torch.Generator().manual_seed(t))         # rows change their places
        order = order[perm]
        logits, cache = gen.step(ids[order, t].cuda(), cache, perm.cuda())
        assert float((logits.cpu().double() - want[order, t]).abs().max()) <= tol, t


@pytest.mark.parametrize("eos", [None, 7])
def test_beam_search_is_the_search_over_whole_sequences(eos):
    """Against a search that scores every continuation of every beam by the whole sequence in float64."""
    from atomic_gdn2.generation import Generator
    model = _small_lm(seed=3)
    gen, ref = Generator(model, group_size=32), _lm64(model, 32)
    B, L, n, T, V = 2, 9, 3, 12, 61
    ids = torch.randint(0, V, (B, L), generator=torch.Generator().manual_seed(11))
    r = gen.beam_search(ids.cuda(), n, T, eos_id=eos)
    assert r.tokens.shape == (B, n, T) and r.scores.shape == (B, n)
    for b in range(B):
        beams = [((), 0.0, False)]
        gap = math.inf
        for _ in range(T):
            cand = []
            for seq, score, done in beams:
                if done:
                    cand.append((score, seq + (eos,), True))
                    continue
                lp = torch.log_softmax(ref(torch.cat([ids[b], torch.tensor(seq, dtype=torch.long)])[None])[0, -1], -1)
                cand += [(score + float(lp[v]), seq + (v,), eos is not None and v == eos) for v in range(V)]
            cand.sort(key=lambda c: -c[0])
            gap = min([gap] + [x[0] - y[0] for x, y in zip(cand[:n], cand[1:n + 1])])
            beams = [(seq, score, done) for score, seq, done in cand[:n]]
        print(f"[gpu-test] smallest gap between candidates {gap:.2g}", flush=True)
        assert gap > 1e-4, "choose another seed: the reference's own order is in doubt"
        assert [tuple(x) for x in r.tokens[b].tolist()] == [s for s, _, _ in beams]
        assert torch.allclose(r.scores[b].cpu().double(), torch.tensor([s for _, s, _ in beams], dtype=torch.float64), atol=2e-3)
    if eos is not None:
        ended = (r.tokens == eos).cummax(-1).values
        assert bool(((r.tokens == eos) == ended).all())


@pytest.mark.parametrize("eos", [None, 7])
def test_beam_search_by_graph_replays_gives_the_same(eos):
    """Every replay works on the caches that the one before left; the searches run eager work and
    synchronise between them."""
    from atomic_gdn2.generation import Generator
    gen = Generator(_small_lm(seed=3), group_size=32)
    for seed, (B, n, T) in enumerate(((2, 3, 30), (1, 1, 5), (3, 4, 2), (2, 8, 20))):
        ids = torch.randint(0, 61, (B, 9), generator=torch.Generator().manual_seed(seed)).cuda()
        a = gen.beam_search(ids, n, T, eos_id=eos, graph=True)
        torch.cuda.synchronize()
        b = gen.beam_search(ids, n, T, eos_id=eos, graph=False)
        assert torch.equal(a.tokens, b.tokens) and torch.equal(a.scores, b.scores)


def test_generator_refusals():
    from atomic_gdn2.generation import Generator
    with pytest.raises(ValueError, match="d_head"):
        Generator(_small_lm(d_head=32))
    with pytest.raises(ValueError, match="ROCm device"):
        Generator(_small_lm().cpu())
    gen = Generator(_small_lm())
    ids = torch.zeros((1, 4), dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="token ids"):
        gen.prefill(ids[0])
    with pytest.raises(ValueError, match="token ids"):
        gen.prefill(ids[:, :0])
    with pytest.raises(ValueError, match="token ids are on cpu"):
        gen.prefill(ids.cpu())
    with pytest.raises(ValueError, match="max_new_tokens"):
        gen.beam_search(ids, 2, 0)
