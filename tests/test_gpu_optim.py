"""AdamW over many tensors: against the definition in 64 bits and, bit by bit, against the same steps in torch
operations of 32 bits (products and sums rounded one by one, as the kernels round them)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
B1, B2, EPS, LR, WD = 0.9, 0.99, 1e-8, 1e-2, 0.1


def _dither(n, ordinal, step):
    low = 0xFFFFFFFF
    x = (torch.arange(n, device="cuda") * 0x9E3779B1 + ordinal * 0x7F4A7C15 + step * 0x6C62272F) & low
    x = ((x ^ (x >> 16)) * 0x5D8AF3B5) & low
    x = ((x ^ (x >> 15)) * 0x2F6B4E1D) & low
    x = x ^ (x >> 16)
    return ((x & 0xFFFF).float() + 0.5) / 65536, ((x >> 16).float() + 0.5) / 65536


class Plain:
    """One tensor's state and step in torch operations."""

    def __init__(self, p, bits, ordinal):
        self.w, self.dt, self.bits, self.ordinal, self.t = p.detach().float().clone().view(-1), p.dtype, bits, ordinal, 0
        self.m, self.v = torch.zeros_like(self.w), torch.zeros_like(self.w)

    def step(self, g, c=1.0):
        self.t += 1
        g = g.float().view(-1) * torch.tensor(c, dtype=torch.float32)
        self.m = self.m * B1 + g * (1 - B1)
        self.v = self.v * B2 + (g * g) * (1 - B2)
        root, size = 1 / math.sqrt(1 - B2 ** self.t), LR / (1 - B1 ** self.t)
        self.w = self.w * (1 - LR * WD) - (self.m / (torch.sqrt(self.v) * root + EPS)) * size
        if self.bits == 8:
            self.m, self.v = self.round(self.m, self.v)
        return self.w.to(self.dt)

    def round(self, m, v):
        n = m.numel()
        r_m, r_v = _dither(n, self.ordinal, self.t)
        blocks = -(-n // 256)
        pad = lambda x: torch.nn.functional.pad(x, (0, blocks * 256 - n)).view(blocks, 256)  # noqa: E731
        m, v, r_m, r_v = pad(m), pad(v), pad(r_m), pad(r_v)
        ok = torch.isfinite(m).all(1, keepdim=True), torch.isfinite(v).all(1, keepdim=True)
        self.s_m = torch.where(ok[0], m.abs().amax(1, keepdim=True) * (1.0 / 16129), torch.nan)
        self.s_v = torch.where(ok[1], torch.sqrt(v.amax(1, keepdim=True)) * (1.0 / 65025), torch.nan)

        def code(x, root, s, top, value, r):
            unit = s > 0
            c = torch.sqrt(root / torch.where(unit, s, 1.0)).floor().clamp(max=top - 1)
            lo, hi = value(c), value(c + 1)
            return torch.where(unit, torch.where(x - lo > r * (hi - lo), c + 1, c), 0.0)

        c = torch.sign(m) * code(m.abs(), m.abs(), self.s_m, 127, lambda c: c * c * self.s_m, r_m)
        u = code(v, torch.sqrt(v), self.s_v, 255, lambda u: (u * u * self.s_v).square(), r_v)
        u = torch.where((v > 0) & (self.s_v > 0), u.clamp(min=1), u)
        c = torch.where(self.s_m > 0, c, 0.0)
        self.c, self.u = c.view(-1)[:n], u.view(-1)[:n]
        return (c * c.abs() * self.s_m).view(-1)[:n], (u * u * self.s_v).square().view(-1)[:n]


def _params(sizes, dt, seed=0, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for n in sizes:
        n = n if isinstance(n, tuple) else (n,)
        flat = torch.randn(math.prod(n) + offset, device="cuda", generator=gen).to(dt)
        out.append(torch.nn.Parameter(flat[offset:].view(n)))
    return out


def _grads(ps, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(p.shape, device="cuda", generator=gen) * scale * math.exp(i % 5 - 2)).to(p.dtype) for i, p in enumerate(ps)]


def _opt(ps, **kw):
    from atomic_gdn2.optim import AdamW
    return AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, **kw)


SIZES = [1, 3, 255, 256, 257, (5, 7), 8191, 8192, 8193, (130, 129), 70001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
def test_same_bits_as_torch_operations(dtype, bits, offset):
    dt = DTYPES[dtype]
    ps = _params(SIZES, dt, offset=offset)
    plain = [Plain(p, bits, i) for i, p in enumerate(ps)]
    opt = _opt(ps, state_bits=bits)
    for step in range(4):
        for p, g in zip(ps, _grads(ps, 10 + step)):
            p.grad = g
        opt.step()
        values = opt.unpack_states() if bits == 8 else None
        for i, (p, q) in enumerate(zip(ps, plain)):
            want = q.step(p.grad)
            s = opt.state[p]
            assert torch.equal(p.detach().view(-1), want), (step, i)
            assert s["step"].item() == step + 1
            if dt != torch.float32:
                assert torch.equal(s["master"].view(-1), q.w)
            m, v = (s["exp_avg"], s["exp_avg_sq"]) if bits == 32 else (values[0][i], values[1][i])
            assert torch.equal(m.view(-1), q.m) and torch.equal(v.view(-1), q.v), (step, i)
            if bits == 8:
                assert torch.equal(s["exp_avg"].view(-1).float(), q.c) and torch.equal(s["exp_avg_sq"].view(-1).float(), q.u)


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_over_mixed_types_and_many_tensors(bits):
    """More tensors than an argument block holds, of three types, clipped by one norm."""
    ps = []
    for i in range(230):
        ps += _params([1 + 37 * i % 900], list(DTYPES.values())[i % 3], seed=i)
    plain = [Plain(p, bits, i) for i, p in enumerate(ps)]
    opt = _opt(ps, state_bits=bits, max_norm=0.5)
    for step in range(3):
        for p, g in zip(ps, _grads(ps, 20 + step, scale=1e-4 if step == 1 else 1.0)):
            p.grad = g
        opt.step()
        norm = math.sqrt(sum(p.grad.double().square().sum().item() for p in ps))
        assert abs(opt.norm.item() - norm) <= 2.0 ** -23 * norm and (norm > 0.5) == (step != 1)
        c = torch.tensor(0.5 / max(norm, 0.5), dtype=torch.float64).float().item()
        for i, (p, q) in enumerate(zip(ps, plain)):
            assert torch.equal(p.detach().view(-1), q.step(p.grad, c)), (step, i)


@pytest.mark.parametrize("dtype", DTYPES)
def test_against_the_definition_in_64_bits(dtype):
    """Five roundings of 2^-24 each in m, v and what is taken from p; the 16-bit p is its master, rounded."""
    dt = DTYPES[dtype]
    p, = _params([5000], dt, seed=3)
    opt = _opt([p], max_norm=1.0)
    w, m, v = p.detach().double(), torch.zeros(5000, dtype=torch.float64, device="cuda"), torch.zeros(5000, dtype=torch.float64, device="cuda")
    for t in range(1, 5):
        p.grad, = _grads([p], t)
        g = p.grad.double()
        g = g * min(1.0, 1.0 / g.norm().item())
        opt.step()
        m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
        w = w * (1 - LR * WD) - LR / (1 - B1 ** t) * m / (torch.sqrt(v / (1 - B2 ** t)) + EPS)
    s = opt.state[p]
    got = s["master"] if dt != torch.float32 else p.detach()
    e = 2.0 ** -24
    # (m is a difference where gradients change sign: 4 steps' roundings of its largest terms)
    assert ((s["exp_avg"].double() - m).abs() <= 4 * 6 * e * (1 - B1) * 4 * g.abs().max()).all()
    assert ((s["exp_avg_sq"].double() - v).abs() <= 4 * 8 * e * v + 1e-40).all()
    assert ((got.double() - w).abs() <= 4 * (3 * e * w.abs() + 1e-6 * LR * 4)).all()
    if dt != torch.float32:
        assert torch.equal(p.detach(), got.to(dt))


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_gradient_and_groups(bits):
    """Steps are counted for each tensor; groups have their own lr; a tensor without gradient is left as it is."""
    from atomic_gdn2.optim import AdamW
    a, b, c = _params([300, 40, 500], torch.float32, seed=5)
    opt = AdamW([{"params": [a, b]}, {"params": [c], "lr": 0.0, "weight_decay": 0.5}], lr=LR, state_bits=bits)
    before = b.detach().clone(), c.detach().clone()
    a.grad, c.grad = torch.randn_like(a), torch.randn_like(c)
    opt.step()
    assert torch.equal(b.detach(), before[0]) and not opt.state[b] and torch.equal(c.detach(), before[1])
    b.grad = torch.randn_like(b)
    opt.step()
    assert opt.state[a]["step"].item() == 2 and opt.state[b]["step"].item() == 1
    opt.zero_grad()
    assert opt.step() is None and opt.step(lambda: 3.0) == 3.0


def test_eight_bits_keep_the_mean_and_decay():
    """Over many steps of no gradient v decays as b2^t in the mean, which nearest rounding would stop, and a state's
    expectation is the value rounded: for 20000 elements within six deviations of a code's distance."""
    from atomic_gdn2.optim import AdamW
    n, steps = 256 * 80, 100
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.999), state_bits=8)
    p.grad = torch.randn(n, device="cuda")
    opt.step()
    v0 = opt.unpack_states()[1][0].double()
    p.grad = torch.zeros(n, device="cuda")
    for _ in range(steps):
        opt.step()
    v = opt.unpack_states()[1][0].double()
    # a value's codes lie 4 / c of it apart; most of the sum has c above 60
    want = 0.999 ** steps * v0.sum()
    spread = (v0 * 4 / 60).square().sum().sqrt() * math.sqrt(steps)
    assert abs(v.sum() - want) < 6 * spread and v.sum() < 0.96 * v0.sum()
    assert ((v > 0) == (v0 > 0)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_nan_and_infinity_stay_where_they_are(bits):
    ps = _params([2000, 700], torch.float32, seed=6)
    opt = _opt(ps, state_bits=bits)
    for p in ps:
        p.grad = torch.randn_like(p)
    ps[0].grad[600], ps[0].grad[1999] = float("nan"), float("inf")
    for _ in range(2):
        opt.step()
    bad = ~torch.isfinite(ps[0].detach())
    want = torch.zeros(2000, dtype=torch.bool, device="cuda")
    for i in (600, 1999):
        want[slice(i // 256 * 256, min(2000, i // 256 * 256 + 256)) if bits == 8 else i] = True
    assert torch.equal(bad, want) and torch.isfinite(ps[1].detach()).all()
    opt = _opt(ps[1:], state_bits=bits, max_norm=1.0)
    ps[1].grad[3] = float("nan")
    opt.step()
    assert torch.isnan(opt.norm) and torch.isnan(ps[1].detach()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(dtype, bits):
    import io
    dt = DTYPES[dtype]
    ps, qs = _params([700, (20, 30)], dt, seed=7), _params([700, (20, 30)], dt, seed=7)
    one, two = _opt(ps, state_bits=bits, max_norm=1.0), _opt(qs, state_bits=bits, max_norm=1.0)
    for k in range(2):
        for p, g in zip(ps, _grads(ps, k)):
            p.grad = g
        one.step()
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    f = io.BytesIO()
    torch.save(one.state_dict(), f)
    f.seek(0)
    two.load_state_dict(torch.load(f, weights_only=True))
    for p, q in zip(ps, qs):
        for k, t in one.state[p].items():
            assert two.state[q][k].dtype == t.dtype and torch.equal(two.state[q][k], t), k
    for p, q, g in zip(ps, qs, _grads(ps, 9)):
        p.grad, q.grad = g, g.clone()
    one.step(), two.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_states_of_torch_are_taken_over():
    ps, qs = _params([300, 40], torch.float32, seed=8), _params([300, 40], torch.float32, seed=8)
    ref = torch.optim.AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    opt = _opt(qs)
    for k in range(3):
        for p, q, g in zip(ps, qs, _grads(ps, k)):
            p.grad, q.grad = g, g.clone()
        ref.step()
        if k == 0:
            opt.load_state_dict(ref.state_dict())
            with torch.no_grad():
                [q.copy_(p) for p, q in zip(ps, qs)]
        else:
            opt.step()
    assert all(torch.allclose(p, q, rtol=1e-5, atol=1e-6) for p, q in zip(ps, qs))
    with pytest.raises(ValueError, match="exp_avg"):
        _opt(qs, state_bits=8).load_state_dict(ref.state_dict())


def test_autograd_notices_the_update():
    p, = _params([20], torch.float32)
    y = (p * p).sum()
    opt = _opt([p])
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError):
        y.backward()


def test_strided_gradients_and_scheduler():
    ps = _params([(30, 40)], torch.float32, seed=9)
    plain = Plain(ps[0], 32, 0)
    opt = _opt(ps)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 1.0)
    ps[0].grad = torch.randn(40, 30, device="cuda").t()
    opt.step()
    sched.step()
    assert torch.equal(ps[0].detach().view(-1), plain.step(ps[0].grad.contiguous()))
    ps[0].grad = torch.ones(1, device="cuda").expand(30, 40)
    opt.step()
    assert torch.equal(ps[0].detach().view(-1), plain.step(ps[0].grad.contiguous()))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    ps, qs = _params([900, 5000], torch.bfloat16, seed=10), _params([900, 5000], torch.bfloat16, seed=10)
    one, two = _opt(ps, state_bits=bits, max_norm=1.0), _opt(qs, state_bits=bits, max_norm=1.0)
    for p, q, g in zip(ps, qs, _grads(ps, 0)):
        p.grad, q.grad = g, g.clone()
    one.step(), two.step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        two.step()
    torch.cuda.current_stream().wait_stream(s)
    for k in range(4):
        for p, q, g in zip(ps, qs, _grads(ps, 1 + k)):
            p.grad.copy_(g)
            q.grad.copy_(g)
        one.step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and torch.equal(one.norm, two.norm), k
        assert all(torch.equal(one.state[p]["exp_avg"], two.state[q]["exp_avg"]) for p, q in zip(ps, qs))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_values_written_into_a_parameter_count(dtype, bits):
    """A checkpoint loaded into the model between steps is what the next step updates, its master with it."""
    p, = _params([1000], DTYPES[dtype], seed=11)
    opt, plain = _opt([p], state_bits=bits), Plain(p, bits, 0)
    for k in range(3):
        p.grad, = _grads([p], k)
        if k == 1:
            p.data.copy_(torch.linspace(-2, 2, 1000, device="cuda"))
            keep = torch.arange(1000, device="cuda") % 3 == 0           # (and some that stay as they were)
            p.data[keep] = plain.w.to(p.dtype)[keep]
            plain.w = torch.where(plain.w.to(p.dtype) == p.detach(), plain.w, p.detach().float())
        opt.step()
        assert torch.equal(p.detach(), plain.step(p.grad)) and torch.equal(opt.state[p]["master"], plain.w), k


def test_norm_without_clipping():
    """max_norm inf: the norm is formed, nothing is scaled."""
    p, = _params([5000], torch.float32, seed=12)
    opt, plain = _opt([p], max_norm=math.inf), Plain(p, 32, 0)
    p.grad = torch.randn_like(p) * 100
    opt.step()
    assert torch.equal(p.detach(), plain.step(p.grad))
    assert abs(opt.norm.item() - p.grad.double().norm().item()) <= 2.0 ** -23 * opt.norm.item()


def test_copied_and_pickled():
    import copy
    import pickle
    p, = _params([300], torch.float32, seed=13)
    opt = _opt([p], state_bits=8, max_norm=2.0)
    p.grad = torch.randn_like(p)
    opt.step()
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        q = other.param_groups[0]["params"][0]
        q.grad = torch.ones_like(q)
        other.step()
        assert other.state_bits == 8 and other.max_norm == 2.0 and other.state[q]["step"].item() == 2
    assert opt.state[p]["step"].item() == 1


def test_unpacked_states_of_tensors_without_one_are_zero():
    ps = _params([300, 50], torch.float32, seed=14)
    opt = _opt(ps, state_bits=8)
    m, v = opt.unpack_states()
    assert not any(t.any() for t in (*m, *v))
    ps[1].grad = torch.randn_like(ps[1])
    opt.step()
    outs = [[torch.full_like(p, 7.0) for p in ps] for _ in range(2)]
    opt.unpack_states(*outs)
    assert not outs[0][0].any() and outs[0][1].any() and not outs[1][0].any() and outs[1][1].any()
    with pytest.raises(ValueError):
        opt.unpack_states([outs[0][0]], outs[1])
    with pytest.raises(ValueError):
        opt.unpack_states(outs[0], [t.half() for t in outs[1]])
    with pytest.raises(ValueError):
        _opt(ps).unpack_states()


def test_states_that_do_not_fit_are_refused():
    p, = _params([300], torch.float32, seed=15)
    for key, bad in (("exp_avg", torch.zeros(299, device="cuda")), ("exp_avg", torch.zeros(300, device="cuda").half()),
                     ("exp_avg_sq", torch.zeros(300)), ("step", torch.zeros(2, device="cuda")), ("exp_avg", torch.zeros(600, device="cuda")[::2])):
        opt = _opt([p])
        p.grad = torch.ones_like(p)
        opt.step()
        opt.state[p][key] = bad
        before = p.detach().clone()
        with pytest.raises(ValueError, match=key):
            opt.step()
        assert torch.equal(p.detach(), before)
    opt = _opt([p])
    opt.param_groups[0]["lr"] = torch.tensor(1e-3, device="cuda")
    with pytest.raises(TypeError, match="lr"):
        opt.step()
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError, match="lr"):
        opt.step()
