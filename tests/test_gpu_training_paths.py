"""The native call paths of linear, cross_entropy and AdamW against the Python paths they stand for (the same bits), and
calls that overlap on two streams."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


def _python_only(monkeypatch):
    from atomic_gdn2 import _lib
    no = lambda *a: None  # noqa: E731
    monkeypatch.setattr(_lib, "bind", lambda: types.SimpleNamespace(linear=no, cross_entropy=no, adamw=no, adamw_unpack=no))


def _linear(dt, act, M):
    from atomic_gdn2.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(M)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(dt).requires_grad_(True)  # noqa: E731
    out = []
    for turned in (False, True):
        x, b, res, dy = r(2, M, 200), r(264), r(2, M, 264), r(2, M, 264).detach()
        w = r(264, 200) if turned else r(200, 264)
        y = linear(x, w.t() if turned else w, bias=b, residual=res, activation=act)
        out += [y.detach(), *torch.autograd.grad(y, (x, w, b, res), dy, retain_graph=True)]
        out += [*torch.autograd.grad(y, (b,), dy, retain_graph=True), *torch.autograd.grad(y, (res,), dy, retain_graph=True),
                *torch.autograd.grad(y, (w,), dy)]
        with torch.no_grad():
            out.append(linear(x, w.t() if turned else w, residual=res))
    return out


def _loss(dt, reduction):
    from atomic_gdn2.losses import cross_entropy
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((4, 9, 777), device="cuda", generator=gen).to(dt).requires_grad_(True)
    t = torch.randint(-1, 777, (4, 9), device="cuda", generator=gen)
    loss = cross_entropy(x, t, ignore_index=-1, label_smoothing=0.1, z_loss=1e-3, reduction=reduction)
    f = torch.full_like(loss, 0.3)
    return [loss.detach(), torch.autograd.grad(loss, x, f, retain_graph=True)[0], torch.autograd.grad(loss, x, f)[0]]


def _steps(dt, bits):
    from atomic_gdn2.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(4)
    ps = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen).to(dt)) for n in (5, 256, 3001)]
    opt = AdamW([{"params": ps[:1], "lr": 0.1}, {"params": ps[1:]}], max_norm=0.7, state_bits=bits)
    out = []
    for _ in range(3):
        for p in ps:
            p.grad = torch.randn(p.shape, device="cuda", generator=gen).to(dt)
        opt.step()
        out.append(opt.norm)
    if bits == 8:
        for ts in opt.unpack_states([torch.empty(p.shape, device="cuda") for p in ps], [torch.empty(p.shape, device="cuda") for p in ps]):
            out += ts
    return out + [p.detach() for p in ps] + [t for p in ps for t in opt.state[p].values()]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_same_bits_as_python(monkeypatch, dtype):
    run = lambda: (_linear(dtype, None, 3) + _linear(dtype, "gelu", 70) + _loss(dtype, "mean") + _loss(dtype, "none")  # noqa: E731
                   + _steps(dtype, 32) + _steps(dtype, 8))
    got = run()
    _python_only(monkeypatch)
    want = run()
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b), i


def test_two_streams_at_once():
    """Products in parts and losses whose workspaces would meet if calls shared one."""
    from atomic_gdn2.linear import linear
    from atomic_gdn2.losses import cross_entropy
    xs = [torch.randn(100, 4096, device="cuda").bfloat16() for _ in range(2)]
    ws = [torch.randn(4096, 200, device="cuda").bfloat16() for _ in range(2)]
    ts = [torch.randint(0, 200, (100,), device="cuda") for _ in range(2)]
    run = lambda i: [(y := linear(xs[i], ws[i], out_dtype=torch.float32)), cross_entropy(y, ts[i])]  # noqa: E731
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert torch.equal(r[0], want[i][0]) and torch.equal(r[1], want[i][1])


def test_two_graphs_of_one_model():
    """Graphs captured after one another, replayed in turn with eager calls between them."""
    from atomic_gdn2.linear import linear
    w = torch.randn(2048, 264, device="cuda").bfloat16()
    xs, outs, graphs = [torch.randn(n, 2048, device="cuda").bfloat16() for n in (40, 90)], [], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for x in xs:
            linear(x, w)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(linear(x, w, activation="silu"))
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(s)
    for k in range(3):
        for x in xs:
            x.copy_(torch.randn(x.shape))
        want = [linear(x, w, activation="silu") for x in xs]
        for g in graphs:
            g.replay()
        linear(xs[0], w)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), k
