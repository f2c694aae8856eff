"""Products with bias, activation and residual, and their gradients, against the definition in 64 bits.

Bounds, element by element, u = half a step of the dtype (finfo.eps / 2):
  sum      an instruction adds 32 products to a float32: (K / 32 + 8) 2^-22 of the sum of the absolute products;
           float32 operands as pieces: 2^-22 of it again for the products of pieces that are left out;
  act      slopes are below 1.13 and second derivatives below 1.0; evaluated in float32: 2^-20 (|z| + 1);
  y        u |y| for the rounding;
  dz       z is kept rounded (u |z|, times the second derivative and |dy|) and dz is rounded (u |dz|).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = [None, "silu", "gelu", "gelu_tanh"]


def _act(z, act):
    F = torch.nn.functional
    return z if act is None else F.silu(z) if act == "silu" else F.gelu(z, approximate="tanh" if act == "gelu_tanh" else "none")


def _half(dt):
    return torch.finfo(dt).eps / 2


def _sum_bound(a, b):
    K = a.shape[1]
    return (K / 32 + 12) * 2.0 ** -22 * (a.abs() @ b.abs())


def _tiny(dt):
    """Half the distance of the dtype's smallest numbers."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def _close(got, want, bound, what):
    off = (got.double() - want).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert got.shape == want.shape and torch.isfinite(got).all() and worst <= 1.0, (what, worst, off.max().item())


def check(M, K, N, dt, act=None, bias=False, residual=False, grad=True, out_dtype=None, seed=0, make=None, bias_dtype=None):
    from atomic_gdn2.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    od = out_dtype or dt
    make = make or (lambda t: t)
    x, w = make(randn(M, K).to(dt)), make((randn(K, N) / K ** 0.5).to(dt))
    b = randn(N).to(bias_dtype or dt) if bias else None
    r = make(randn(M, N).to(od)) if residual else None
    dy = randn(M, N).to(od)
    leaves = [t for t in (x, w, b, r) if t is not None]
    if grad:
        leaves = [t.requires_grad_(True) for t in leaves]
    y = linear(x, w, bias=b, residual=r, activation=act, out_dtype=out_dtype)
    assert y.dtype == od and y.shape == (M, N) and y.is_contiguous()
    X, W = x.detach().double(), w.detach().double()
    z = (X @ W + (b.detach().double() if bias else 0.0)).requires_grad_(True)
    a = _act(z, act)
    Y = a.detach() + (r.detach().double() if residual else 0.0)
    eps = _sum_bound(X, W) + 2.0 ** -23 * (z.detach().abs() + (b.detach().double().abs() if bias else 0.0))
    err = 1.13 * eps + (2.0 ** -20 * (z.detach().abs() + 1) if act else 0.0) + 2.0 ** -23 * Y.abs()
    _close(y, Y, err + _half(od) * Y.abs() + _tiny(od), "y")
    if not grad:
        return
    grads = dict(zip([n for n, t in zip("xwbr", (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    slope, = torch.autograd.grad(a, z, torch.ones_like(z)) if act else (torch.ones_like(z),)
    dz = dy.double() * slope
    e_slope = (_half(dt) * z.detach().abs() + eps + 2.0 ** -19 * (z.detach().abs() + 1)) if act else 0.0
    e_dz = dy.double().abs() * e_slope + _half(dt) * (1 + _half(dt)) * dz.abs() + _tiny(dt)
    big = dz.abs() + e_dz
    for n, want, bound, t in (
            ("x", dz @ W.t(), e_dz @ W.abs().t() + _sum_bound(big, W.t()), x),
            ("w", X.t() @ dz, X.abs().t() @ e_dz + _sum_bound(X.abs().t(), big), w),
            ("b", dz.sum(0), (dy.double().abs() * e_slope).sum(0) + (M / 64 + 72) * 2.0 ** -23 * big.sum(0), b),
            ("r", dy.double(), 0.0, r)):
        if t is None:
            continue
        assert grads[n].dtype == t.dtype and grads[n].shape == t.shape
        _close(grads[n], want, bound + _half(t.dtype) * want.abs() + _tiny(t.dtype), "d" + n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 64, 8), (2, 7, 3), (3, 200, 130), (17, 33, 65), (128, 64, 128), (129, 72, 136),
                                   (130, 127, 257), (70, 40, 1), (66, 48, 62), (300, 40, 191), (77, 16, 127), (270, 33, 129), (300, 512, 264), (64, 1000, 777)])
def test_sizes(dtype, M, K, N):
    check(M, K, N, DTYPES[dtype], act="silu", bias=True, residual=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_epilogues(dtype, act, bias, residual):
    check(70, 96, 200, DTYPES[dtype], act=act, bias=bias, residual=residual, seed=1)
    check(5, 96, 72, DTYPES[dtype], act=act, bias=bias, residual=residual, seed=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 4096, 1024), (4, 2048, 4096), (9, 4100, 520), (16, 1024, 2048), (40, 8192, 256), (2048, 768, 512),
                                   (4096, 256, 128), (1000, 2000, 1500), (64, 64, 8192), (8, 9000, 515), (30, 2052, 4100), (33, 1100, 260)])
def test_large(dtype, M, K, N):
    check(M, K, N, DTYPES[dtype], act="gelu", bias=True, residual=True, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(5, 64, 48), (200, 264, 136)])
def test_strides_and_alignment(dtype, M, K, N):
    dt = DTYPES[dtype]

    def wider(t):                       # columns of a wider matrix, rows at odd places
        wide = torch.zeros((t.shape[0], t.shape[1] + 5), dtype=t.dtype, device=t.device)
        wide[:, 3:3 + t.shape[1]] = t
        return wide[:, 3:3 + t.shape[1]].detach()

    def wider8(t):                      # ... at whole 16 bytes
        wide = torch.zeros((t.shape[0], t.shape[1] + 16), dtype=t.dtype, device=t.device)
        wide[:, 8:8 + t.shape[1]] = t
        return wide[:, 8:8 + t.shape[1]].detach()

    def turned(t):                      # as a transposed view
        return t.t().contiguous().t().detach()

    for make in (wider, wider8, turned):
        check(M, K, N, dt, act="silu", bias=True, residual=True, make=make, seed=4)
        check(M, K, N, dt, make=make, seed=5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_float32_output_and_bias(dtype):
    dt = DTYPES[dtype]
    for M in (3, 150):
        check(M, 128, 96, dt, act="silu", bias=True, residual=True, out_dtype=torch.float32, bias_dtype=torch.float32)
        check(M, 128, 96, dt, bias=True, residual=True, out_dtype=torch.float32)


def test_leading_dimensions_and_empty_rows():
    from atomic_gdn2.linear import linear
    x = torch.randn(2, 3, 5, 64, device="cuda", requires_grad=True)
    w = torch.randn(64, 24, device="cuda", requires_grad=True)
    r = torch.randn(2, 3, 5, 24, device="cuda")
    y = linear(x, w, residual=r)
    assert y.shape == (2, 3, 5, 24)
    y.square().sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    b = torch.randn(24, device="cuda", requires_grad=True)
    w.grad = None
    y = linear(e, w, bias=b, activation="silu")
    assert y.shape == (0, 24)
    y.sum().backward()
    assert e.grad.shape == (0, 64) and not w.grad.any() and not b.grad.any()


def test_row_of_nans_touches_no_other_row():
    from atomic_gdn2.linear import linear
    for dt in DTYPES.values():
        for M in (3, 140):
            x, w = torch.randn(M, 200, device="cuda").to(dt), torch.randn(200, 72, device="cuda").to(dt)
            want = linear(x, w)
            x[1, 5], x[2, 7] = float("nan"), float("inf")
            got = linear(x, w)
            keep = [i for i in range(M) if i not in (1, 2)]
            assert torch.equal(got[keep], want[keep]) and not torch.isfinite(got[1:3]).any()


def test_memory_behind_the_operands_is_not_read():
    """NaN right behind x and W, in the same allocation, and in the columns beside them."""
    from atomic_gdn2.linear import linear
    for dt in DTYPES.values():
        for M, K, N in ((5, 72, 40), (130, 72, 40), (130, 100, 36)):
            a = torch.full((M + 1, K + 8), float("nan"), device="cuda").to(dt)
            b = torch.full((K + 1, N + 8), float("nan"), device="cuda").to(dt)
            x, w = a[:M, :K], b[:K, :N]
            x.copy_(torch.randn(M, K))
            w.copy_(torch.randn(K, N))
            x.requires_grad_(True), w.requires_grad_(True)
            y = linear(x, w)
            gx, gw = torch.autograd.grad(y, (x, w), torch.randn_like(y))
            assert all(torch.isfinite(t).all() for t in (y, gx, gw))


def test_gradient_against_differences():
    from atomic_gdn2.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(7)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    for act in ACTS:
        x, w, b = randn(12, 40).requires_grad_(True), (randn(40, 24) / 6).requires_grad_(True), randn(24).requires_grad_(True)
        c = randn(12, 24)
        grads = torch.autograd.grad((linear(x, w, bias=b, activation=act) * c).sum(), (x, w, b))
        for t, g in zip((x, w, b), grads):
            d = randn(*t.shape)
            h = 2.0 ** -7
            with torch.no_grad():
                up, down = ([u + s * h * d if u is t else u for u in (x, w, b)] for s in (1, -1))
                f = lambda p: (linear(p[0], p[1], bias=p[2], activation=act).double() * c.double()).sum()  # noqa: E731
                slope = (f(up) - f(down)) / (2 * h)
            # third derivatives (below 2) over the 24 x 12 results, steps of a few times h: h^2 / 6 of their sum; rounding
            # 2^-21 of the results over 2 h
            scale = (c.abs().double().sum() * 40).item()
            assert abs(slope.item() - (g.double() * d.double()).sum().item()) < scale * (h * h + 2.0 ** -21 / h), act


def test_once_differentiable_and_saved_hooks():
    from atomic_gdn2.linear import linear
    x, w = (torch.randn(s, device="cuda", requires_grad=True) for s in ((9, 16), (16, 8)))
    g, = torch.autograd.grad(linear(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    want = torch.autograd.grad(linear(x, w, activation="silu").sum(), (x, w))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().double(), lambda t: t.to("cuda")):
        y = linear(x, w, activation="silu")
    got = torch.autograd.grad(y.sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_other_stream_and_captured_graph():
    from atomic_gdn2.linear import linear
    x, w, r = (torch.randn(s, device="cuda").bfloat16() for s in ((200, 520), (520, 264), (200, 264)))
    want = linear(x, w, residual=r, activation="gelu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = linear(x, w, residual=r, activation="gelu")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            held = linear(x, w, residual=r, activation="gelu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    for i in range(3):
        x.copy_(torch.randn(200, 520))
        want = linear(x, w, residual=r, activation="gelu")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want), i


def test_equal_calls_give_equal_bits():
    from atomic_gdn2.linear import linear
    for dt in DTYPES.values():
        x, w = (torch.randn(s, device="cuda").to(dt).requires_grad_(True) for s in ((700, 900), (900, 300)))
        runs = []
        for _ in range(3):
            y = linear(x, w, activation="silu")
            runs.append((y, *torch.autograd.grad(y, (x, w), torch.ones_like(y))))
        assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))


# float32 in each of its ways: on the float32 matrix cores, as pieces that a wave or a pass cuts, rows of whole and odd widths
@pytest.mark.parametrize("M,K,N", [(45, 131, 77), (640, 2052, 1028), (300, 8196, 612), (301, 7001, 331), (300, 1501, 1403),
                                   (1025, 1027, 1001), (2050, 1000, 1030), (9, 12001, 6007)])
def test_float32_ways(M, K, N):
    check(M, K, N, torch.float32, act="gelu", bias=True, residual=True, seed=M)


@pytest.mark.parametrize("lead", [1, 4])
@pytest.mark.parametrize("M,K,N", [(64, 132, 80), (300, 4100, 1200)])
def test_float32_views(M, K, N, lead):
    """Rows of a wider tensor, from its column `lead` on; what lies beside them is not a number and stays unread."""
    def view(t):
        wide = t.new_full((t.shape[0], t.shape[1] + 2 * lead), float("nan"))
        wide[:, lead:-lead] = t
        return wide[:, lead:-lead]
    check(M, K, N, torch.float32, act="silu", bias=True, seed=M + lead, make=view)


def test_float32_equal_bits_and_captured():
    from atomic_gdn2.linear import linear
    for M, K, N in [(640, 2052, 1028), (301, 7001, 331)]:
        x, w = torch.randn(M, K, device="cuda"), torch.randn(K, N, device="cuda")
        y = linear(x, w)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            z = linear(x, w)
        for i in range(3):
            z.zero_()
            graph.replay()
            assert torch.equal(linear(x, w), y) and torch.equal(z, y), (M, K, N, i)
            torch.cuda.synchronize()
