"""Gradients of small products of 16 bits: formed from dz and from what its rounding leaves out, so that each is the definition's
but for its own rounding (half a step u) and float32 sums.

Bounds, element by element: z and the slope in float32, 2^-19 (|z| + 1) |dy| and the products' own (K / 32 + 12) 2^-22; dz as two
numbers, u^2 of it and the type's smallest number; its products (terms / 32 + 12) 2^-22 of the sums of absolute products."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _act(z, act):
    F = torch.nn.functional
    return z if act is None else F.silu(z) if act == "silu" else F.gelu(z, approximate="tanh" if act == "gelu_tanh" else "none")


def _sums(a, b):
    return (a.shape[1] / 32 + 12) * 2.0 ** -22 * (a.abs() @ b.abs())


def check(M, K, N, dt, act, bias=True, out_dtype=None, turned=False, wide=0, seed=0):
    from atomic_gdn2.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    od = out_dtype or dt
    x = torch.full((M, K + wide), float("nan"), device="cuda").to(dt)
    x[:, :K] = randn(M, K).to(dt)
    x = x[:, :K].requires_grad_(True)
    w = (randn(K, N) / K ** 0.5).to(dt)
    w = (w.t().contiguous().t() if turned else w).requires_grad_(True)
    b = randn(N).to(dt).requires_grad_(True) if bias else None
    y = linear(x, w, bias=b, activation=act, out_dtype=out_dtype)
    dy = randn(M, N).to(od)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    X, W = x.detach().double(), w.detach().double().contiguous()
    z = (X @ W + (b.detach().double() if bias else 0.0)).requires_grad_(True)
    a = _act(z, act)
    slope, = torch.autograd.grad(a, z, torch.ones_like(z)) if act else (torch.ones_like(z),)
    dz = dy.double() * slope
    u, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    e = dy.double().abs() * (2.0 ** -19 * (z.detach().abs() + 1) + 1.13 * _sums(X, W)) if act else torch.zeros_like(dz)
    e = e + 2.0 ** -22 * dz.abs() + u * u * dz.abs() + tiny
    big = dz.abs() + e
    for got, want, bound in zip(grads, (dz @ W.t().contiguous(), X.t().contiguous() @ dz, dz.sum(0)),
                                (e @ W.abs().t().contiguous() + 2 * _sums(big, W.t().contiguous()),
                                 X.abs().t().contiguous() @ e + 2 * _sums(X.t().contiguous(), big),
                                 e.sum(0) + (M / 64 + 72) * 2.0 ** -23 * big.sum(0))):
        assert got.dtype == dt
        assert ((got.double() - want).abs() <= bound + u * want.abs() + tiny).all(), ((got.double() - want).abs() / (bound + u * want.abs() + tiny)).max()


SIZES = [(1, 1, 1), (1, 500, 32), (1, 5412, 127), (2, 1793, 441), (3, 72, 40), (4, 130, 64), (5, 64, 48), (8, 512, 100), (16, 1000, 77),
         (39, 300, 301), (64, 32, 32), (130, 127, 257), (300, 512, 264), (1000, 33, 32), (700, 800, 900), (3000, 64, 100), (16384, 32, 1000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_sizes(dtype, act, M, K, N):
    check(M, K, N, DTYPES[dtype], act)
    check(M, K, N, DTYPES[dtype], act, bias=False, turned=True, seed=1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 96, 40), (7, 96, 41), (150, 128, 96), (70, 97, 33)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_float32_results_and_strided_rows(dtype, act, M, K, N):
    """A gradient of y in float32 is rounded to no 16 bits on its way either."""
    for turned in (False, True):
        check(M, K, N, DTYPES[dtype], act, out_dtype=torch.float32, turned=turned, seed=2)
        check(M, K, N, DTYPES[dtype], act, turned=turned, wide=5, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_worse_than_one_rounding(dtype):
    """In the mean over 40 small products the error is that of rounding the exact gradients (dz rounded gave 1.46 times that,
    and up to twice in a single one)."""
    from atomic_gdn2.linear import linear
    dt, got, best = DTYPES[dtype], [], []
    gen = torch.Generator(device="cuda").manual_seed(11)
    for i in range(40):
        M, K, N = (1, 300, 64) if i % 2 else (20, 64, 50)
        x, w = (torch.randn(s, device="cuda", generator=gen).to(dt).requires_grad_(True) for s in ((M, K), (K, N)))
        dy = torch.randn(M, N, device="cuda", generator=gen).to(dt)
        grads = torch.autograd.grad(linear(x, w, activation="gelu"), (x, w), dy)
        X, W = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
        exact = torch.autograd.grad(torch.nn.functional.gelu(X @ W), (X, W), dy.double())
        for g, v in zip(grads, exact):
            got.append(((g.double() - v).norm() / v.norm()).item())
            best.append(((v.to(dt).double() - v).norm() / v.norm()).item())
    assert sum(got) <= 1.01 * sum(best) and all(a <= 1.05 * b + 1e-6 for a, b in zip(got, best))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1000, 1000, 1000), (1400, 700, 1498), (1400, 700, 1500), (5000, 2000, 60), (2100, 2000, 50), (5000, 4096, 1)])
def test_larger_ones_round_dz_once(dtype, M, K, N):
    """Beyond: dz is rounded (u of it), z as well from 2^21 results on (u |z| of the slope, whose derivative is below 1)."""
    from atomic_gdn2.linear import linear
    dt = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(12)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    x, w = randn(M, K).to(dt).requires_grad_(True), (randn(K, N) / K ** 0.5).to(dt).requires_grad_(True)
    dy = randn(M, N).to(dt)
    grads = torch.autograd.grad(linear(x, w, activation="silu"), (x, w), dy)
    X, W = x.detach().double(), w.detach().double()
    z = (X @ W).requires_grad_(True)
    slope, = torch.autograd.grad(torch.nn.functional.silu(z).sum(), z)
    dz, u = dy.double() * slope, torch.finfo(dt).eps / 2
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    kept = u * z.detach().abs() if M * N > 2 ** 21 else 0.0
    e = dy.double().abs() * (kept + 2.0 ** -19 * (z.detach().abs() + 1) + 1.13 * _sums(X, W)) + u * (1 + u) * dz.abs() + tiny
    big = dz.abs() + e
    for got, want, bound in zip(grads, (dz @ W.t().contiguous(), X.t().contiguous() @ dz),
                                (e @ W.abs().t().contiguous() + _sums(big, W.t().contiguous()),
                                 X.abs().t().contiguous() @ e + _sums(X.t().contiguous(), big))):
        assert ((got.double() - want).abs() <= bound + u * want.abs() + tiny).all()


def test_an_overflowing_dz():
    """float16: what is infinite stays so, and leaves nothing."""
    from atomic_gdn2.linear import linear
    x, w = torch.ones(3, 8, device="cuda").half().requires_grad_(True), torch.ones(8, 16, device="cuda").half().requires_grad_(True)
    dy = torch.ones(3, 16, device="cuda")
    dy[1, 5] = 1e6
    gx, gw = torch.autograd.grad(linear(x, w, out_dtype=torch.float32), (x, w), dy)
    assert torch.isinf(gx[1]).all() and (gx[[0, 2]] == 16).all() and torch.isinf(gw[:, 5]).all() and torch.isfinite(gw[:, :5]).all()


def test_captured_and_equal_bits():
    from atomic_gdn2.linear import linear
    x, w, b = (torch.randn(s, device="cuda").bfloat16().requires_grad_(True) for s in ((40, 200), (200, 72), (72,)))
    dy = torch.randn(40, 72, device="cuda").bfloat16()
    run = lambda: torch.autograd.grad(linear(x, w, bias=b, activation="silu"), (x, w, b), dy)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            held = run()
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(40, 200))
            dy.copy_(torch.randn(40, 72))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
