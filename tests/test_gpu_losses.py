"""Cross-entropy and its gradient against the definition in 64 bits.

Bounds: exponentials of x - max in float32, 2^-22 (|x - max| + 2) each relative, weighted by the softmax the argument's
part stays below 2^-22 (log V + 2); their sum V / 256 + 16 roundings of 2^-24; the loss is a difference of numbers up to
max |x| + log V; the gradient is rounded to its dtype (half a step), after a factor on the loss once more.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _definition(x, t, ignore, e, z, reduction):
    """loss (a graph of x, in 64 bits)."""
    kept = t != ignore
    at = torch.where(kept, t, 0)
    lse = torch.logsumexp(x, -1)
    mean = x.mean(-1) if e else 0.0
    rows = lse - (1 - e) * x.gather(-1, at[..., None])[..., 0] - e * mean + z * lse * lse
    rows = torch.where(kept, rows, torch.zeros_like(rows))
    return rows if reduction == "none" else rows.sum() / (max(1, int(kept.sum())) if reduction == "mean" else 1)


def check(rows, V, dt, e=0.0, z=0.0, reduction="mean", ignored=0.2, factor=None, seed=0, wide=0, spread=3.0, targets=None,
          index=torch.int64):
    from atomic_gdn2.losses import cross_entropy
    gen = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.full((rows, V + wide), float("nan"), device="cuda").to(dt)
    base[:, :V] = (torch.randn((rows, V), device="cuda", generator=gen) * spread).to(dt)
    x = base[:, :V].detach().requires_grad_(True)
    t = torch.randint(0, V, (rows,), device="cuda", generator=gen)
    t = torch.where(torch.rand(rows, device="cuda", generator=gen) < ignored, -100, t) if targets is None else targets
    loss = cross_entropy(x, t.to(index), label_smoothing=e, z_loss=z, reduction=reduction)
    X = x.detach().double().requires_grad_(True)
    want = _definition(X, t, -100, e, z, reduction)
    n = max(1, int((t != -100).sum())) if reduction == "mean" else 1
    top = X.detach().abs().max().item() + math.log(V)
    rel = 2.0 ** -22 * (math.log(V) + 4) + (V / 256 + 16) * 2.0 ** -24 + 2.0 ** -22 * top
    off = (rel + 2.0 ** -22 * top) * (1 + 2 * z * top) + (V / 256 + 16) * 2.0 ** -24 * e * top
    assert loss.dtype == torch.float32 and loss.shape == want.shape
    sums = 1 if reduction in ("none", "mean") else max(1, int((t != -100).sum()))
    assert ((loss.double() - want).abs() <= off * sums + 2.0 ** -24 * want.abs()).all(), (loss.double() - want).abs().max()
    f = torch.ones_like(want) if factor is None else torch.full_like(want, factor) * (torch.arange(max(1, want.numel()), device="cuda").view(want.shape) % 3 + 1)
    got, = torch.autograd.grad(loss, x, f.float())
    ref, = torch.autograd.grad(want, X, f)
    p = torch.softmax(X.detach(), -1)
    s = f.abs().max().item() / n
    u = torch.finfo(dt).eps / 2
    bound = s * (rel * (1 + 2 * z * top) * p + 2.0 ** -22 * (e / V)) + 2.0 ** -22 * s * (t[:, None] == torch.arange(V, device="cuda"))
    bound = bound + (2 * u + u * u) * ref.abs() + 2 * torch.finfo(dt).smallest_normal * torch.finfo(dt).eps * max(1.0, s)
    assert got.dtype == dt and got.shape == (rows, V)
    bad = (got.double() - ref).abs() > bound
    assert not bad.any(), ((got.double() - ref).abs() / bound).max()
    assert not got[t == -100].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 64, 255, 256, 1000, 2049, 8192, 33333, 50257, 131072, 300001])
def test_sizes(dtype, V):
    check(5, V, DTYPES[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("e,z", [(0.0, 0.0), (0.1, 0.0), (0.0, 1e-3), (0.2, 1e-3), (1.0, 0.0)])
def test_terms(dtype, reduction, e, z):
    for V in (100, 5000):
        check(37, V, DTYPES[dtype], e=e, z=z, reduction=reduction, seed=1)
        check(6, V, DTYPES[dtype], e=e, z=z, reduction=reduction, seed=2, factor=0.37, index=torch.int32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(1, 256), (1, 40000), (3000, 256), (16384, 256), (2100, 70), (700, 4100)])
def test_rows(dtype, rows, V):
    check(rows, V, DTYPES[dtype], seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,wide", [(64, 1), (257, 3), (4096, 7), (4096, 8), (20001, 5)])
def test_strided_rows(dtype, V, wide):
    """Rows at odd places; NaN beside them."""
    check(9, V, DTYPES[dtype], wide=wide, seed=4, e=0.1)


def test_leading_dimensions_and_other_strides():
    from atomic_gdn2.losses import cross_entropy
    x = torch.randn(3, 8, 300, device="cuda", requires_grad=True)
    t = torch.randint(0, 300, (3, 8), device="cuda")
    want = torch.nn.functional.cross_entropy(x.reshape(-1, 300).double(), t.reshape(-1))
    for y in (x, x[:, :, :], x.transpose(1, 2).contiguous().transpose(1, 2), x.expand(3, 8, 300)):
        assert abs(cross_entropy(y, t).item() - want.item()) < 1e-5
    a = cross_entropy(x[:, :-1], t[:, 1:], reduction="none")
    assert a.shape == (3, 7)
    g, = torch.autograd.grad(a.sum(), x)
    assert g.shape == x.shape and not g[:, -1].any() and g[:, :-1].abs().sum() > 0


def test_nothing_counts():
    from atomic_gdn2.losses import cross_entropy
    for dt in DTYPES.values():
        x = torch.randn(4, 50, device="cuda").to(dt).requires_grad_(True)
        t = torch.full((4,), -100, device="cuda")
        for r in ("mean", "sum", "none"):
            loss = cross_entropy(x, t, reduction=r)
            g, = torch.autograd.grad(loss.sum(), x)
            assert not loss.any() and not g.any()
    # rows that are ignored may hold anything
    x = torch.randn(4, 50, device="cuda")
    want = cross_entropy(x[:2], t[:2] * 0 + 3)
    x[2:], t[:2] = float("nan"), 3
    x.requires_grad_(True)
    loss = cross_entropy(x, t)
    g, = torch.autograd.grad(loss, x)
    assert torch.equal(loss, want) and torch.isfinite(g).all() and not g[2:].any()


def test_banned_tokens_and_extremes():
    from atomic_gdn2.losses import cross_entropy
    inf = float("inf")
    for dt in DTYPES.values():
        for V in (90, 9000):
            x = torch.randn(6, V, device="cuda").to(dt)
            x[:, 10:60] = -inf
            x[1] = torch.finfo(dt).min
            x[2] = torch.finfo(dt).max
            x[3, :] = -inf
            x[3, 5] = 2.0                        # one token is left
            t = torch.full((6,), 5, device="cuda")
            x = x.requires_grad_(True)
            loss = cross_entropy(x, t, reduction="none")
            g, = torch.autograd.grad(loss.sum(), x)
            assert torch.isfinite(loss).all() and torch.isfinite(g).all() and not g[0, 10:60].any()
            assert abs(loss[1].item() - math.log(V)) < 1e-3 and abs(loss[2].item() - math.log(V)) < 1e-3 and loss[3].item() == 0.0
            y = x.detach().clone()
            y[0, 5], y[1], y[2, 7], y[3, 5] = -inf, -inf, inf, float("nan")
            y.requires_grad_(True)
            loss = cross_entropy(y, t, reduction="none")
            ref = torch.nn.functional.cross_entropy(y.detach().float(), t, reduction="none")
            assert loss[0].item() == inf and torch.isnan(loss[1:4]).all() and torch.isnan(ref[1:4]).all()
            assert torch.isfinite(loss[4:]).all()


def test_targets_outside_are_nan_and_read_nothing():
    from atomic_gdn2.losses import cross_entropy
    x = torch.randn(5, 40, device="cuda", requires_grad=True)
    t = torch.tensor([0, 40, -1, 2 ** 40, 39], device="cuda")
    loss = cross_entropy(x, t, reduction="none")
    g, = torch.autograd.grad(loss.sum(), x)
    bad = torch.tensor([False, True, True, True, False], device="cuda")
    assert torch.equal(torch.isnan(loss), bad) and torch.equal(torch.isnan(g).any(1), bad)


def test_backward_twice_and_without_gradients():
    from atomic_gdn2.losses import cross_entropy
    for dt in DTYPES.values():
        x = torch.randn(30, 700, device="cuda").to(dt).requires_grad_(True)
        t = torch.randint(0, 700, (30,), device="cuda")
        loss = cross_entropy(x, t)
        a, = torch.autograd.grad(2.0 * loss, x, retain_graph=True)
        b, = torch.autograd.grad(2.0 * loss, x, retain_graph=True)
        c, = torch.autograd.grad(0.0 * loss, x)
        off = (a.double() - b.double()).abs()
        assert (off <= torch.finfo(dt).eps * a.double().abs()).all() and not c.any()
        with torch.no_grad():
            assert torch.equal(cross_entropy(x, t), loss)
        loss = cross_entropy(x, t)
        g, = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_changed_logits_are_noticed():
    from atomic_gdn2.losses import cross_entropy
    x = torch.randn(4, 30, device="cuda", requires_grad=True)
    y = x * 1.0
    loss = cross_entropy(y, torch.zeros(4, dtype=torch.int64, device="cuda"))
    y.add_(1.0)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_scaled_float16_does_not_underflow():
    from atomic_gdn2.losses import cross_entropy
    x = torch.randn(4096, 512, device="cuda").half().requires_grad_(True)
    t = torch.randint(0, 512, (4096,), device="cuda")
    g, = torch.autograd.grad(cross_entropy(x, t) * 65536.0, x)
    X = x.detach().double().requires_grad_(True)
    ref, = torch.autograd.grad(torch.nn.functional.cross_entropy(X, t) * 65536.0, X)
    assert (g.double() - ref).norm() / ref.norm() < 2.0 ** -11


def test_captured_graph():
    from atomic_gdn2.losses import cross_entropy
    for rows, V in ((64, 300), (8, 40000)):
        x = torch.randn(rows, V, device="cuda").bfloat16().requires_grad_(True)
        t = torch.randint(0, V, (rows,), device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.autograd.grad(cross_entropy(x, t), x)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                loss = cross_entropy(x, t)
                g, = torch.autograd.grad(loss, x)
        torch.cuda.current_stream().wait_stream(s)
        for i in range(3):
            with torch.no_grad():
                x.copy_(torch.randn(rows, V))
                t.copy_(torch.randint(0, V, (rows,)))
            y = x.detach().clone().requires_grad_(True)
            want = cross_entropy(y, t)
            wg, = torch.autograd.grad(want, y)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(loss, want) and torch.equal(g, wg), i
