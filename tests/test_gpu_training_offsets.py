"""Tensors of more than 2^31 elements: linear, cross_entropy and AdamW at their last rows, and where an offset cut to 32 bits
would read or write."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _fill(t, gen, scale=1.0):
    for part in t.split(max(1, 2 ** 26 // t[0].numel())):
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen) * scale)
    return t


def _near(got, a, b):
    """(sums of float32: (K / 32 + 12) 2^-22 of the absolute products, what pieces leave out, and half a step)"""
    want, size = a.double() @ b.double(), a.double().abs() @ b.double().abs()
    bound = ((a.shape[1] / 32 + 12) * 2.0 ** -22 + 2.0 ** -21) * size + torch.finfo(got.dtype).eps / 2 * want.abs()
    return ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,stride", [(torch.bfloat16, 8192), (torch.bfloat16, 8195), (torch.float32, 8192), (torch.float32, 8195)])
def test_products_of_long_operands(dtype, stride):
    from atomic_gdn2.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(1)
    M, K, N = 262144 + 1057, 8192, 40
    x = _fill(torch.empty((M, stride), dtype=dtype, device="cuda"), gen)[:, :K].requires_grad_(True)
    w = (torch.randn((K, N), device="cuda", generator=gen) / 90).to(dtype).requires_grad_(True)
    dy = torch.randn((M, N), device="cuda", generator=gen).to(dtype)
    y = linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for rows in (slice(0, 200), slice(261900, 262300), slice(M - 300, M)):
        assert _near(y.detach()[rows], x.detach()[rows], w.detach()) and _near(dx[rows], dy[rows], w.detach().t().contiguous())
    want = torch.zeros((K, N), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for a, b in zip(x.detach().split(2 ** 15), dy.split(2 ** 15)):
        a, b = a.double().t().contiguous(), b.double()
        want += a @ b
        size += a.abs() @ b.abs()
    assert ((dw.double() - want).abs() <= ((M / 32 + 12) * 2.0 ** -22 + 2.0 ** -21) * size + torch.finfo(dtype).eps / 2 * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [32001, 32000])
def test_products_of_long_results(dtype, N):
    from atomic_gdn2.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(2)
    M, K = 70001, 40
    x, w = torch.randn((M, K), device="cuda", generator=gen).to(dtype), torch.randn((K, N), device="cuda", generator=gen).to(dtype)
    res = _fill(torch.empty((M, N), dtype=dtype, device="cuda"), gen)
    y = linear(x, w, residual=res)
    for rows in (slice(0, 50), slice(2 ** 31 // N - 50, 2 ** 31 // N + 50), slice(M - 50, M)):
        one = torch.cat([x[rows], torch.eye(x[rows].shape[0], device="cuda", dtype=dtype)], 1)       # (the residual as products by 1)
        assert _near(y[rows], one, torch.cat([w, res[rows]], 0))


@pytest.mark.parametrize("V", [131071, 131072])
def test_losses_of_long_logits(V):
    from atomic_gdn2.losses import cross_entropy
    gen = torch.Generator(device="cuda").manual_seed(3)
    rows = 17001
    x = _fill(torch.empty((rows, V), dtype=torch.bfloat16, device="cuda"), gen, 3.0).requires_grad_(True)
    t = torch.randint(0, V, (rows,), device="cuda", generator=gen)
    f = torch.rand(rows, device="cuda", generator=gen)
    loss = cross_entropy(x, t, reduction="none")
    g, = torch.autograd.grad(loss, x, f)
    for part in (slice(0, 300), slice(16200, 16600), slice(rows - 300, rows)):
        y = x.detach()[part].requires_grad_(True)
        want = cross_entropy(y, t[part], reduction="none")
        d, = torch.autograd.grad(want, y, f[part])
        assert torch.equal(loss[part], want) and torch.equal(g[part], d)


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 32), (torch.float32, 8), (torch.bfloat16, 8)])
def test_a_long_tensor_of_adamw(dtype, bits):
    """Its ends beside parameters of their own: a first step is the same, whatever the dither of the states."""
    from atomic_gdn2.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(4)
    n, part = 2 ** 31 + 256 * 1000 + 77, 256 * 3000 + 77
    p = torch.nn.Parameter(torch.empty(n, dtype=dtype, device="cuda"))
    for s in p.data.split(2 ** 28):
        s.copy_(torch.randn(s.shape, device="cuda", generator=gen))
    p.grad = torch.empty_like(p)
    for s in p.grad.split(2 ** 28):
        s.copy_(torch.randn(s.shape, device="cuda", generator=gen))
    ends = [slice(0, 256 * 1000), slice(n - part, n)]
    qs = [torch.nn.Parameter(p.detach()[e].clone()) for e in ends]
    for q, e in zip(qs, ends):
        q.grad = p.grad[e].clone()
    one, two = AdamW([p], lr=1e-2, state_bits=bits, max_norm=float("inf")), AdamW(qs, lr=1e-2, state_bits=bits)
    one.step(), two.step()
    norm = sum(s.double().square().sum().item() for s in p.grad.split(2 ** 28)) ** 0.5
    assert abs(one.norm.item() - norm) <= 2.0 ** -23 * norm
    for q, e in zip(qs, ends):
        assert torch.equal(p.detach()[e], q.detach())
        if bits == 32:
            assert torch.equal(one.state[p]["exp_avg"][e], two.state[q]["exp_avg"])
        else:
            blocks = slice(e.start // 256, -(-e.stop // 256))
            assert torch.equal(one.state[p]["exp_avg_scale"][blocks], two.state[q]["exp_avg_scale"])
    if bits == 8:
        del two, qs
        m = one.unpack_states()[0][0]
        scale = one.state[p]["exp_avg_scale"]
        for e in ends:
            c = one.state[p]["exp_avg"][e].float()
            assert torch.equal(m[e], c * c.abs() * scale[slice(e.start // 256, -(-e.stop // 256))].repeat_interleave(256)[:c.numel()])
