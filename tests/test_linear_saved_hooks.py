"""linear under saved-tensor hooks that give back other layouts: z is read as one array, x by rows, the weight by rows or
turned."""
import pytest
import torch

from atomic_gdn2 import linear


def _wider(t):
    """t as rows of a wider matrix."""
    wide = t.new_full((t.shape[0], t.shape[1] + 3), 7.0)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _columns(t):
    """t with its columns in one piece."""
    return t.t().contiguous().t()


HOOKS = [lambda t: t, _wider, _columns, lambda t: t.double()]


@pytest.mark.parametrize("hook", HOOKS, ids=["same", "wider", "columns", "types"])
def test_what_the_backward_pass_hands_to_the_kernels(monkeypatch, hook):
    """(the kernels' arguments are looked at here, on the host)"""
    seen = []

    def product(form, a, b, M, K, N, out, *rest):
        seen.extend((a, b))
        return out.zero_()

    def slope(dy, z, dtype, act, bias_dtype, need_dz, fine):
        assert z.is_contiguous() and torch.equal(z, kept) and z.dtype == dtype
        return torch.ones_like(dy), None

    kept = torch.randn(5, 6)
    monkeypatch.setattr(linear, "_product", product)
    monkeypatch.setattr(linear, "_slope", slope)
    monkeypatch.setattr(linear, "_forward", lambda x, w, *rest: (torch.zeros(5, 6), kept))
    x, w = torch.randn(5, 4, requires_grad=True), torch.randn(4, 6, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook):
        y = linear._Linear.apply(x, w, None, None, 1, torch.float32)
    y.sum().backward()
    # dz W^T and x^T dz, or with W turned dz (W^T) as it lies and dz^T x
    assert len(seen) == 4
    assert all(t.dtype == torch.float32 and t.stride(1) == 1 and t.stride(0) >= t.shape[1] for t in seen)
    assert torch.equal(seen[1] if seen[1].shape == w.shape else seen[1].t(), w)
    assert torch.equal(seen[2] if seen[2].shape == x.shape else seen[3], x)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_are_the_same(dtype, native):
    gen = torch.Generator(device="cuda").manual_seed(8)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(dtype).requires_grad_(True)  # noqa: E731
    x, w, b = r(2, 33, 48), r(48, 40), r(40)
    rows = lambda: x.reshape(66, 48) if native else x.transpose(0, 1)  # noqa: E731
    run = lambda: linear.linear(rows(), w, bias=b, activation="silu")  # noqa: E731
    dy = torch.randn(run().shape, device="cuda", generator=gen).to(dtype)
    want = torch.autograd.grad(run(), (x, w, b), dy)
    for hook in HOOKS:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: hook(t) if t.dim() == 2 else t):
            y = run()
        got = torch.autograd.grad(y, (x, w, b), dy)
        assert all(torch.equal(g, v) for g, v in zip(got, want))
