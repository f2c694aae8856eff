"""Backward passes of cross_entropy in a graph of their own: every replay forms the gradient of the factor it finds."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _wanted(x, t, f, reduction):
    from atomic_gdn2.losses import cross_entropy
    y = x.detach().clone().requires_grad_(True)
    return torch.autograd.grad(cross_entropy(y, t, reduction=reduction), y, f)[0].double()


@pytest.mark.parametrize("how", ["eager", "captured"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("strided", [False, True])
def test_replays_of_a_backward_pass(dtype, reduction, how, strided):
    """The forward pass once (eagerly, or in a graph of its own), its backward pass several times.  A kept gradient that is
    multiplied is rounded twice (2 u + u^2, u half a step), one that is formed anew once, and so is what it is compared with: they
    differ by (4 u + 2 u^2) / (1 - 2 u) at most, below 4.1 u."""
    from atomic_gdn2.losses import cross_entropy
    dt = DTYPES[dtype]
    base = torch.randn(33, 520 if strided else 500, device="cuda").to(dt)
    base = base.view(3, 11, -1)[..., 3:503] if strided else base        # (strided: not a call of the native path)
    x, t = base.detach().requires_grad_(True), torch.randint(0, 500, base.shape[:-1], device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(cross_entropy(x, t, reduction=reduction).sum(), x)
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        if how == "captured":
            with torch.cuda.graph(first, stream=s):
                loss = cross_entropy(x, t, reduction=reduction)
        else:
            loss = cross_entropy(x, t, reduction=reduction)
        f = torch.ones_like(loss)
        torch.cuda.synchronize()
        with torch.cuda.graph(second, stream=s):
            g, = torch.autograd.grad(loss, x, f, retain_graph=True)
    torch.cuda.current_stream().wait_stream(s)
    if how == "captured":
        first.replay()
    u = torch.finfo(dt).eps / 2
    for k, factor in enumerate((0.3, 7.0, 1.0, 0.3, 0.3)):
        f.fill_(factor)
        second.replay()
        torch.cuda.synchronize()
        want = _wanted(x, t, f, reduction)
        assert ((g.double() - want).abs() <= (4.1 * u + 2.0 ** -22) * want.abs() + 2 * torch.finfo(dt).smallest_normal * torch.finfo(dt).eps).all(), k
    # and an eager pass over the same graph afterwards
    got, = torch.autograd.grad(loss, x, f)
    assert ((got.double() - want).abs() <= (4.1 * u + 2.0 ** -22) * want.abs() + 2 * torch.finfo(dt).smallest_normal * torch.finfo(dt).eps).all()
