"""cross_entropy of more short rows than one launch's threads can take."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 8), (torch.float32, 4)])
def test_rows_beyond_the_threads_of_a_launch(dtype, V):
    """2^26 + 5 rows, a wave each: parts of them give the same bits in calls of their own."""
    from atomic_gdn2.losses import cross_entropy
    rows = 2 ** 26 + 5
    x = torch.empty((rows, V), dtype=dtype, device="cuda")
    for part in x.split(2 ** 22):
        part.copy_(torch.randn(part.shape, device="cuda"))
    t = torch.randint(0, V, (rows,), dtype=torch.int32, device="cuda")
    t[::7] = -100
    x.requires_grad_(True)
    parts = [slice(0, 999), slice(2 ** 25 - 500, 2 ** 25 + 501), slice(2 ** 26 - 500, rows)]
    loss = cross_entropy(x, t, reduction="none")
    f = torch.rand(rows, device="cuda")
    g, = torch.autograd.grad(loss, x, f)
    for p in parts:
        y = x.detach()[p].requires_grad_(True)
        want = cross_entropy(y, t[p], reduction="none")
        d, = torch.autograd.grad(want, y, f[p])
        assert torch.equal(loss[p], want) and torch.equal(g[p], d)
    assert not loss[::7].any() and (loss > 0).sum() > 0.8 * rows
    count = int((t != -100).sum())
    mean = cross_entropy(x.detach(), t)
    assert abs(mean.item() - loss.double().sum().item() / count) <= 2.0 ** -23 * mean.item()
