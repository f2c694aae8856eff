"""Slopes of the activations at values far out, where they are 0 or 1."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 3e4), (torch.bfloat16, 1e19), (torch.bfloat16, 3e25), (torch.float32, 1e19),
                                        (torch.float32, 3e25)])
@pytest.mark.parametrize("bias", [False, True])
def test_slopes_far_out(act, dtype, size, bias):
    """z = 4 size x0 with x0 of both signs: float16 keeps it as an infinity, its y in float32 is finite.  Above, the slope is 1,
    below, 0, so that dx = dy W^T there is a sum of powers of two of one size, or nothing."""
    from atomic_gdn2.linear import linear
    for M in (6, 200):
        x = torch.zeros(M, 16, device="cuda", dtype=dtype)
        x[::2, :4], x[1::2, :4] = 1.0, -1.0
        w = torch.full((16, 24), size, device="cuda", dtype=dtype)
        b = torch.zeros(24, device="cuda", dtype=dtype) if bias else None
        leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
        y = linear(x, w, bias=b, activation=act, out_dtype=torch.float32)
        assert torch.isfinite(y).all() and (y[::2] > size).all() and (y[1::2].abs() < 1e-6).all()
        dy = torch.full((M, 24), 2.0 ** -60 if dtype != torch.float16 else 2.0 ** -10, device="cuda")
        grads = torch.autograd.grad(y, leaves, dy)
        assert torch.equal(grads[0][1::2], torch.zeros_like(grads[0][1::2]))
        want = 24 * dy[0, 0].double().item() * w[0, 0].double().item()
        assert ((grads[0][::2].double() - want).abs() <= torch.finfo(dtype).eps * want).all()
        rows = math.ceil(M / 2)
        assert torch.equal(grads[1][:4].double(), torch.full((4, 24), rows * dy[0, 0].double().item(), dtype=torch.float64, device="cuda"))
        if bias:
            assert torch.equal(grads[2].double(), torch.full((24,), rows * dy[0, 0].double().item(), dtype=torch.float64, device="cuda"))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_slopes_of_nan(act):
    from atomic_gdn2.linear import linear
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        x, w = torch.randn(9, 16, device="cuda").to(dt), torch.randn(16, 24, device="cuda").to(dt)
        x[4, 3] = math.nan
        x.requires_grad_(True)
        g, = torch.autograd.grad(linear(x, w, activation=act).sum(), x)
        bad = ~torch.isfinite(g).all(1)
        assert bad[4] and bad.sum() == 1
