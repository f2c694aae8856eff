"""What a loss is multiplied with: rows that are ignored have no gradient, whatever stands beside them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", DTYPES)
def test_factors_of_ignored_rows(dtype, bad):
    """Weights of padded rows are often 0 / 0."""
    from atomic_gdn2.losses import cross_entropy
    gen = torch.Generator(device="cuda").manual_seed(6)
    for V in (64, 999, 40000):
        x = torch.randn((9, V), device="cuda", generator=gen).to(DTYPES[dtype]).requires_grad_(True)
        t = torch.randint(0, V, (9,), device="cuda", generator=gen)
        t[[2, 5]] = -100
        f = torch.full((9,), 0.25, device="cuda")
        want, = torch.autograd.grad(cross_entropy(x, t, reduction="none"), x, f)
        f[[2, 5]] = bad
        loss = cross_entropy(x, t, reduction="none")
        for _ in range(2):
            got, = torch.autograd.grad(loss, x, f, retain_graph=True)
            assert not got[[2, 5]].any()
            assert torch.equal(got, want)           # (a power of two: neither pass rounds twice)
        for reduction in ("sum", "mean"):
            loss = cross_entropy(x, t, reduction=reduction)
            for _ in range(2):
                got, = torch.autograd.grad(loss, x, torch.full_like(loss, bad), retain_graph=True)
                assert not got[[2, 5]].any() and not torch.isfinite(got[:2]).all(1).any()
