"""8-bit states whose values lie at codes' own: without a gradient a state and its scale decay alike, and the quotient that a code
is found from is a square but for its rounding."""
import pytest
import torch

from test_gpu_optim import B1, B2, EPS, LR, WD, Plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-16])
def test_decaying_states_have_the_same_codes(dtype, size):
    """Every code of four million elements, step by step, as torch's correctly rounded quotients and roots give it."""
    from atomic_gdn2.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(9)
    n = 1 << 22
    p = torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen).to(dtype))
    opt, plain = AdamW([p], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8), Plain(p, 8, 0)
    for step in range(8):
        g = torch.randn(n, device="cuda", generator=gen) * size
        # after the first: no gradient, or one far below what the state holds
        p.grad = (g if step == 0 else g * (0.0 if step % 2 else 1e-3)).to(dtype)
        opt.step()
        want = plain.step(p.grad)
        s = opt.state[p]
        assert (s["exp_avg"].float() != plain.c).sum() == 0 and (s["exp_avg_sq"].float() != plain.u).sum() == 0, step
        assert torch.equal(p.detach().view(-1), want), step
