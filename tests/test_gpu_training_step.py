"""A training step of the LM on linear, cross_entropy and AdamW together."""
import pytest
import torch

from atomic_gdn2 import e2e_lm

pytestmark = pytest.mark.gpu

SMALL = dict(vocab_size=61, d_model=128, n_heads=2, d_head=64, n_layers=2)


def _lm(**kw):
    return e2e_lm.make_lm(e2e_lm.LMConfig(**{**SMALL, **kw}), seed=1)


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


def _grads(model, ids, fused):
    loss = e2e_lm.lm_loss(model, ids, fused)
    return loss.detach(), dict(zip([n for n, _ in model.named_parameters()], torch.autograd.grad(loss, list(model.parameters()))))


def test_fused_loss_is_the_loss():
    """The same logits: both losses are float32 sums of theirs, the gradients differ by float32 rounding (2^-20 of each)."""
    model, ids = _lm(), e2e_lm.synthetic_tokens(e2e_lm.LMConfig(**SMALL), batch=3, length=128)
    (a, ga), (b, gb) = _grads(model, ids, False), _grads(model, ids, True)
    assert abs(a.item() - b.item()) < 2.0 ** -20 * a.item()
    assert all(_rel(gb[n], ga[n]) < 2.0 ** -18 for n in ga)


@pytest.mark.parametrize("length", [64, 192])
def test_products_in_bfloat16(length):
    """Each of the 2 x 6 products and their 24 gradient products rounds two operands (2^-9 / sqrt 3 of a product's norm
    each, 1.6e-3 together); through the chain they add up as squares to below 1e-2, and the norms and gates between
    them stretch a relative error at most a few times."""
    ids = e2e_lm.synthetic_tokens(e2e_lm.LMConfig(**SMALL), batch=3, length=length)
    full, half = _lm(), _lm(products="bfloat16")
    assert all(torch.equal(p, q) for p, q in zip(full.parameters(), half.parameters()))
    with torch.no_grad():
        assert _rel(half(ids), full(ids)) < 0.02 and half(ids).dtype == torch.float32
    (a, ga), (b, gb) = _grads(full, ids, False), _grads(half, ids, True)
    assert abs(a.item() - b.item()) < 0.01 * a.item()
    far = {n: _rel(gb[n], ga[n]) for n in ga}
    assert all(g.dtype == torch.float32 for g in gb.values()) and max(far.values()) < 0.05, far


def test_products_in_bfloat16_once_differentiable_and_refused_elsewhere():
    model, ids = _lm(products="bfloat16"), e2e_lm.synthetic_tokens(e2e_lm.LMConfig(**SMALL), batch=1, length=64)
    x = torch.randn(1, 64, 128, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="once differentiable"):
        torch.autograd.grad(model.blocks[0](x).sum(), x, create_graph=True)
    model.blocks[0].out_proj.register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="bfloat16"):
        model(ids)


@pytest.mark.parametrize("bits,products", [(32, "float32"), (8, "float32"), (32, "bfloat16"), (8, "bfloat16")])
def test_steps(bits, products):
    """The first update of the fused step is the plain step's: lr times the signs of the gradients, nearly, whose
    rounding moves it where a gradient is near eps; later ones go the same way (the second moments' bits apart)."""
    cfg = e2e_lm.LMConfig(**SMALL)
    ids = e2e_lm.synthetic_tokens(cfg, batch=2, length=128)
    plain, fused = _lm(), _lm(products=products)
    start = [p.detach().clone() for p in plain.parameters()]
    one, two = e2e_lm.TrainStep(plain), e2e_lm.TrainStep(fused, fused=True, state_bits=bits)
    for _ in range(3):
        a, b = one(ids), two(ids)
        assert torch.isfinite(b) and abs(a.item() - b.item()) < (1e-4 if products == "float32" and bits == 32 else 0.02) * a.item()
        assert two.opt.norm.item() > 0
    if products == "float32" and bits == 32:
        moved = [(p.detach() - s, q.detach() - s) for p, q, s in zip(plain.parameters(), fused.parameters(), start)]
        num = sum((u - v).double().square().sum().item() for u, v in moved)
        assert num < 1e-4 * sum(u.double().square().sum().item() for u, _ in moved)
