"""LMConfig(products="bfloat16") where the HIP kernels cannot run them: refused in every part of the model, the logits among them."""
import pytest
import torch

from atomic_gdn2 import e2e_lm


def test_logits_of_a_model_without_blocks():
    cfg = dict(vocab_size=16, d_model=8, n_heads=2, d_head=4, n_layers=0)
    ids = torch.zeros(1, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="bfloat16"):
        e2e_lm.LM(e2e_lm.LMConfig(**cfg, products="bfloat16"), lambda q, k, v, w, b, g: v)(ids)
    assert e2e_lm.LM(e2e_lm.LMConfig(**cfg), lambda q, k, v, w, b, g: v)(ids).shape == (1, 4, 16)


@pytest.mark.gpu
def test_a_hooked_final_norm():
    """(the logits were float32 products then)"""
    cfg = e2e_lm.LMConfig(vocab_size=61, d_model=128, n_heads=2, d_head=64, n_layers=1, products="bfloat16")
    model, ids = e2e_lm.make_lm(cfg, seed=1), e2e_lm.synthetic_tokens(cfg, batch=1, length=64)
    want = model(ids).detach()
    hook = model.final_norm.register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="bfloat16"):
        model(ids)
    hook.remove()
    assert torch.equal(model(ids), want)
