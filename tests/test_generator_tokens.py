"""Token ids outside the vocabulary never index the embedding."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_tokens_outside_the_vocabulary():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    from atomic_gdn2 import e2e_lm
    from atomic_gdn2.generation import Generator
    V = 61
    gen = Generator(e2e_lm.make_lm(e2e_lm.LMConfig(vocab_size=V, d_model=128, n_heads=2, d_head=64, n_layers=2)), group_size=32)
    ids = torch.arange(10, device="cuda").view(2, 5)
    for bad in (V, -1, 2 ** 40):
        wrong = ids.clone()
        wrong[1, 3] = bad
        with pytest.raises(ValueError, match="token ids must lie in 0 .. 60"):
            gen.prefill(wrong)
        with pytest.raises(ValueError, match="token ids must lie in 0 .. 60"):
            gen.beam_search(wrong, 2, 3)
    with pytest.raises(ValueError, match="whole numbers"):
        gen.prefill(ids.to(torch.complex64))
    logits, cache = gen.prefill(ids)
    a, _ = gen.step(torch.tensor([V + 5, -3], device="cuda"), cache)        # (not looked at by the host: the nearest ones)
    b, _ = gen.step(torch.tensor([V - 1, 0], device="cuda"), cache)
    assert torch.equal(a, b)
    c, _ = gen.step(torch.tensor([2 ** 40, -2 ** 40], device="cuda"), cache)
    assert torch.equal(c, b)
    d, _ = gen.step(torch.tensor([60, 0], device="cuda", dtype=torch.uint8), cache)
    assert torch.equal(d, b)
