"""Sizes and strides above 32 bits: refused or served, never cut."""
import pytest
import torch


def test_more_than_32_bits_of_tokens_or_rows_are_refused():
    from atomic_gdn2 import w4
    from atomic_gdn2.generation import beam_step
    one = torch.zeros((1, 1))
    with pytest.raises(ValueError, match="2\\^31"):
        beam_step(one.expand(1, 2 ** 32 + 5), one, n=1)
    with pytest.raises(ValueError, match="2\\^31"):
        beam_step(one.expand(3, 2 ** 30), torch.zeros((1, 3)), n=1)
    with pytest.raises(ValueError, match="2\\^31"):
        beam_step(one.expand(2 ** 32 + 1, 1), one.expand(2 ** 32 + 1, 1), n=1)
    W = w4.quantize_w4(torch.randn(64, 8), 64)
    with pytest.raises(ValueError, match="2\\^31"):
        w4.w4_linear(torch.zeros((1, 64)).expand(2 ** 32 + 3, 64), W)


@pytest.mark.gpu
def test_premix_rows_more_than_32_bits_apart():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    from atomic_gdn2.generation import premix_step
    C, H, far = 64, 1, 2 ** 32 + 1000
    gen = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    near = randn(2, 6 * C + H)
    y = torch.empty(far + 6 * C + H, device="cuda").as_strided((2, 6 * C + H), (far, 1))
    y[0], y[1] = near[0], near[1]
    y.as_strided((6 * C + H,), (1,), 1000).zero_()           # where a stride cut to 32 bits would look
    args = (randn(2, 3, 3 * C), [randn(C, 4) for _ in range(3)], [randn(C) for _ in range(3)], [randn(C) for _ in range(2)],
            randn(H), randn(H))
    got, want = (premix_step(t, *args, n_heads=H, g_max=1.0) for t in (y, near))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
