"""``premix_step`` and ``beam_step`` on arguments that do not fit: the entry's own errors, on the native call
path too."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def _premix(H=1):
    C = 64 * H
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    return dict(y=z(2, 6 * C + H), history=z(2, 3, 3 * C), conv_w=[z(C, 4) for _ in range(3)], conv_b=[z(C) for _ in range(3)],
                gate_b=[z(C) for _ in range(2)], decay_b=z(H), decay_a=z(H), n_heads=H, g_max=1.0)


@pytest.mark.parametrize("name", ["decay_b", "decay_a"])
def test_premix_parameters_without_dimensions(name):
    from atomic_gdn2.generation import premix_step
    premix_step(**_premix())
    with pytest.raises(ValueError, match=f"{name} must be"):
        premix_step(**{**_premix(), name: torch.zeros((), device="cuda")})
    kw = _premix()
    kw["conv_b"][1] = torch.zeros((), device="cuda")
    with pytest.raises(ValueError, match="conv_b.1. must be"):
        premix_step(**kw)


def test_premix_parameters_of_another_count():
    """Ten tensors in all are not enough: three taps, three biases of theirs, two of the gates."""
    from atomic_gdn2.generation import premix_step
    for a, b in (("conv_b", "gate_b"), ("gate_b", "conv_b"), ("conv_w", "conv_b")):
        kw = _premix()
        kw[b].append(kw[a].pop())
        with pytest.raises(ValueError):
            premix_step(**kw)


def test_beam_scores_without_dimensions():
    from atomic_gdn2.generation import beam_step
    with pytest.raises(ValueError, match="scores must be"):
        beam_step(torch.zeros((1, 10), device="cuda"), torch.tensor(0.0, device="cuda"))


def test_beam_count_is_checked_before_memory_is_taken():
    from atomic_gdn2.generation import beam_step
    x, s = torch.zeros((64, 9), device="cuda"), torch.zeros((64, 1), device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.max_memory_reserved()
    for n in (129, 1 << 20, (1 << 31) - 1):
        with pytest.raises(ValueError, match=f"n={n}"):
            beam_step(x, s, n=n)
    assert torch.cuda.max_memory_reserved() == before
