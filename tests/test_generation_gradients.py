"""The operators of token generation have no gradients: an input's is not lost in silence, asking for it
raises.  Calls that ask for none keep their results."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def _calls():
    """name -> (function of its float tensors, those tensors)"""
    from atomic_gdn2 import generation, w4
    gen = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    W, C, fin = w4.quantize_w4(randn(64, 24), 32), 64, torch.zeros((1, 3), dtype=torch.bool, device="cuda")
    par = torch.tensor([1, 0, 1], device="cuda")
    return {
        "w4_linear": (lambda x, b, r: w4.w4_linear(x, W, bias=b, residual=r), [randn(3, 64), randn(24), randn(3, 24)]),
        "beam_step": (lambda x, s: generation.beam_step(x, s, n=4, finished=fin, eos_id=2), [randn(3, 50), randn(1, 3)]),
        "premix_step": (lambda y, h, *w: generation.premix_step(y, h, w[:3], w[3:6], w[6:8], w[8], w[9], n_heads=1, g_max=1.0,
                                                               parents=par),
                        [randn(3, 6 * C + 1), randn(2, 3, 3 * C), *(randn(C, 4) for _ in range(3)), *(randn(C) for _ in range(5)),
                         randn(1), randn(1)]),
    }


def _floats(out):
    return [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None and t.is_floating_point()]


@pytest.mark.parametrize("name", ["w4_linear", "beam_step", "premix_step"])
def test_a_gradient_raises_instead_of_being_lost(name):
    fn, ts = _calls()[name]
    want = fn(*ts)
    for i in range(len(ts)):
        xs = [t.clone().requires_grad_(j == i) for j, t in enumerate(ts)]
        with torch.no_grad():
            got = fn(*xs)
        assert type(got) is type(want) and not any(t.requires_grad for t in _floats(got))
        got = fn(*xs)
        assert type(got) is type(want)
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a, b)
        for t in _floats(got):
            assert t.requires_grad
            with pytest.raises(RuntimeError, match=f"{name} is for inference"):
                t.sum().backward(retain_graph=True)
        assert xs[i].grad is None


@pytest.mark.parametrize("name", ["w4_linear", "beam_step", "premix_step"])
def test_a_tangent_raises_instead_of_being_lost(name):
    fn, ts = _calls()[name]
    with fwd.dual_level():
        for i in range(len(ts)):
            xs = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(ts)]
            with pytest.raises(RuntimeError):
                fn(*xs)
        out = fn(*ts)
    for a, b in zip(_floats(out), _floats(fn(*ts))):
        assert torch.equal(a, b)


def test_refusals_come_before_the_gradients():
    fn, (x, b, r) = _calls()["w4_linear"]
    with pytest.raises(ValueError, match="bias must be"):
        fn(x.requires_grad_(), b[:3], r)
