"""cross_entropy under saved-tensor hooks: whatever they give back, the kernels get logits and targets in the form in which
they were saved."""
import pytest
import torch

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _spread_out(t):
    """t with another stride between its elements."""
    wide = t.new_zeros((*t.shape, 2))
    wide[..., 0] = t
    return wide[..., 0]


@pytest.mark.parametrize("hook", [lambda t: t, lambda t: t.to(torch.int32 if t.dtype == torch.int64 else torch.float64), _spread_out,
                                  lambda t: t[:1].expand(t.shape) if t.dim() == 2 else t.flip(0).flip(0)],
                         ids=["same", "types", "strides", "expanded"])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_what_the_backward_pass_hands_to_the_kernels(monkeypatch, hook, dtype):
    """(the kernels' arguments are looked at here, on the host; float16, and a second pass over a kept graph, form the gradient
    in the backward pass)"""
    from atomic_gdn2 import losses
    seen = []

    def run(x, targets, how, loss, dlogits, upstream=None, upstream_ld=0):
        seen.append((x, targets))
        for out in (loss, dlogits):
            if out is not None:
                out.zero_()

    monkeypatch.setattr(losses, "_run", run)
    x = torch.randn(4, 6).to(DTYPES[dtype]).requires_grad_(True)
    t = torch.tensor([1, 5, -100, 0])
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, hook):
        loss = losses._CrossEntropy.apply(x, t, (-100, 0.0, 0.0, 1))
    if dtype == "fp32":
        loss.grad_fn.grad = None            # (as after a first pass)
    loss.backward()
    assert len(seen) == 2
    got_x, got_t = seen[1]
    assert got_t.dtype == torch.int64 and got_t.device == t.device and got_t.is_contiguous() and torch.equal(got_t, t)
    assert got_x.dtype == x.dtype and got_x.device == x.device and got_x.shape == x.shape and got_x.stride() == (6, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_targets_left_on_the_host(dtype, strided):
    """Hooks that leave what was saved on the host, in other types: the same gradients, in a first and in a second pass."""
    from atomic_gdn2.losses import cross_entropy
    gen = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn((3, 9, 300), device="cuda", generator=gen).to(DTYPES[dtype]).requires_grad_(True)
    t = torch.randint(0, 300, (3, 8), device="cuda", generator=gen)
    logits = lambda: base[:, :-1] if strided else base[:, :-1].contiguous()  # noqa: E731
    want, = torch.autograd.grad(cross_entropy(logits(), t, label_smoothing=0.1), base)
    for pack in (lambda s: s.cpu(), lambda s: s.cpu().double() if s.is_floating_point() else s.cpu().to(torch.int32)):
        x = logits()
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda s: s):
            loss = cross_entropy(x, t, label_smoothing=0.1)
        for _ in range(2):
            got, = torch.autograd.grad(loss, base, retain_graph=True)
            assert torch.equal(got, want)
