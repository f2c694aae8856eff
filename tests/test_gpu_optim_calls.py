"""Calls of optim.AdamW beside the ordinary step."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _opt(sizes, seed=0, dt=torch.float32, **kw):
    from atomic_gdn2.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen).to(dt)) for n in sizes]
    return ps, AdamW(ps, lr=1e-2, **kw)


def test_states_are_unpacked_into_a_tensor_for_each_parameter():
    """Lists of as many tensors as there are states are refused, whatever their sizes, and left as they are."""
    ps, opt = _opt([300, 300, 50], state_bits=8)
    ps[1].grad = torch.randn_like(ps[1])
    opt.step()
    few = [[torch.full((300,), 7.0, device="cuda")] for _ in range(2)]
    with pytest.raises(ValueError, match="each parameter"):
        opt.unpack_states(*few)
    assert all((t == 7.0).all() for out in few for t in out)
    outs = [[torch.full_like(p, 7.0) for p in ps] for _ in range(2)]
    opt.unpack_states(*outs)
    assert not any(out[i].any() for out in outs for i in (0, 2)) and all(out[1].any() for out in outs)
    assert all(torch.equal(a, b) for got, want in zip(outs, opt.unpack_states()) for a, b in zip(got, want))
    for p in ps:
        p.grad = torch.randn_like(p)
    opt.step()
    opt.unpack_states(*outs)
    assert all(torch.equal(a, b) for got, want in zip(outs, opt.unpack_states()) for a, b in zip(got, want))
