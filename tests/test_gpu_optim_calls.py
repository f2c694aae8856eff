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


@pytest.mark.parametrize("bits", [32, 8])
def test_a_first_step_is_not_captured(bits):
    """Its states would be made anew, as zeros, by every replay."""
    ps, opt = _opt([300, 50], dt=torch.bfloat16, state_bits=bits, max_norm=1.0)
    ps[0].grad = torch.randn_like(ps[0])
    opt.step()
    ps[1].grad = torch.randn_like(ps[1])
    before = [p.detach().clone() for p in ps]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.stream(s), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            opt.step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, ps)) and opt.state[ps[0]]["step"].item() == 1 and not opt.state[ps[1]]
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        opt.step()
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        graph.replay()
    assert [opt.state[p]["step"].item() for p in ps] == [5, 4]


@pytest.mark.parametrize("bits", [32, 8])
def test_an_empty_group_comes_first(bits):
    """(as where parameters are split by their decay and one side has none)"""
    from atomic_gdn2.optim import AdamW
    ps, one = _opt([300, 50], seed=1, state_bits=bits)
    qs, _ = _opt([300, 50], seed=1)
    two = AdamW([{"params": [], "weight_decay": 0.0}, {"params": qs}], lr=1e-2, state_bits=bits)
    for p, q in zip(ps, qs):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    one.step(), two.step(), two.step(), one.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    if bits == 8:
        assert all(torch.equal(a, b) for got, want in zip(two.unpack_states(), one.unpack_states()) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="device"):
        two.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))]})
    assert len(two.param_groups) == 2
    three = AdamW([{"params": []}])
    three.add_param_group({"params": qs})


def test_norm_of_no_gradients():
    """A step without a gradient has the norm 0, not that of the step before."""
    ps, opt = _opt([300, 50], max_norm=1.0)
    ps[0].grad = torch.ones_like(ps[0])
    opt.step()
    assert opt.norm.item() > 17
    opt.zero_grad()
    before = [p.detach().clone() for p in ps]
    opt.step()
    assert opt.norm.item() == 0.0 and opt.norm.dtype == torch.float32 and opt.norm.shape == () and opt.norm.is_cuda
    assert all(torch.equal(a, b) for a, b in zip(before, ps)) and opt.state[ps[0]]["step"].item() == 1
    qs, other = _opt([300])
    other.step()
    assert other.norm is None
    from atomic_gdn2.optim import AdamW
    empty = AdamW([{"params": []}], max_norm=1.0)
    empty.step()
    assert empty.norm is None


def _set_bad(p, at, value):
    p.grad = torch.linspace(-1, 1, p.numel(), device="cuda")
    p.grad[at] = value


def _bad(n, at, bits):
    want = torch.zeros(n, dtype=torch.bool, device="cuda")
    want[slice(at // 256 * 256, at // 256 * 256 + 256) if bits == 8 else at] = True
    return want


@pytest.mark.parametrize("bits", [32, 8])
def test_an_infinite_gradient_makes_the_factor_0(bits):
    """max_norm / infinity: NaN where 0 times the infinity is, a step of no gradient everywhere else."""
    ps, opt = _opt([1000, 700], max_norm=1.0, state_bits=bits)
    qs, ref = _opt([1000, 700], max_norm=1.0, state_bits=bits)
    _set_bad(ps[0], 600, float("inf"))
    ps[1].grad = torch.ones_like(ps[1])
    for q in qs:
        q.grad = torch.zeros_like(q)
    opt.step(), ref.step()
    assert opt.norm.item() == float("inf")
    one = torch.zeros(1000, dtype=torch.bool, device="cuda")
    one[600] = True
    assert torch.equal(torch.isnan(ps[0].detach()), one)
    assert torch.equal(ps[0].detach()[~one], qs[0].detach()[~one]) and torch.equal(ps[1], qs[1])
    _set_bad(ps[0], 600, 0.0)
    opt.step()
    assert torch.equal(torch.isnan(ps[0].detach()), _bad(1000, 600, bits)) and torch.isfinite(ps[1].detach()).all()


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("bits", [32, 8])
def test_an_infinite_max_norm_scales_nothing(bits, value):
    """The norm is formed, infinite or not a number, and every other element steps as without max_norm."""
    ps, opt = _opt([1000, 700], max_norm=float("inf"), state_bits=bits)
    qs, ref = _opt([1000, 700], state_bits=bits)
    for a, b in (ps, qs):
        _set_bad(a, 600, value)
        b.grad = torch.ones_like(b)
    for _ in range(2):
        opt.step(), ref.step()
    assert str(opt.norm.item()) == str(value)
    for p, q in zip(ps, qs):
        assert torch.equal(torch.isnan(p.detach()), torch.isnan(q.detach()))
        assert torch.equal(p.detach().nan_to_num(), q.detach().nan_to_num())
    assert torch.equal(~torch.isfinite(ps[0].detach()), _bad(1000, 600, bits)) and torch.isfinite(ps[1].detach()).all()
