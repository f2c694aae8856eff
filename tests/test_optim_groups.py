"""Groups and states of optim.AdamW on the host, where no step runs: what it takes over, refuses and looks at."""
import pytest
import torch

from atomic_gdn2.optim import AdamW


@pytest.fixture
def on_the_host(monkeypatch):
    """(parameters of any device: nothing here reaches a kernel)"""
    monkeypatch.setattr(AdamW, "_check", lambda self, p: None)


def _params(*sizes):
    return [torch.nn.Parameter(torch.linspace(-1, 1, n)) for n in sizes]


def _stepped(ps, **kw):
    opt = torch.optim.AdamW(ps, lr=1e-2, **kw)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    return opt


@pytest.mark.parametrize("key", ["maximize", "amsgrad"])
def test_other_steps_of_torch_are_refused(on_the_host, key):
    """A checkpoint of a run that maximised is not one to minimise with; amsgrad keeps a maximum that has no place here."""
    ref = _stepped(_params(5, 3), **{key: True})
    ps = _params(5, 3)
    opt = AdamW(ps, lr=0.5)
    with pytest.raises(ValueError, match=key):
        opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5 and not opt.state and key not in opt.param_groups[0]
    with pytest.raises(ValueError, match=key):
        AdamW([{"params": ps, key: True}])
    with pytest.raises(ValueError, match=key):
        opt.add_param_group({"params": _params(2), key: True})
    assert len(opt.param_groups) == 1


def test_states_of_a_plain_run_are_taken_over(on_the_host):
    ref = _stepped(_params(5, 3))
    ps = _params(5, 3)
    opt = AdamW(ps, lr=0.5)
    opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 1e-2
    for p, q in zip(ps, ref.param_groups[0]["params"]):
        assert all(torch.equal(opt.state[p][k], ref.state[q][k]) for k in ("step", "exp_avg", "exp_avg_sq"))


def test_weight_decay_in_the_gradient_is_refused(on_the_host):
    """Adam adds its decay to the gradient; without a decay it takes AdamW's steps."""
    def adam(wd):
        ps = _params(4)
        opt = torch.optim.Adam(ps, lr=1e-2, weight_decay=wd)
        ps[0].grad = torch.ones_like(ps[0])
        opt.step()
        return opt.state_dict()

    opt = AdamW(_params(4))
    with pytest.raises(ValueError, match="decoupled"):
        opt.load_state_dict(adam(0.1))
    opt.load_state_dict(adam(0.0))
    assert opt.param_groups[0]["weight_decay"] == 0.0
