"""What linear, cross_entropy, AdamW and their entry points refuse; nothing here reaches a GPU."""
import ctypes

import pytest
import torch

from atomic_gdn2 import _lib, e2e_lm
from atomic_gdn2.linear import linear
from atomic_gdn2.losses import cross_entropy
from atomic_gdn2.optim import AdamW


def test_linear_arguments():
    x, w = torch.zeros(3, 8), torch.zeros(8, 4)
    with pytest.raises(ValueError, match="ROCm device"):
        linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="relu6")
    with pytest.raises(TypeError, match="x must be"):
        linear(x.double(), w)
    with pytest.raises(TypeError, match="weight must be"):
        linear(x, w.bfloat16())
    with pytest.raises(TypeError, match="out_dtype"):
        linear(x, w, out_dtype=torch.bfloat16)
    for bad in (w[0], w[:0], torch.zeros(8, 0), w[None]):
        with pytest.raises(ValueError, match="weight must be"):
            linear(x, bad)
    for bad in (torch.zeros(3, 7), torch.zeros(())):
        with pytest.raises(ValueError, match="x must be"):
            linear(bad, w)
    for bad in (torch.zeros(5), torch.zeros(1, 4), torch.zeros(())):
        with pytest.raises(ValueError, match="bias must be"):
            linear(x, w, bias=bad)
    with pytest.raises(TypeError, match="bias must be"):
        linear(x, w, bias=torch.zeros(4).half())
    for bad in (torch.zeros(4), torch.zeros(3, 8), torch.zeros(2, 4)):
        with pytest.raises(ValueError, match="residual must be"):
            linear(x, w, residual=bad)


def test_cross_entropy_arguments():
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="ROCm device"):
        cross_entropy(x, t)
    with pytest.raises(TypeError, match="logits"):
        cross_entropy(x.double(), t)
    for bad in (t.float(), t.bool()):
        with pytest.raises(TypeError, match="targets"):
            cross_entropy(x, bad)
    for a, b in ((x, t[:2]), (x, t[None]), (x[:0], t[:0]), (torch.zeros(3, 0), t), (torch.zeros(()), t)):
        with pytest.raises(ValueError, match="logits must be"):
            cross_entropy(a, b)
    with pytest.raises(ValueError, match="reduction"):
        cross_entropy(x, t, reduction="max")
    for e in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="label_smoothing"):
            cross_entropy(x, t, label_smoothing=e)
    for z in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="z_loss"):
            cross_entropy(x, t, z_loss=z)


def test_adamw_arguments():
    p = torch.nn.Parameter(torch.zeros(4))
    for kw, what in ((dict(state_bits=16), "state_bits"), (dict(max_norm=0.0), "max_norm"), (dict(max_norm=-1.0), "max_norm"),
                     (dict(lr=-1.0), "lr"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1.0), "eps"),
                     (dict(weight_decay=-1.0), "weight_decay")):
        with pytest.raises(ValueError, match=what):
            AdamW([p], **kw)
    with pytest.raises(ValueError, match="ROCm device"):
        AdamW([p])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))])


def test_model_arguments():
    with pytest.raises(ValueError, match="products"):
        e2e_lm.LMConfig(products="float8")
    model = e2e_lm.LM(e2e_lm.LMConfig(vocab_size=16, d_model=8, n_heads=2, d_head=4, n_layers=1, products="bfloat16"), lambda q, k, v, w, b, g: v)
    with pytest.raises(ValueError, match="bfloat16"):
        model(torch.zeros(1, 4, dtype=torch.int64))
    model = e2e_lm.LM(e2e_lm.LMConfig(vocab_size=16, d_model=8, n_heads=2, d_head=4, n_layers=1), lambda q, k, v, w, b, g: v)
    with pytest.raises(ValueError, match="state_bits"):
        e2e_lm.TrainStep(model, state_bits=8)


def _status(fn, *args):
    return getattr(_lib.lib(), fn)(*args)


_AT = 1 << 20         # an address that is looked at, never read: every call here is refused before its launch


def _product(**kw):
    a = dict(M=4, K=16, N=8, form=0, dtype=1, out_dtype=1, bias_dtype=1, activation=0, lda=16, ldb=8, ldr=8, a=_AT, b=_AT, bias=None,
             residual=None, y=_AT, z=None)
    return _lib.Gdn2Product(**{**a, **kw})


@pytest.mark.parametrize("kw", [
    dict(M=0), dict(K=-1), dict(N=0), dict(M=2 ** 28), dict(M=2 ** 27, N=2 ** 27, ldb=2 ** 27), dict(form=3), dict(form=-1), dict(dtype=3),
    dict(out_dtype=2), dict(bias=_AT, bias_dtype=2), dict(activation=4), dict(form=2, lda=4, activation=1), dict(form=2, lda=4, bias=_AT),
    dict(form=2, lda=4, z=_AT), dict(lda=15), dict(ldb=7), dict(form=1, ldb=15), dict(form=2, lda=3), dict(residual=_AT, ldr=7), dict(a=None),
    dict(b=None), dict(y=None), dict(a=_AT + 1), dict(z=_AT + 1), dict(y=_AT + 2, out_dtype=0), dict(bias=_AT + 2, bias_dtype=0),
    dict(dtype=0, out_dtype=0, bias_dtype=0, a=_AT + 2)])
def test_gdn2_linear_refuses(kw):
    p = _product(**kw)
    assert _status("gdn2_linear", ctypes.byref(p), ctypes.c_void_p(_AT), None) in (1, 2)
    assert _lib.lib().gdn2_last_error()


def test_gdn2_linear_workspace_is_asked_for():
    p = _product(M=64, K=4096, N=64, ldb=64, lda=4096)          # a sum in parts
    assert _lib.lib().gdn2_linear_workspace_bytes(ctypes.byref(p)) > 0
    assert _status("gdn2_linear", ctypes.byref(p), None, None) == 1
    assert _status("gdn2_linear", ctypes.byref(p), ctypes.c_void_p(_AT + 8), None) == 1
    assert _status("gdn2_linear", None, None, None) == 1
    assert _lib.lib().gdn2_linear_workspace_bytes(None) == 0


@pytest.mark.parametrize("kw", [dict(M=0), dict(N=0), dict(dtype=3), dict(dy_dtype=2), dict(bias_dtype=2), dict(activation=5), dict(dy=None),
                                dict(activation=1, z=None), dict(dz=None, dbias=None), dict(dz=_AT + 1)])
def test_gdn2_linear_slope_refuses(kw):
    a = dict(M=4, N=8, dtype=1, dy_dtype=1, bias_dtype=1, activation=1, dy=_AT, z=_AT, dz=_AT, dbias=_AT)
    assert _status("gdn2_linear_slope", ctypes.byref(_lib.Gdn2Slope(**{**a, **kw})), ctypes.c_void_p(_AT), None) in (1, 2)


@pytest.mark.parametrize("kw", [
    dict(rows=0), dict(V=0), dict(V=2 ** 30 + 1), dict(dtype=4), dict(target_type=3), dict(reduction=3), dict(upstream_ld=1),
    dict(upstream_ld=2, reduction=0), dict(smoothing=1.5), dict(smoothing=float("nan")), dict(z_loss=-1.0), dict(ld=7), dict(logits=None),
    dict(targets=None), dict(loss=None, dlogits=None), dict(logits=_AT + 1), dict(targets=_AT + 4), dict(loss=_AT + 2)])
def test_gdn2_cross_entropy_refuses(kw):
    a = dict(rows=4, V=8, dtype=1, target_type=2, reduction=2, upstream_ld=0, smoothing=0.0, z_loss=0.0, ld=8, ignore_index=-100, logits=_AT,
             targets=_AT, upstream=None, loss=_AT, dlogits=_AT)
    assert _status("gdn2_cross_entropy", ctypes.byref(_lib.Gdn2Loss(**{**a, **kw})), ctypes.c_void_p(_AT), None) in (1, 2)
    assert _status("gdn2_cross_entropy", ctypes.byref(_lib.Gdn2Loss(**a)), None, None) == 1


@pytest.mark.parametrize("kw", [
    dict(numel=0), dict(m=None), dict(v=None), dict(m=_AT + 2), dict(dtype=3), dict(p=None), dict(g=None), dict(step=None), dict(dtype=1, master=None),
    dict(p=_AT + 2), dict(step=_AT + 2), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(lr=float("nan")), dict(weight_decay=-1.0)])
def test_gdn2_adamw_refuses(kw):
    a = dict(p=_AT, g=_AT, m=_AT, v=_AT, m_scale=None, v_scale=None, master=None, step=_AT, numel=8, ordinal=0, dtype=0, lr=1e-3, beta1=0.9,
             beta2=0.99, eps=1e-8, weight_decay=0.0)
    t = _lib.Gdn2AdamwTensor(**{**a, **kw})
    assert _status("gdn2_adamw", ctypes.byref(t), 1, 32, 0.0, None, ctypes.c_void_p(_AT), None) in (1, 2)
    ok = _lib.Gdn2AdamwTensor(**a)
    assert _status("gdn2_adamw", ctypes.byref(ok), 1, 8, 0.0, None, ctypes.c_void_p(_AT), None) == 1       # (no scales)
    assert _status("gdn2_adamw", ctypes.byref(ok), 1, 16, 0.0, None, ctypes.c_void_p(_AT), None) == 1
    assert _status("gdn2_adamw", ctypes.byref(ok), 0, 32, 0.0, None, ctypes.c_void_p(_AT), None) == 1
    assert _status("gdn2_adamw", ctypes.byref(ok), 1, 32, 0.0, None, None, None) == 1


def test_scale_rows_refuses():
    for args in ((None, 0, 4, 8, _AT, 0), (_AT, 3, 4, 8, _AT, 0), (_AT, 0, 0, 8, _AT, 0), (_AT, 0, 4, 0, _AT, 0), (_AT, 0, 4, 8, None, 0),
                 (_AT, 0, 4, 8, _AT, 2), (_AT + 2, 0, 4, 8, _AT, 0), (_AT, 0, 4, 8, _AT + 2, 0)):
        assert _status("gdn2_scale_rows", *args, None) in (1, 2)
