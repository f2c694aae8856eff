"""A ``W4Weight`` whose tensors do not fit its sizes is refused: the kernels' bounds come from the sizes."""
import numpy as np
import pytest
import torch

from atomic_gdn2 import w4


def _parts(K=200, N=40, group=64, device="cpu"):
    W = w4.pack_w4(torch.randint(0, 16, (K, N), dtype=torch.uint8, device=device),
                   torch.ones((-(-K // group), N), device=device), group_size=group)
    return W.q, W.meta, K, N, group


def test_parts_of_a_packed_weight_are_taken():
    q, meta, K, N, group = _parts()
    W = w4.W4Weight(q, meta, K, N, group)
    assert W.shape == (K, N) and torch.equal(W.dequantize(), w4.W4Weight(q.clone(), meta.clone(), K, N, group).dequantize())
    assert w4.W4Weight(q, meta, 129, 33, group).shape == (129, 33)        # (the same blocks)
    assert type(w4.W4Weight(q, meta, np.int64(K), np.int32(N), np.int64(group)).group_size) is int
    assert w4.quantize_w4(torch.randn(64, 8), np.int64(32)).group_size == 32


@pytest.mark.parametrize("what,change", [
    ("meta", lambda q, m, K, N, g: (q, m, K, N, 32)),             # another group size: twice the rows of meta
    ("meta", lambda q, m, K, N, g: (q, m, K, N, 128)),
    ("q", lambda q, m, K, N, g: (q, m, K + 128, N, g)),
    ("q", lambda q, m, K, N, g: (q, m, 128, N, g)),
    ("q", lambda q, m, K, N, g: (q, m, K, N + 16, g)),
    ("q", lambda q, m, K, N, g: (q[:-1], m, K, N, g)),
    ("q", lambda q, m, K, N, g: (q.flatten(), m, K, N, g)),
    ("meta", lambda q, m, K, N, g: (q, m[:, :-1].contiguous(), K, N, g)),
    ("q", lambda q, m, K, N, g: (q.long(), m, K, N, g)),
    ("meta", lambda q, m, K, N, g: (q, m.float(), K, N, g)),
    ("q", lambda q, m, K, N, g: (q.transpose(2, 3).contiguous().transpose(2, 3), m, K, N, g)),
    ("meta", lambda q, m, K, N, g: (q, m[:1].expand_as(m), K, N, g)),
    ("q", lambda q, m, K, N, g: (q.numpy(), m, K, N, g)),
    ("is on", lambda q, m, K, N, g: (q, m.to("meta"), K, N, g)),
    ("group_size", lambda q, m, K, N, g: (q, m, K, N, 16)),
    ("group_size", lambda q, m, K, N, g: (q, m, K, N, 64.0)),
    ("in_features", lambda q, m, K, N, g: (q, m, 0, N, g)),
    ("out_features", lambda q, m, K, N, g: (q, m, K, 40.0, g)),
])
def test_parts_that_do_not_fit_are_refused(what, change):
    with pytest.raises((ValueError, TypeError), match=what):
        w4.W4Weight(*change(*_parts()))


def test_a_weight_changed_afterwards_is_refused():
    W = w4.W4Weight(*_parts())
    W.group_size = 32
    with pytest.raises(ValueError, match="meta"):
        w4.w4_linear(torch.randn(2, 200), W)


@pytest.mark.gpu
def test_a_weight_changed_afterwards_is_refused_before_a_launch():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    q, meta, K, N, group = _parts(device="cuda")
    x = torch.randn((2, K), device="cuda")
    W = w4.W4Weight(q, meta, K, N, group)
    want = w4.w4_linear(x, W)
    for name, value, what in (("group_size", 32, "meta"), ("q", q[:-1], "q"), ("meta", meta[:, :1].contiguous(), "meta"),
                              ("out_features", N + 16, "q"), ("meta", meta.long(), "meta"), ("group_size", 48, "group_size")):
        W = w4.W4Weight(q, meta, K, N, group)
        setattr(W, name, value)
        with pytest.raises((ValueError, TypeError), match=what):
            w4.w4_linear(x, W)
    W = w4.W4Weight(q, meta, K, N, group)
    W.in_features = K + 128
    with pytest.raises(ValueError, match="q"):
        w4.w4_linear(torch.randn((2, K + 128), device="cuda"), W)
    assert torch.equal(want, w4.w4_linear(x, w4.W4Weight(q, meta, K, N, group)))
