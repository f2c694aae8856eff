"""Weights at the ends of float32's range: the quantiser's scales and zeros stay finite, and what it keeps
lies within a level of the matrix."""
import pytest
import torch

from atomic_gdn2 import w4


def _check(w, group, symmetric):
    W = w4.quantize_w4(w, group, symmetric)
    _, scales, zeros = W.unpack()
    assert bool(torch.isfinite(scales).all()) and bool((scales > 0).all()) and bool(torch.isfinite(zeros).all())
    d = W.dequantize()
    assert bool(torch.isfinite(d).all())
    return d


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("least", [1e-45, 2e-40, 6e-40, 1e-38])
def test_subnormal_groups(least, symmetric):
    # bfloat16's smallest positive scale is 2^-133; a level of it at most, or the entry itself, is lost
    w = torch.zeros(64, 3)
    w[1:5, 0] = least
    w[0, 1], w[7, 1] = -least, least
    w[:, 2] = torch.linspace(-1, 1, 64)
    w[32:, :2] = 0.25
    d = _check(w, 32, symmetric)
    assert float((d - w)[:32, :2].abs().max()) <= 15 * 2.0 ** -134 + least * 0.6
    assert torch.equal(d[32:, 2], w4.quantize_w4(w[:, 2:], 32, symmetric).dequantize()[32:, 0])


@pytest.mark.parametrize("symmetric", [False, True])
def test_groups_whose_range_is_above_float32(symmetric):
    w = torch.zeros(64, 2)
    w[0, 0], w[1, 0], w[2, 0] = 3e38, -3e38, 1e38
    w[40:, 1] = 0.5
    d = _check(w, 32, symmetric)
    step = 6e38 / 15
    assert float((d - w)[:32, 0].double().abs().max()) <= step * (1 + 15 * 2 ** -9)
    assert float((d - w)[32:, 1].abs().max()) < 0.05


def test_weights_that_float32_cannot_hold_are_refused():
    w = torch.zeros(32, 1, dtype=torch.float64)
    w[3] = 1e39
    with pytest.raises(ValueError, match="finite"):
        w4.quantize_w4(w, 32)
