"""Sizes that 32 bits do not hold: refused by linear and cross_entropy, never cut.  (Expanded tensors of one element.)"""
import pytest
import torch

from atomic_gdn2.linear import linear
from atomic_gdn2.losses import cross_entropy

FAR = 2 ** 32 + 4


def test_products():
    one = torch.zeros((1, 1))
    for x, w in ((one.expand(FAR, 1), one), (one.expand(2, FAR), one.expand(FAR, 1)), (one, one.expand(1, FAR)),
                 (one.expand(2 ** 27 + 1, 1), one), (one.expand(2 ** 20, 1)[None].expand(2 ** 14, 2 ** 20, 1), one)):
        with pytest.raises(ValueError, match="2\\^27"):
            linear(x, w)


def test_losses():
    one, zero = torch.zeros((1, 1)), torch.zeros(1, dtype=torch.int64)
    for x, t in ((one.expand(FAR, 1), zero.expand(FAR)), (one.expand(1, FAR), zero), (one.expand(2 ** 30 + 1, 1), zero.expand(2 ** 30 + 1)),
                 (one.expand(2 ** 16, 2 ** 16, 1), zero.expand(2 ** 16, 2 ** 16))):
        with pytest.raises(ValueError, match="2\\^30"):
            cross_entropy(x, t)
