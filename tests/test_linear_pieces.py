"""float32 products as six products of bfloat16 pieces: what the three others would have added.

A value of [1, 2) cut to eight significant bits leaves less than 2^-7, and that cut to eight less than 2^-15, which has eight bits
or fewer.  Left out are mid lo + lo mid + lo lo < 2 2^-7 2^-15 (1 - 2^-8)^2 + 2^-30 < 2^-21 of products of at least 1."""
import numpy as np
import pytest

WORST = np.uint32(0x3F80FFFF).view(np.float32)          # 1 + 2^-7 - 2^-23: every bit behind the first piece is set


def _cut(x):
    top = lambda v: (v.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)  # noqa: E731
    hi = top(x)
    mid = top(x - hi)
    lo = top(x - hi - mid)
    assert np.array_equal(hi.astype(np.float64) + mid + lo, x.astype(np.float64))
    return [p.astype(np.float64) for p in (hi, mid, lo)]


def test_what_is_left_out():
    rng = np.random.default_rng(0)
    x = np.concatenate([np.array([WORST], np.float32), np.float32(1.0) + rng.random(2000, dtype=np.float32),
                        (np.uint32(0x3F800000) | (rng.integers(0, 128, 500, dtype=np.uint32) << 16) | np.uint32(0xFFFF)).view(np.float32)])
    a, b = _cut(x), _cut(x)
    left = sum(np.outer(a[i], b[j]) for i, j in ((1, 2), (2, 1), (2, 2)))
    share = left / np.outer(x.astype(np.float64), x.astype(np.float64))
    assert (left >= 0).all() and share.max() < 2.0 ** -21
    assert share[0, 0] > 2.0 ** -21.05              # (close to it: half of it would not be a bound)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(4, 4096, 512), (512, 512, 512), (1024, 4096, 512), (301, 7001, 331), (4096, 4096, 4096), (2050, 1000, 1030)])
def test_operands_of_one_sign_with_every_bit_set(M, K, N):
    """The worst case of each way that float32 takes: nothing cancels.  What is left out, and the sums' own
    (K / 32 + 12) 2^-22."""
    import torch
    from atomic_gdn2.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(K)
    bits = lambda *s: (torch.randint(0, 128, s, device="cuda", generator=gen, dtype=torch.int32) << 16 | 0x3F80FFFF).view(torch.float32)  # noqa: E731
    x, w = bits(M, K), bits(K, N)
    y = linear(x, w)
    want = x.double() @ w.double()
    assert ((y.double() - want).abs() <= (2.0 ** -21 + (K / 32 + 12) * 2.0 ** -22) * want).all()
