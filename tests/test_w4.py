"""Host side of the 4-bit products (atomic_gdn2.w4): the layout round trip, the quantiser's grid, and
what the entry points refuse."""
import pytest
import torch

from atomic_gdn2 import w4


@pytest.mark.parametrize("K,N,group", [(1, 1, 32), (128, 16, 128), (130, 5, 64), (1000, 33, 32), (257, 17, 128)])
def test_pack_keeps_codes_scales_and_zeros(K, N, group):
    gen = torch.Generator().manual_seed(K + N)
    groups = -(-K // group)
    codes = torch.randint(0, 16, (K, N), dtype=torch.uint8, generator=gen)
    scales = torch.randn(groups, N, generator=gen).to(torch.bfloat16)
    zeros = torch.randint(0, 16, (groups, N), generator=gen)
    W = w4.pack_w4(codes, scales, zeros, group)
    c, s, z = W.unpack()
    assert torch.equal(c, codes) and torch.equal(s, scales) and torch.equal(z, zeros.to(torch.bfloat16))
    assert W.shape == (K, N) and W.group_size == group
    want = (codes.float() - zeros.float().repeat_interleave(group, 0)[:K]) * scales.float().repeat_interleave(group, 0)[:K]
    assert torch.equal(W.dequantize(), want)
    assert torch.equal(w4.pack_w4(codes.long(), scales, None, group).unpack()[2], torch.full_like(scales, 8))


def test_layout_of_one_entry():
    """Row 32 j + 8 c + e of column r is element e of word j of lane 16 c + r (include/gdn2.h)."""
    for j, c, e, r in ((0, 0, 0, 0), (3, 2, 1, 15), (1, 3, 4, 7), (2, 1, 7, 9)):
        codes = torch.zeros((128, 16), dtype=torch.uint8)
        codes[32 * j + 8 * c + e, r] = 13
        q = w4.pack_w4(codes, torch.ones(1, 16), group_size=128).q
        nibble = 2 * e if e < 4 else 2 * e - 7
        want = torch.zeros_like(q)
        want[0, 0, 16 * c + r, j] = 13 << (4 * nibble) if nibble < 7 else (13 << 28) - (1 << 32)
        assert torch.equal(q, want), (j, c, e, r)


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_rounds_to_the_nearest_level(group, symmetric):
    gen = torch.Generator().manual_seed(3)
    w = torch.randn(200, 12, generator=gen) * 0.1
    w[:, 1] = 0                           # a column of zeros
    w[:, 2] = w[:, 2].abs() + 0.3         # 0 lies outside the entries' range
    w[:, 3] = -0.25
    W = w4.quantize_w4(w, group, symmetric)
    _, scales, _ = W.unpack()
    # half a step; the scale's own rounding to 8 bits can cut the range short by 15 2^-9 steps, and the
    # zero's rounding to a whole number by half a step
    step = scales.float().repeat_interleave(group, 0)[:200]
    err = (W.dequantize() - w).abs()
    assert bool((err <= step * (0.5 + 15 * 2 ** -9 + (0.0 if symmetric else 0.5)) + 1e-7).all())
    assert bool((W.dequantize()[:, 1] == 0).all())
    assert float((err / step).pow(2).mean().sqrt()) < 0.32     # a uniform error of one step: 0.289


def test_refusals_of_pack_and_quantize():
    codes, scales = torch.zeros((64, 8), dtype=torch.uint8), torch.ones(1, 8)
    for bad in (0, 16, 96, 256):
        with pytest.raises(ValueError, match="group_size"):
            w4.pack_w4(codes, scales, group_size=bad)
    with pytest.raises(ValueError, match="codes must be"):
        w4.pack_w4(codes[0], scales, group_size=64)
    with pytest.raises(TypeError, match="whole numbers"):
        w4.pack_w4(codes.float(), scales, group_size=64)
    with pytest.raises(ValueError, match="0 .. 15"):
        w4.pack_w4(codes + 16, scales, group_size=64)
    with pytest.raises(ValueError, match="0 .. 15"):
        w4.pack_w4(codes.to(torch.int8) - 1, scales, group_size=64)
    with pytest.raises(ValueError, match="scales must be"):
        w4.pack_w4(codes, scales, group_size=32)
    with pytest.raises(ValueError, match="zeros must be"):
        w4.pack_w4(codes, scales, torch.ones(2, 8), group_size=64)
    with pytest.raises(ValueError, match="finite"):
        w4.quantize_w4(torch.full((4, 4), float("nan")))
    with pytest.raises(ValueError, match="floating-point"):
        w4.quantize_w4(codes)


def test_refusals_of_the_product():
    W = w4.quantize_w4(torch.randn(64, 8), 64)
    x = torch.randn(3, 64)
    with pytest.raises(TypeError, match="W4Weight"):
        w4.w4_linear(x, torch.randn(64, 8))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        w4.w4_linear(x.double(), W)
    with pytest.raises(ValueError, match=r"x must be \(..., 64\)"):
        w4.w4_linear(x[:, :63], W)
    with pytest.raises(ValueError, match="bias must be"):
        w4.w4_linear(x, W, bias=torch.zeros(7))
    with pytest.raises(ValueError, match="residual must be"):
        w4.w4_linear(x, W, residual=torch.zeros(3, 7))
    with pytest.raises(ValueError, match="ROCm device"):
        w4.w4_linear(x, W)
    with pytest.raises(ValueError, match="is on meta"):
        w4.w4_linear(x, W, bias=torch.zeros(8, device="meta"))
