"""Every bit of a float32 x takes part in a 4-bit product, in each of its kernels.

A row with one entry that is not zero has a result of one term, s (q - z) x.  Its products are exact, x's pieces
(three of 8 bits) are added up as q x and as x or z x: at most 12 additions and 4 roundings of the scaling, 2^-23
of |s| (q + |z|) |x| each at most.  Where z or q is 0, x without its lowest piece is 2^-17 off on
average, four times the bound: an oracle that drops that piece fails, which is checked too."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def _cut(x, bits):
    """x without its lowest bits."""
    return (x.view(torch.int32) & -(1 << bits)).view(torch.float32)


# M, K, N: rows (four, two and one steps of the sum an operand), sums in parts, tiles, many rows; x read in
# sixteens of bytes and not
SHAPES = [(1, 512, 640), (7, 512, 640), (16, 512, 640), (12, 9000, 60), (40, 8200, 520), (520, 512, 4100), (521, 501, 4100),
          (1500, 512, 4100), (1500, 301, 4100)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_each_piece_of_a_float32_row_counts(M, K, N, group):
    from atomic_gdn2.w4 import pack_w4, w4_linear
    print(f"[gpu-test] w4 pieces {M}x{K}x{N} group {group}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(M + K + N + group)
    groups = -(-K // group)
    at = torch.randint(0, K, (M,), device="cuda", generator=gen)
    v = torch.randn(M, device="cuda", generator=gen) * 8
    x = torch.zeros((M, K), device="cuda")
    x[torch.arange(M, device="cuda"), at] = v
    scales = (torch.rand((groups, N), device="cuda", generator=gen) + 0.5).to(torch.bfloat16)
    codes = torch.randint(1, 16, (K, N), dtype=torch.uint8, device="cuda", generator=gen)
    zeros = torch.randint(1, 16, (groups, N), device="cuda", generator=gen).to(torch.bfloat16)
    for kind, c, z in (("codes", codes, zeros * 0), ("zeros", codes * 0, zeros), ("both", codes, zeros)):
        y = w4_linear(x, pack_w4(c, scales, z, group)).double()
        s, zz, q = scales[at // group].double(), z[at // group].double(), c[at].double()
        bound = 16 * 2.0 ** -23 * s * (q + zz) * v.double().abs()[:, None]
        value = lambda t: s * (q - zz) * t.double()[:, None]  # noqa: E731
        assert bool(((y - value(v)).abs() <= bound).all()), kind
        if kind != "both" and M >= 7:
            assert float(((value(_cut(v, 8)) - value(v)).abs() > bound).double().mean()) > 0.3, "the bound would not show a lost piece"
