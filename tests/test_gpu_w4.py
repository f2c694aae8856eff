"""The 4-bit products on the GPU against the definition in 64 bits.

Bound of an entry's error: every product q x is exact and everything is summed in float32, so a sum of
t terms is within t 2^-23 of the sum of its terms' magnitudes (2^-23, not 2^-24: the matrix cores may
cut where they align).  Here t <= 3 group (three pieces of a float32 x) + groups + 16 (waves, bias,
residual), and the magnitudes are sum_k |s| (q + |z|) |x| plus those of bias and residual.  Then one
rounding to the result's type, which keeps order: the result lies between the rounded ends."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def _weights(K, N, group, zeros, gen):
    from atomic_gdn2.w4 import pack_w4
    groups = -(-K // group)
    codes = torch.randint(0, 16, (K, N), dtype=torch.uint8, device="cuda", generator=gen)
    scales = (torch.rand((groups, N), device="cuda", generator=gen) * 0.02 + 0.001).to(torch.bfloat16)
    scales *= torch.where(torch.rand((groups, N), device="cuda", generator=gen) < 0.1, -1.0, 1.0).to(torch.bfloat16)
    z = torch.randint(0, 16, (groups, N), device="cuda", generator=gen).to(torch.bfloat16) if zeros else None
    return codes, scales, z, pack_w4(codes, scales, z, group)


def _check(y, x, codes, scales, z, group, bias, residual, dtype):
    K = codes.shape[0]
    spread = lambda t: t.double().repeat_interleave(group, 0)[:K]  # noqa: E731
    s, zz = spread(scales), (8.0 if z is None else spread(z))
    x, q = x.double(), codes.double()
    want = x @ ((q - zz) * s)
    mag = x.abs() @ (s.abs() * (q + zz))
    for t in (bias, residual):
        if t is not None:
            want, mag = want + t.double(), mag + t.double().abs()
    terms = 3 * group + -(-K // group) + 16
    bound = terms * 2.0 ** -23 * mag
    lo, hi = ((want + side * bound).to(TYPES[dtype]) for side in (-1, 1))
    print(f"[gpu-test] rms error / rms bound {float((y.double() - want).norm() / bound.norm()):.3g}", flush=True)
    assert bool(((y >= lo) & (y <= hi)).all())


CASES = [
    # M, K, N, group: one entry, one tile, ragged in each direction, rows past a tile, long sums
    (1, 1, 1, 32), (1, 128, 16, 128), (1, 512, 4614, 64), (2, 40, 24, 32), (3, 1000, 777, 32), (5, 433, 50, 64),
    (16, 256, 96, 128), (17, 384, 33, 128), (31, 1001, 130, 64), (33, 160, 1, 32), (64, 2048, 48, 128),
    (65, 129, 257, 64), (1, 16384, 64, 128), (7, 5003, 200, 32), (129, 512, 640, 128), (300, 1032, 272, 64),
    (513, 264, 130, 32), (257, 640, 384, 128),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N,group", CASES)
def test_product_matches_the_definition(M, K, N, group, dtype):
    from atomic_gdn2.w4 import w4_linear
    print(f"[gpu-test] w4 {M}x{K}x{N} group {group} {dtype}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(M * 7 + K * 3 + N)
    dt = TYPES[dtype]
    for zeros, extras in ((True, False), (False, True)):
        codes, scales, z, W = _weights(K, N, group, zeros, gen)
        x = torch.randn((M, K), device="cuda", generator=gen).to(dt)
        bias = torch.randn(N, device="cuda", generator=gen).to(dt) if extras else None
        res = torch.randn((M, N), device="cuda", generator=gen).to(dt) if extras else None
        y = w4_linear(x, W, bias=bias, residual=res)
        assert y.dtype == dt and y.shape == (M, N)
        _check(y, x, codes, scales, z, group, bias, res, dtype)
        assert torch.equal(y, w4_linear(x, W, bias=bias, residual=res))        # the same bits again


# Long sums and many entries: one part, sums in parts, rows that 16-byte accesses cannot take, and tiles of
# many rows with x read in place (K a multiple of 128) and not, and with groups past a block of 32 of them
LARGE = [
    (17, 8321, 40, 32), (40, 9000, 130, 64), (500, 8200, 2040, 64), (520, 500, 4100, 128), (521, 501, 4100, 32),
    (2100, 100, 4100, 32), (1500, 256, 4100, 128), (1500, 264, 4096, 64), (1537, 301, 4111, 32), (1500, 1152, 4100, 32),
    (1290, 4229, 4800, 128), (1409, 2176, 4353, 64),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N,group", LARGE)
def test_large_product_matches_the_definition(M, K, N, group, dtype):
    test_product_matches_the_definition(M, K, N, group, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N", [(520, 500, 4100), (1500, 300, 4100), (1500, 256, 4100)])
def test_many_strided_rows_and_one_that_is_not_finite(M, K, N, dtype):
    from atomic_gdn2.w4 import w4_linear
    gen = torch.Generator(device="cuda").manual_seed(9)
    dt, group = TYPES[dtype], 64
    codes, scales, z, W = _weights(K, N, group, True, gen)
    wide = torch.randn((M, K + 13), device="cuda", generator=gen).to(dt)
    print(f"[gpu-test] w4 strided {M}x{K}x{N} {dtype}", flush=True)
    for x in (wide[:, 8:8 + K], wide[:, 3:3 + K]):
        y = w4_linear(x, W)
        _check(y, x, codes, scales, z, group, None, None, dtype)
        assert torch.equal(y, w4_linear(x.contiguous(), W))
    x = wide[:, 3:3 + K].contiguous()
    clean = w4_linear(x, W)
    x[1, 7], x[M - 1, K - 1] = float("nan"), float("inf")
    y = w4_linear(x, W)
    assert not torch.isfinite(y[1]).any() and not torch.isfinite(y[M - 1]).any()
    keep = [i for i in range(M) if i not in (1, M - 1)]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [1, 9, 40, 200])
def test_strided_and_misaligned_rows(M, dtype):
    from atomic_gdn2.w4 import w4_linear
    gen = torch.Generator(device="cuda").manual_seed(5)
    dt, K, N, group = TYPES[dtype], 264, 70, 32
    codes, scales, z, W = _weights(K, N, group, True, gen)
    wide = torch.randn((M, 2 * K + 3), device="cuda", generator=gen).to(dt)
    wres = torch.randn((M, N + 5), device="cuda", generator=gen).to(dt)
    print(f"[gpu-test] w4 strided M {M} {dtype}", flush=True)
    for x in (wide[:, 1:K + 1], wide[:, 8:8 + K], wide[:, ::2][:, :K], wide[:, :K].t().contiguous().t(),
              wide[:1, :K].expand(M, K)):
        y = w4_linear(x, W, residual=wres[:, 2:N + 2])
        _check(y, x, codes, scales, z, group, None, wres[:, 2:N + 2], dtype)
    # what a row gives does not depend on where it lies or on its neighbours
    x = wide[:, 8:8 + K]
    assert torch.equal(w4_linear(x.contiguous(), W), w4_linear(x, W))


def test_leading_dimensions_bias_cast_and_empty_rows():
    from atomic_gdn2.w4 import quantize_w4, w4_linear
    gen = torch.Generator(device="cuda").manual_seed(6)
    w = torch.randn((96, 40), device="cuda", generator=gen)
    W, x = quantize_w4(w, 32), torch.randn((2, 3, 96), device="cuda", generator=gen)
    y = w4_linear(x, W, bias=torch.ones(40, device="cuda", dtype=torch.float64))
    assert y.shape == (2, 3, 40)
    assert torch.equal(y.view(6, 40), w4_linear(x.view(6, 96), W, bias=torch.ones(40, device="cuda")))
    assert w4_linear(x[:0], W).shape == (0, 3, 40)
    assert w4_linear(x[0, 0], W).shape == (40,)
    assert float((y - 1 - x @ w).norm() / (x @ w).norm()) < 0.12       # 16 levels: about 0.08


def test_one_row_is_not_touched_by_another():
    """NaN and infinities stay in their rows."""
    from atomic_gdn2.w4 import w4_linear
    gen = torch.Generator(device="cuda").manual_seed(7)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        for M in (3, 40, 200):
            *_, W = _weights(200, 50, 64, True, gen)
            x = torch.randn((M, 200), device="cuda", generator=gen).to(dt)
            clean = w4_linear(x, W)
            x[1, 7], x[2, 150] = float("nan"), float("inf")
            y = w4_linear(x, W)
            assert not torch.isfinite(y[1:3]).any()
            keep = [i for i in range(M) if i not in (1, 2)]
            assert torch.equal(y[keep], clean[keep])


def test_another_stream_and_graph_replay():
    from atomic_gdn2.w4 import quantize_w4, w4_linear
    gen = torch.Generator(device="cuda").manual_seed(8)
    W = quantize_w4(torch.randn((512, 256), device="cuda", generator=gen), 64)
    x = torch.randn((4, 512), device="cuda", generator=gen)
    want = w4_linear(x, W)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = w4_linear(x, W)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    buf = x.clone()
    with torch.cuda.graph(graph):
        out = w4_linear(buf, W)
    for i in range(4):
        buf.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w4_linear(x * (i + 1), W))
