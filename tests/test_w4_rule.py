"""Which kernel a 4-bit product runs: few rows of a wide matrix take the tiles of 32 rows, not the many-row kernel's
of 128 (float32: 64), which would multiply rows that are not there."""
import ctypes

import pytest


def _workspace(M, K, N, group, dtype):
    from atomic_gdn2 import _lib
    a = _lib.Gdn2W4(M, K, N, group, dtype, K, 0, *([1 << 20] * 3), None, None, 1 << 20)
    return _lib.lib().gdn2_w4_workspace_bytes(ctypes.byref(a))


def _sums(M, K, group):
    """The many-row kernel's workspace for rows that it reads in place."""
    groups = -(-K // 128) * (128 // group)
    return 3 * -(-M // 16) * -(-groups // 32) * 1024


@pytest.mark.parametrize("N", [49152, 131072])
def test_few_rows_of_a_wide_matrix(N):
    for M in (9, 16, 33, 64):
        assert _workspace(M, 4096, N, 128, 1) == 0, M               # (one part, rows read in place)
    for M in (65, 96, 128, 300):
        assert _workspace(M, 4096, N, 128, 1) == _sums(M, 4096, 128), M
    assert _workspace(32, 4096, N, 128, 0) == 0
    assert _workspace(33, 4096, N, 128, 0) == _sums(33, 4096, 128) + 3 * 33 * 4096 * 2
    assert _workspace(2048, 4096, 4096, 128, 1) == _sums(2048, 4096, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N,group", [(16, 2056, 49300, 64), (33, 1288, 50000, 128), (64, 1032, 65544, 32), (65, 1032, 65541, 32)])
def test_products_on_both_sides_of_the_rule(M, K, N, group, dtype):
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    from test_gpu_w4 import test_product_matches_the_definition
    test_product_matches_the_definition(M, K, N, group, dtype)
