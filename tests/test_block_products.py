"""The plan of 8-bit products without a GPU (148 SMs): which tile, how many splits of K, how long a sum."""

import ctypes

import pytest

from saeflow_b200 import _abi


def plan(M, N, K, dtype):
    a, b = (_abi.SfBlocks(256, 256, n, K, -(-K // 16) * 16, -(-K // 512) * 4, 0, 0) for n in (M, N))
    out, p = _abi.SfMatrix(256, dtype, 0, M, N, N, 1), _abi.SfBlockPlan()
    _abi.check(_abi.load().sf_block_matmul_plan(ctypes.byref(a), ctypes.byref(b), ctypes.byref(out), ctypes.byref(p)))
    return p.tile_rows, p.tile_cols, p.splits, p.range


@pytest.mark.parametrize("M,N,K,dtype,want", [
    (16384, 65536, 2304, _abi.SF_BF16, (256, 256, 1, 2304)),   # a batch: one sum
    (16384, 2304, 65536, _abi.SF_BF16, (256, 256, 1, 2560)),   # its input gradient: ranges in registers
    (16384, 65536, 2304, _abi.SF_F32, (256, 256, 1, 1024)),
    (16384, 2304, 65536, _abi.SF_F32, (256, 256, 8, 1024)),    # splits of 8192 in a workspace, in ranges
    (1, 65536, 2304, _abi.SF_BF16, (32, 128, 1, 2304)),        # one token
    (64, 65536, 2304, _abi.SF_BF16, (64, 128, 1, 2304)),
    (100, 16384, 768, _abi.SF_BF16, (128, 128, 1, 768)),
    (64, 64, 16384, _abi.SF_BF16, (64, 128, 8, 2048)),         # idle SMs take splits of 2048
    (0, 64, 768, _abi.SF_BF16, (0, 0, 0, 0)),
])
def test_plan(M, N, K, dtype, want):
    assert plan(M, N, K, dtype) == want


@pytest.mark.parametrize("K", [1, 512, 513, 1024, 1025, 2560, 2561, 8192, 8193, 65537])
def test_sums_are_never_longer_than_their_type_allows(K):
    for M, N in ((4096, 4096), (1, 64), (640, 640)):
        for dtype, most in ((_abi.SF_F32, 1024), (_abi.SF_BF16, 2560), (_abi.SF_F16, 2560)):
            assert plan(M, N, K, dtype)[3] <= min(most, K)


@pytest.mark.parametrize("M,N,K,dtype", [(262144, 65536, 2304, _abi.SF_BF16), (1 << 20, 16384, 768, _abi.SF_BF16),
                                         (65536, 1 << 20, 16384, _abi.SF_F32), (134217800, 1, 16, _abi.SF_BF16)])
def test_large_outputs_are_planned(M, N, K, dtype):
    """Tens of GB of output: tiles are counted as they are cut, up to what 32 bits number."""
    assert plan(M, N, K, dtype)[0] in (128, 256)


@pytest.mark.parametrize("M,N", [(1 << 30, 1 << 30), ((1 << 31) - 5000, (1 << 31) - 5000), (1 << 25, 1 << 24)])
def test_too_many_tiles_are_refused(M, N):
    with pytest.raises(RuntimeError, match="too many output tiles"):
        plan(M, N, 128, _abi.SF_BF16)
