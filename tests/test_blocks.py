"""The 8-bit operators without a GPU: the oracle's rounding, the library's argument checks, refusals of CPU
tensors."""

import ctypes

import pytest
import torch

import saeflow_b200
from oracle import blocks as ob
from saeflow_b200 import _abi
from saeflow_b200.kernels import BlockScaled, block_matmul, quantize, quantize_both, write_rows
from saeflow_b200.training import linear8


def test_oracle_rounds_as_torch_does():
    """The oracle's search over the e4m3 grid against torch's conversion, every bf16 pattern up to 448."""
    t = torch.arange(0x10000, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    t = t[torch.isfinite(t) & (t.abs() <= 448)].double()
    assert torch.equal(ob.round_e4m3(t), t.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("tile", [False, True])
def test_oracle_scales_are_the_smallest_that_fit(tile):
    x = torch.randn(150, 300) * torch.exp2(torch.randint(-20, 20, (150, 1)).float())
    q, s = ob.quantize(x, tile)
    assert q.abs().max() <= 448
    per_block = ob._spread(s, x.shape, tile)
    halved = x.double().abs() / torch.exp2(per_block.double() - 128)
    for rows in ([slice(0, 128), slice(128, 150)] if tile else [slice(i, i + 1) for i in range(150)]):
        for c in (slice(0, 128), slice(128, 256), slice(256, 300)):
            assert halved[rows, c].max() > 448  # half the scale would not do
    # a number is off by at most half a step of its binade (2^-4 of it), or half the smallest subnormal
    off = (ob.dequantize(q, s, tile) - x.double()).abs()
    assert (off <= torch.maximum(x.double().abs() / 16, torch.exp2(per_block.double() - 127 - 10))).all()


def fake(rows, cols, tile=0, data=256, scales=256, pitch=None, scale_pitch=None):
    """A structure with placeholder addresses, never read."""
    nb = -(-cols // 128)
    return _abi.SfBlocks(data, scales, rows, cols, -(-cols // 16) * 16 if pitch is None else pitch,
                         -(-nb // 4) * 4 if scale_pitch is None else scale_pitch, tile, 0)


def test_library_checks_block_arguments():
    lib = _abi.load()
    x = _abi.SfMatrix(256, 0, 0, 4, 64, 64, 1)
    r = ctypes.byref

    def refused(status, words):
        assert status == _abi.SF_ERR_INVALID
        assert words in lib.sf_last_error().decode()

    refused(lib.sf_blocks_write(r(x), None, None, None), "NULL")
    refused(lib.sf_blocks_write(r(x), None, r(fake(4, 65)), None), "columns")
    refused(lib.sf_blocks_write(r(x), None, r(fake(3, 64)), None), "more rows")
    refused(lib.sf_blocks_write(r(x), None, r(fake(4, 64, tile=1)), None), "row blocks")
    refused(lib.sf_blocks_write(r(x), None, r(fake(4, 64, data=8)), None), "16-byte")
    refused(lib.sf_blocks_write(r(x), None, r(fake(4, 64, pitch=72)), None), "16-byte")
    refused(lib.sf_blocks_write(r(x), None, r(fake(4, 64, pitch=48)), None), "16-byte")
    refused(lib.sf_blocks_write(r(x), None, r(fake(4, 64, scales=258)), None), "4-byte")
    refused(lib.sf_blocks_write(r(x), None, r(fake(4, 1000, scale_pitch=4)), None), "4-byte")
    refused(lib.sf_blocks_write(r(x), None, r(fake(4, 64, data=None)), None), "NULL")
    bad = _abi.SfMatrix(256, 9, 0, 4, 64, 64, 1)
    refused(lib.sf_blocks_write(r(bad), None, r(fake(4, 64)), None), "dtype")
    refused(lib.sf_blocks_read(r(fake(3, 64)), None, r(x), None), "more rows")
    refused(lib.sf_blocks_take(r(fake(3, 64)), None, r(fake(4, 64)), None), "more rows")
    refused(lib.sf_blocks_quantize(r(x), None, None, None, None, 0, None), "both NULL")
    refused(lib.sf_blocks_quantize(r(x), r(fake(4, 64)), r(fake(64, 4, tile=1)), None, None, 0, None), "both")
    refused(lib.sf_blocks_quantize(r(x), None, r(fake(4, 64)), None, None, 0, None), "transpose")
    assert lib.sf_blocks_quantize(r(x), r(fake(4, 64)), None, 256, None, 0, None) == _abi.SF_ERR_WORKSPACE
    need = ctypes.c_size_t(0)
    out = _abi.SfMatrix(256, 0, 0, 4, 5, 5, 1)
    refused(lib.sf_block_matmul_workspace(r(fake(4, 64)), r(fake(5, 65)), r(out), r(need)), "columns")
    refused(lib.sf_block_matmul_workspace(r(fake(4, 64)), r(fake(6, 64)), r(out), r(need)), "out must be")
    refused(lib.sf_block_matmul_workspace(r(fake(4, 0)), r(fake(5, 0)), r(out), r(need)), "no columns")
    refused(lib.sf_block_matmul(r(fake(4, 64)), r(fake(5, 64)), None, None, 7, r(out), None, 0, None), "activation")
    refused(lib.sf_block_matmul(r(fake(4, 64)), r(fake(5, 64)), None, None, 1, r(out), None, 0, None), "threshold")
    dy = _abi.SfMatrix(256, 0, 0, 0, 5, 5, 1)
    refused(lib.sf_linear8_backward(r(dy), 256, 64, 7, None, None, None, 256, 0, None), "no rows")


def test_long_products_ask_for_partial_sums():
    """fp32 outputs sum at most 8192 of K at a time; 16-bit outputs of many tiles do not split."""
    lib = _abi.load()
    need = ctypes.c_size_t(0)
    a, b = fake(4096, 16384), fake(4096, 16384, tile=1)
    out = _abi.SfMatrix(256, 0, 0, 4096, 4096, 4096, 1)
    assert lib.sf_block_matmul_workspace(ctypes.byref(a), ctypes.byref(b), ctypes.byref(out), ctypes.byref(need)) == 0
    assert need.value == 2 * 4096 * 4096 * 4
    out = _abi.SfMatrix(256, 1, 0, 4096, 4096, 4096, 1)
    assert lib.sf_block_matmul_workspace(ctypes.byref(a), ctypes.byref(b), ctypes.byref(out), ctypes.byref(need)) == 0
    assert need.value == 0
    assert lib.sf_block_matmul(ctypes.byref(fake(64, 16384)), ctypes.byref(fake(64, 16384)), None, None, -1,
                               ctypes.byref(_abi.SfMatrix(256, 1, 0, 64, 64, 64, 1)), None, 0, None) == \
        _abi.SF_ERR_WORKSPACE


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    data, scales = torch.zeros(4, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8)
    for call in (lambda: quantize(x), lambda: quantize_both(x), lambda: BlockScaled(data, scales),
                 lambda: BlockScaled.empty(4, 64, device="cpu"), lambda: saeflow_b200.ActivationStore(4, 64, "cpu"),
                 lambda: linear8(x, x.T), lambda: saeflow_b200.QuantizedSAE(saeflow_b200.SAE(64, 128)),
                 lambda: write_rows(x, None)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_argument_errors_precede_device_checks():
    with pytest.raises(ValueError, match="linear8 takes"):
        linear8(torch.zeros(4, 5), torch.zeros(4, 5))
    with pytest.raises(ValueError, match="b must be"):
        linear8(torch.zeros(4, 5), torch.zeros(5, 3), torch.zeros(4))
    with pytest.raises(ValueError, match="at least one row"):
        saeflow_b200.ActivationStore(0, 5)
    with pytest.raises(ValueError, match="top-k"):
        saeflow_b200.QuantizedSAE(saeflow_b200.SAE(8, 16, "topk", k=2))
    assert saeflow_b200.ActivationStore.bytes_per_row(2304) == 2304 + 20
    assert callable(block_matmul)
