"""Kernel-level API, a drop-in for saeflow.kernels (saeflow/kernels/__init__.py:1-9).

There is no interpreter mode: every op runs a CUDA kernel of libsaeflow_b200.so on
sm_100a, so INTERPRET is always False.
"""

from .._abi import device_error
from .blocks import BlockScaled, block_matmul, quantize, quantize_both, read_rows, take_rows, write_rows
from .decode import csr_to_dense, dense_to_csr, sparse_decode, topk_encode
from .encode import best_config, encode_csr, fused_encode

INTERPRET = False

__all__ = ["INTERPRET", "BlockScaled", "best_config", "block_matmul", "csr_to_dense", "dense_to_csr", "device_error",
           "encode_csr", "fused_encode", "quantize", "quantize_both", "read_rows", "sparse_decode", "take_rows",
           "topk_encode", "write_rows"]
