"""An SAE with 8-bit encoder weights, for activations held in 8 bits (saeflow_b200.store).

    pre = (x - b_dec) @ W_enc + b_enc = x @ W8 + (b_enc - b_dec @ W8)

x stays as the store holds it, so the b_dec shift moves into the bias, taken with the quantised
weights W8 (tiles of 128 x 128) that the product uses. Decoding is the 16 / 32-bit path unchanged.

A NaN pre-activation (a row that was stored with an infinity or NaN) is an inactive feature, as in SAE.encode and
encode_sparse: `pre > 0` is false. block_matmul's own "relu" keeps the NaN, so ReLU is its "jumprelu" with
thresholds of 0 here (4096 x 768 x 16384: bf16 68.7 against 69.7 us, fp32 81 against 89).
"""

from __future__ import annotations

import torch

from .kernels import dense_to_csr, sparse_decode
from .kernels.backward import matvec
from .kernels.blocks import BlockScaled, block_matmul, quantize


class QuantizedSAE:
    """The encode / encode_sparse / decode_sparse / forward of `sae` (ReLU or JumpReLU) on BlockScaled
    activations, for inference: nothing here has a gradient. The weights are laid out here, once; build it again after an update of `sae`."""

    def __init__(self, sae):
        if sae.activation not in ("relu", "jumprelu"):
            raise ValueError(f"QuantizedSAE supports relu and jumprelu, got {sae.activation!r}; read the rows back "
                             "for a top-k SAE")
        if sae.activation == "jumprelu" and sae.threshold is None:
            raise ValueError("jumprelu needs a threshold")
        self.activation = sae.activation
        self.w8 = quantize(sae.W_enc.detach(), tile=True, transpose=True)  # [d_sae, d_in]
        shift = matvec(self.w8.dequantize(torch.float32), sae.b_dec.detach().float())
        self.bias = sae.b_enc.detach().float() - shift
        self.threshold = (sae.threshold.detach().float() if sae.activation == "jumprelu"
                          else torch.zeros_like(self.bias))
        self.W_dec, self.b_dec = sae.W_dec.detach(), sae.b_dec.detach()

    def encode(self, x8, dtype=None):
        """Dense features [M, d_sae] of x8 (BlockScaled [M, d_in], row blocks), in `dtype` (default W_dec's)."""
        if not isinstance(x8, BlockScaled):
            raise ValueError("QuantizedSAE encodes BlockScaled activations (store.take, store.view, quantize)")
        return block_matmul(x8, self.w8, self.bias, "jumprelu", self.threshold,
                            out_dtype=dtype or self.W_dec.dtype)

    def encode_sparse(self, x8, dtype=None):
        """The same as CSR (indptr, indices, values)."""
        return dense_to_csr(self.encode(x8, dtype))

    def decode_sparse(self, csr):
        return sparse_decode(*csr, self.W_dec, self.b_dec)

    def forward(self, x8):
        """encode_sparse then decode_sparse: x_hat [M, d_in] in W_dec's dtype."""
        return self.decode_sparse(self.encode_sparse(x8))

    __call__ = forward
