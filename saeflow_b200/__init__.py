"""saeflow_b200: the saeflow SAE hot path (encode -> CSR -> decode) on B200 (sm_100a).

Drop-in for saeflow's `encode / encode_sparse / decode_sparse / forward` and
`saeflow.kernels`, backed by hand-written CUDA kernels in libsaeflow_b200.so.
"""

from .ops import HostForward, decode_sparse, encode, encode_sparse, forward, forward_host, forward_host_async
from .quantized import QuantizedSAE
from .sae import SAE
from .store import ActivationStore

__version__ = "0.1.0"
__all__ = ["SAE", "ActivationStore", "HostForward", "QuantizedSAE", "decode_sparse", "encode", "encode_sparse",
           "forward", "forward_host", "forward_host_async"]
