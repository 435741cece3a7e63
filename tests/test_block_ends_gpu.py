"""8-bit matrices and operators on the GPU: how their parts are held, and calls at the ends of their range."""

import pytest
import torch

from saeflow_b200.kernels import device_error, quantize
from saeflow_b200.store import ActivationStore

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_device_errors():
    device_error()
    yield
    assert device_error() == 0, "a kernel reported a device-side error"


def test_a_matrix_keeps_the_tensors_it_was_made_of():
    """The library is given the addresses of data and scales once; none of a matrix's parts is replaced after that."""
    store = ActivationStore(10, 64)
    other = quantize(torch.randn(10, 64, device="cuda"))
    for blocks in (store.blocks, other, store.view(2, 5)):
        for name in ("data", "scales", "tile", "shape", "device"):
            with pytest.raises(AttributeError):
                setattr(blocks, name, getattr(other, name))
        assert blocks._c.data == blocks.data.data_ptr() and blocks._c.scales == blocks.scales.data_ptr()
