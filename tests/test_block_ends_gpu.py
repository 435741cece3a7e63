"""8-bit matrices and operators on the GPU: how their parts are held, and calls at the ends of their range."""

import pytest
import torch
from torch.autograd import forward_ad

import saeflow_b200
from saeflow_b200.kernels import block_matmul, device_error, quantize, quantize_both
from saeflow_b200.store import ActivationStore
from saeflow_b200.training import linear8

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ["relu", "jumprelu"])
@pytest.mark.parametrize("rows", [7, 1000])
def test_rows_that_are_not_finite_have_no_features(rows, activation, dtype):
    """As in the 16 and 32-bit encoders: a NaN pre-activation is no feature, whatever the activation."""
    sae = saeflow_b200.SAE(200, 3000, activation, device="cuda", dtype=dtype)
    if activation == "jumprelu":
        sae.threshold.uniform_(0.1, 0.2)
    x = torch.randn(rows, 200, device="cuda", dtype=dtype)
    x[3, 17] = float("nan")
    x[5, 100] = float("inf")
    x8 = quantize(x)
    q = saeflow_b200.QuantizedSAE(sae)
    plain = x.clone()
    plain[5] = float("nan")  # as the row is held: at least one NaN
    assert (saeflow_b200.encode(sae, plain)[[3, 5]] == 0).all()  # the framework's rule
    f = q.encode(x8)
    assert (f[[3, 5]] == 0).all() and torch.isfinite(f).all() and (f != 0).any(1).sum() == rows - 2
    indptr, _, values = q.encode_sparse(x8)
    assert indptr[4] == indptr[3] and indptr[6] == indptr[5] and torch.isfinite(values).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 300])
def test_linear8_without_features(M, dtype):
    """N = 0: an empty output, a gradient of zeros for x, empty ones for W and b; for every set of wanted gradients."""
    for wanted in range(8):
        x, W, b = (torch.randn(*s, device="cuda", dtype=t).requires_grad_(bool(wanted >> i & 1))
                   for i, (s, t) in enumerate((((M, 100), dtype), ((100, 0), dtype), ((0,), torch.float32))))
        with torch.no_grad():
            assert linear8(x, W, b).shape == (M, 0)
        y = linear8(x, W, b)
        assert y.shape == (M, 0) and y.dtype == dtype and y.requires_grad == bool(wanted)
        if wanted:
            torch.full((1 << 20,), float("nan"), device="cuda")  # what freed memory may hold
            y.sum().backward()
        for i, (t, shape) in enumerate(((x, (M, 100)), (W, (100, 0)), (b, (0,)))):
            if wanted >> i & 1:
                assert t.grad.shape == shape and t.grad.dtype == t.dtype and (t.grad == 0).all()


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_linear8_refuses_forward_mode(which, grad):
    """Tangents stay on under no_grad: they are refused in both modes, not dropped."""
    args = [torch.randn(*s, device="cuda") for s in ((5, 64), (64, 32), (32,))]
    want = linear8(*args)
    with forward_ad.dual_level():
        dual = list(args)
        dual[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with torch.set_grad_enabled(grad):
            assert torch.equal(linear8(*args), want)
            with pytest.raises(NotImplementedError, match="forward.mode"):
                linear8(*dual)


def test_a_product_of_very_many_rows():
    """More than 2^22 tiles of rows, offsets past 32 bits in the operand and the output; small integers, exact."""
    M = 134217800
    a = torch.randint(-3, 4, (M, 4), device="cuda", dtype=torch.int8).bfloat16()
    b = torch.tensor([[1.0, -2.0, 3.0, 1.0]], device="cuda", dtype=torch.bfloat16)
    got = block_matmul(quantize(a), quantize(b))
    for i in range(0, M, 1 << 24):
        assert torch.equal(got[i:i + (1 << 24)], a[i:i + (1 << 24)] @ b.T)


def test_read_into_one_column_of_a_row_major_tensor():
    """A single column's own stride is never used."""
    store = ActivationStore(50, 1)
    x = torch.randn(50, 1, device="cuda")
    store.append(x)
    wide = torch.full((3, 50), 7.0, device="cuda")
    store.read(torch.arange(50, device="cuda"), out=wide.T[:, 1:2])
    assert torch.equal(wide[1:2].T, store.read(torch.arange(50, device="cuda"), torch.float32))
    assert (wide[[0, 2]] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantising_very_many_rows(dtype):
    """More row blocks than a grid's second extent (65535 x 128 rows): in tiles, transposed and with column sums."""
    R, C = 65535 * 128 + 300, 5
    x = torch.randint(-8, 9, (R, C), device="cuda", dtype=torch.int8).to(dtype)
    x[-200:] *= 64
    q, qt, sums = quantize_both(x, col_sums=True)
    rows = quantize(x)
    assert torch.equal(q.data.view(torch.uint8), rows.data.view(torch.uint8)) and torch.equal(q.scales, rows.scales)
    want = quantize(x.T.contiguous())
    assert torch.equal(qt.data.view(torch.uint8), want.data.view(torch.uint8)) and torch.equal(qt.scales, want.scales)
    assert torch.equal(sums.double(), x.double().sum(0))  # small integers: exact in any order
    t = quantize(x, tile=True)
    first = R // 128 * 128 - 128 * 5
    last = quantize(x[first:], tile=True)
    assert torch.equal(t.data[first:].view(torch.uint8), last.data.view(torch.uint8))
    assert torch.equal(t.scales[first // 128:], last.scales)
