"""8-bit products on the GPU over long sums, against the same sums in 64 bits.

Stored numbers are exact, so a product of two quantised matrices differs from its 64-bit value by its
additions and its last rounding alone. The tensor cores add 32 products at a time to an fp32 sum and round
toward zero: of operands of one sign, the i-th of n additions finds i/n of the total and loses half a unit in
its last place on average, (1/2) 2^-23 i/n of the total, n 2^-25 in all. Sums are kept over ranges of K of at
most 1024 (fp32 outputs) and 2560 (16-bit ones), n = 32 and 80, and the ranges added with rounding to
nearest, whose errors have no sign.
"""

import pytest
import torch

from saeflow_b200.kernels import BlockScaled, block_matmul, device_error, quantize

pytestmark = pytest.mark.gpu

SPACING = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # between neighbours, the least there is to a value


@pytest.fixture(autouse=True)
def _clean_device_errors():
    device_error()
    yield
    assert device_error() == 0, "a kernel reported a device-side error"


def one_sign(M, N, K):
    """Operands without a negative number, quantised, and their product in 64 bits (on the GPU)."""
    g = torch.Generator("cuda").manual_seed(M + N + K)
    a8 = quantize(torch.randn(M, K, device="cuda", generator=g).abs())
    b8 = quantize(torch.randn(N, K, device="cuda", generator=g).abs(), tile=True)
    return a8, b8, a8.dequantize().double() @ b8.dequantize().double().T


# more than 148 tiles of 128 x 128: whole sums, for a CTA pair; then a single CTA's tiles of 128, 64 and 32 rows
LONG = [(1000, 3000), (100, 20000), (40, 20000), (7, 20000)]


@pytest.mark.parametrize("M,N", LONG)
@pytest.mark.parametrize("K", [2304, 8192, 20001])
def test_long_fp32_sums_lose_no_more_than_their_ranges(M, N, K):
    a8, b8, want = one_sign(M, N, K)
    got = block_matmul(a8, b8, out_dtype=torch.float32)
    loss = ((want - got.double()) / want).mean().item()
    assert abs(loss) <= 32 * 2.0 ** -25 + 2.0 ** -24, f"sums are off by {loss:.3g} of their value on average"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N", LONG)
def test_long_16_bit_sums_round_as_the_exact_ones(M, N, dtype):
    """A sum that is off by a share e of itself crosses a rounding boundary with probability e / spacing."""
    a8, b8, want = one_sign(M, N, 16384)
    a8.scales.sub_(8)  # fp16's range
    want = (want * 2.0 ** -8).to(dtype)
    got = block_matmul(a8, b8, out_dtype=dtype)
    share = (got != want).double().mean().item()
    assert share <= 80 * 2.0 ** -25 / SPACING[dtype], f"{share:.3g} of the sums round to a neighbour"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1000, 3001, 640), (2500, 4101, 130), (1100, 2902, 2700), (40, 1003, 300)])
def test_nothing_beside_an_output_is_written(M, N, K, dtype):
    """Columns of wider memory whose rows start on 16-byte boundaries and end between them."""
    a8, b8, want = one_sign(M, N, K)
    wide = torch.full((M, 4400), 7.0, dtype=dtype, device="cuda")
    got = block_matmul(a8, b8, out=wide[:, 16:16 + N])
    assert (wide[:, :16] == 7).all() and (wide[:, 16 + N:] == 7).all()
    assert torch.allclose(got.double(), want, rtol=2 * SPACING.get(dtype, 2.0 ** -19))
    assert torch.equal(got, block_matmul(a8, b8, out_dtype=dtype))


@pytest.mark.parametrize("M,N,K", [(1000, 3000, 301), (100, 700, 130), (7, 300, 1)])
def test_nothing_beside_an_operand_is_read(M, N, K):
    """Operands that are columns of wider memory, NaN numbers and NaN scales on both sides of them."""
    a8, b8, want = one_sign(M, N, K)

    def wide(q):
        data = torch.full((q.shape[0] + 3, K + 150), 0x7F, dtype=torch.uint8, device="cuda")
        data = data[:, :(K + 150) // 16 * 16].contiguous()[:, 32:32 + K]
        data[:q.shape[0]] = q.data.view(torch.uint8)
        scales = torch.full((q.scales.shape[0] + 3, 16), 0xFF, dtype=torch.uint8, device="cuda")[:, 4:4 + q.scales.shape[1]]
        scales[:q.scales.shape[0]] = q.scales
        return BlockScaled(data[:q.shape[0]].view(torch.float8_e4m3fn), scales[:q.scales.shape[0]], q.tile)

    got = block_matmul(wide(a8), wide(b8), out_dtype=torch.float32)
    assert torch.equal(got, block_matmul(a8, b8, out_dtype=torch.float32)) and torch.isfinite(got).all()
    assert torch.allclose(got.double(), want, rtol=2.0 ** -18)
