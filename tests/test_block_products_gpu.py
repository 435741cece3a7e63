"""8-bit products on the GPU against the same sums in 64 bits: over long sums, on every tile shape and store of the
product kernel, with every activation. Each test states the plan (tile, splits of K) that it is there for.

Stored numbers are exact, so a product of two quantised matrices differs from its 64-bit value by its
additions and its last rounding alone. The tensor cores add 32 products at a time to an fp32 sum and round
toward zero: of operands of one sign, the i-th of n additions finds i/n of the total and loses half a unit in
its last place on average, (1/2) 2^-23 i/n of the total, n 2^-25 in all. Sums are kept over ranges of K of at
most 1024 (fp32 outputs) and 2560 (16-bit ones), n = 32 and 80, and the ranges added with rounding to
nearest, whose errors have no sign.
"""

import pytest
import torch

from oracle import blocks as ob
from saeflow_b200.kernels import BlockScaled, block_matmul, device_error, quantize
from saeflow_b200.kernels.blocks import product_plan
from saeflow_b200.training import linear8

pytestmark = pytest.mark.gpu

SPACING = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # between neighbours, the least there is to a value
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
PAIR = (256, 256)


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


TILES = {1000: PAIR, 100: (128, 128), 40: (64, 128), 7: (32, 128)}


@pytest.mark.parametrize("M,N", LONG)
@pytest.mark.parametrize("K", [2304, 8192, 20001])
def test_long_fp32_sums_lose_no_more_than_their_ranges(M, N, K):
    a8, b8, want = one_sign(M, N, K)
    assert product_plan(a8, b8, torch.float32) == (*TILES[M], -(-K // 8192), 1024)
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
    assert product_plan(a8, b8, dtype) == (*TILES[M], 1, 2560)
    got = block_matmul(a8, b8, out_dtype=dtype)
    share = (got != want).double().mean().item()
    assert share <= 80 * 2.0 ** -25 / SPACING[dtype], f"{share:.3g} of the sums round to a neighbour"


# ------------------------------------------------------------------------------- every tile and store

def operands(M, N, K, a_tile=False, b_tile=True):
    """Quantised operands whose scales vary along both axes, their 64-bit product and the sums of its products'
    magnitudes."""
    g = torch.Generator("cuda").manual_seed(M + N + K)
    a = torch.randn(M, K, device="cuda", generator=g) * torch.exp2(torch.randint(-4, 5, (M, 1), device="cuda", generator=g).float())
    b = torch.randn(N, K, device="cuda", generator=g) * 0.3
    b[:, :K // 2] *= 2.0 ** -7
    a8, b8 = quantize(a, tile=a_tile), quantize(b, tile=b_tile)
    ad, bd = a8.dequantize().double(), b8.dequantize().double()
    return a8, b8, ad @ bd.T, ad.abs() @ bd.abs().T


def sum_bound(K, magnitude):
    """Each addition of 32 products truncates at most two units in the last place of at most the magnitude: one
    aligning the products, one for the result; joining ranges and splits, and the bias, rounds less."""
    return (-(-K // 32) + 1) * 2.0 ** -22 * magnitude


def check_activated(got, pre, magnitude, K, activation, thr, dtype):
    """got against act(pre); features within the bound of a cut may fall on either side of it."""
    bound = sum_bound(K, magnitude)
    want, sure = pre, torch.ones_like(pre, dtype=torch.bool)
    if activation == "relu":
        want = pre.clamp(min=0)
    elif activation == "jumprelu":
        want = torch.where((pre > thr.double()) & (pre > 0), pre, torch.zeros_like(pre))
        sure = (pre - thr.double()).abs() > bound
        assert sure.double().mean() > 0.99
    bound = bound + HALF_ULP[dtype] * (want.abs() + bound) + TINY[dtype]
    off = (got.double() - want).abs() - bound
    assert got.dtype == dtype and got.shape == want.shape
    assert (off[sure] <= 0).all(), f"off by {off[sure].max():.3g} more than the bound"


def place(M, N, dtype, how):
    """(the tensor it lies in, out [M, N]): rows on 16-byte boundaries or between them."""
    pitch, lead = {"aligned": (-(-N // 8) * 8 + 16, 8), "odd pitch": (N // 2 * 2 + 9, 0), "odd lead": (-(-N // 8) * 8 + 16, 3)}[how]
    wide = torch.full((M, pitch), 7.0, dtype=dtype, device="cuda")
    return wide, lead, wide[:, lead:lead + N]


@pytest.mark.parametrize("how", ["aligned", "odd pitch", "odd lead"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", [None, "relu", "jumprelu"])
@pytest.mark.parametrize("M,N,K", [(900, 3000, 300), (1000, 3001, 640), (2500, 4104, 130), (1025, 3077, 2048)])
def test_pair_products(M, N, K, activation, dtype, how):
    """256 x 256 tiles, ragged in rows and columns, stored by TMA (rows of whole 16-byte units on 16-byte boundaries) or
    shifted to the output's boundaries; nothing beside the output is written."""
    a8, b8, want, mag = operands(M, N, K)
    assert product_plan(a8, b8, dtype)[:3] == (*PAIR, 1)
    bias, thr = torch.randn(N, device="cuda"), torch.rand(N, device="cuda")
    wide, lead, out = place(M, N, dtype, how)
    got = block_matmul(a8, b8, bias, activation, thr, out=out)
    check_activated(got, want + bias.double(), mag + bias.double().abs(), K, activation, thr, dtype)
    assert (wide[:, :lead] == 7).all() and (wide[:, lead + N:] == 7).all()


@pytest.mark.parametrize("a_tile,b_tile", [(False, True), (False, False), (True, True), (True, False)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pair_products_of_blocks_and_tiles(a_tile, b_tile, dtype):
    """Five tiles to a pair, so that both accumulators are used again while the other is read."""
    M, N, K = 4100, 5000, 1000
    a8, b8, want, mag = operands(M, N, K, a_tile, b_tile)
    assert product_plan(a8, b8, dtype)[:3] == (*PAIR, 1)
    check_activated(block_matmul(a8, b8, out_dtype=dtype), want, mag, K, None, None, dtype)


@pytest.mark.parametrize("how", ["aligned", "odd lead"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,splits32", [(1000, 3000, 8300, 2), (4100, 1200, 16384, 2), (1100, 2900, 2700, 1)])
def test_pair_products_over_long_sums(M, N, K, splits32, dtype, how):
    """Ranges of K added in registers; fp32 outputs past 8192 in splits; row tiles in groups of 32 MB, the last
    group short."""
    a8, b8, want, mag = operands(M, N, K)
    tile_rows, tile_cols, splits, most = product_plan(a8, b8, dtype)
    assert (tile_rows, tile_cols, splits) == (*PAIR, splits32 if dtype == torch.float32 else 1) and most < K / splits
    bias, thr = torch.randn(N, device="cuda"), torch.rand(N, device="cuda")
    for activation in (None, "relu", "jumprelu"):
        wide, lead, out = place(M, N, dtype, how)
        got = block_matmul(a8, b8, bias, activation, thr, out=out)
        check_activated(got, want + bias.double(), mag + bias.double().abs(), K, activation, thr, dtype)
        assert (wide[:, :lead] == 7).all() and (wide[:, lead + N:] == 7).all()
        again = block_matmul(a8, b8, bias, activation, thr, out_dtype=dtype)
        assert torch.equal(again, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", [None, "relu", "jumprelu"])
@pytest.mark.parametrize("M,N,K", [(640, 640, 8192), (300, 1001, 5000), (40, 1000, 20000), (5, 130, 4100)])
def test_split_sums(M, N, K, activation, dtype):
    """Few tiles and a long K: partial sums from a workspace, with bias and activation where they are joined."""
    a8, b8, want, mag = operands(M, N, K)
    assert product_plan(a8, b8, dtype)[2] > 1
    bias, thr = torch.randn(N, device="cuda"), torch.rand(N, device="cuda")
    got = block_matmul(a8, b8, bias, activation, thr, out_dtype=dtype)
    check_activated(got, want + bias.double(), mag + bias.double().abs(), K, activation, thr, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(100, 20000, 640), (40, 20000, 2700), (7, 1000, 500)])
def test_single_products_with_jumprelu(M, N, K, dtype):
    a8, b8, want, mag = operands(M, N, K)
    assert product_plan(a8, b8, dtype)[0] < 256
    bias, thr = torch.randn(N, device="cuda"), torch.rand(N, device="cuda")
    got = block_matmul(a8, b8, bias, "jumprelu", thr, out_dtype=dtype)
    check_activated(got, want + bias.double(), mag + bias.double().abs(), K, "jumprelu", thr, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [300, 2900])
def test_pair_products_non_finite(K, dtype):
    """A NaN of a row of either operand reaches that row or column and no other; ReLU keeps it."""
    M, N = 1000, 3001
    a, b = torch.randn(M, K), torch.randn(N, K)
    a[700, 7] = float("inf")
    b[2999, 3] = float("nan")
    a8, b8 = quantize(a.cuda()), quantize(b.cuda(), tile=True)
    assert product_plan(a8, b8, dtype)[:3] == (*PAIR, 1)
    want = torch.zeros(M, N, dtype=torch.bool)
    want[700], want[:, 2999] = True, True
    for act in (None, "relu"):
        assert torch.equal(torch.isnan(block_matmul(a8, b8, activation=act, out_dtype=dtype)).cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N,pairs", [(2000, 1500, 2600, True), (300, 200, 9001, False)])
def test_linear8_against_the_formulas_on_large_products(M, K, N, pairs, dtype):
    """Steps whose three products are all a pair's, and whose dx is in splits of a long sum."""
    x, W = torch.randn(M, K).to(dtype), (torch.randn(K, N) / K ** 0.5).to(dtype)
    b, dy = torch.randn(N), (torch.randn(M, N) * 0.1).to(dtype)
    for (r, c, k), name in zip(((M, N, K), (M, K, N), (K, N, M)), ("y", "dx", "dW")):
        e = [quantize(torch.zeros(n, k, device="cuda", dtype=dtype)) for n in (r, c)]
        plan = product_plan(*e, dtype)
        assert plan[:2] == PAIR if pairs else name != "dx" or plan[2] > 1, name
    g = [t.cuda().requires_grad_() for t in (x, W, b)]
    y = linear8(*g)
    got = (y.detach(), *torch.autograd.grad(y, g, dy.cuda()))
    want, mags = ob.linear(x, W, b, dy)
    for name, v, w, m, n, dt in zip(("y", "dx", "dW", "db"), got, want, mags, (K, N, M, 32 * M),
                                    (dtype, dtype, dtype, torch.float32)):
        check_activated(v.cpu(), w, m + (b.abs() if name == "y" else 0), n, None, None, dt)


@pytest.mark.parametrize("dtype", DTYPES)
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
