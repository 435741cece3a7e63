"""Block-scaled 8-bit operators on the GPU against their plain 64-bit forms (oracle/blocks.py).

Quantising and dequantising are exact definitions, so they are compared for equality. Products: the
tensor cores add 32 products at a time to an fp32 sum, rounding toward zero, so after n = ceil(K / 32)
additions the sum is within (n + 1) 2^-22 of sum_k |a||b| (two units in the last place of at most that
sum per addition: one for the alignment inside it, one for its result); then one rounding to the
output's type.
"""

import pytest
import torch

import saeflow_b200
from oracle import blocks as ob
from saeflow_b200.kernels import (BlockScaled, block_matmul, device_error, quantize, quantize_both, read_rows,
                                  take_rows, write_rows)
from saeflow_b200.store import ActivationStore
from saeflow_b200.training import linear8

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
SHAPES = [(1, 1), (1, 128), (3, 127), (5, 129), (130, 300), (33, 1001), (257, 256)]


@pytest.fixture(autouse=True)
def _clean_device_errors():
    device_error()
    yield
    assert device_error() == 0, "a kernel reported a device-side error"


def activations(rows, d, dtype):
    """Token norms over several powers of two, one loud channel, a row of zeros."""
    x = torch.randn(rows, d) * torch.exp2(torch.randint(-6, 7, (rows, 1)).float())
    x[:, d // 2] *= 50
    if rows > 2:
        x[rows // 2] = 0
    return x.to(dtype)


def layout(x, how):
    """x's values on the GPU in another memory layout."""
    g = x.cuda()
    if how == "rows":
        return g
    if how == "columns":
        return g.T.contiguous().T
    wide = torch.zeros(x.shape[0], x.shape[1] + 24, dtype=x.dtype, device="cuda")
    lead = {"aligned slice": 8, "odd slice": 3}[how]
    wide[:, lead:lead + x.shape[1]] = g
    return wide[:, lead:lead + x.shape[1]]


def same(got, q, s):
    """The stored numbers and bytes equal the oracle's."""
    data = got.data.cpu().double()
    assert torch.equal(torch.isnan(data), torch.isnan(q))
    assert torch.equal(torch.nan_to_num(data), torch.nan_to_num(q))
    assert torch.equal(got.scales.cpu().long(), s)


def close(got, want, magnitude, K, dtype):
    got, want = got.cpu().double(), want.cpu()
    bound = (-(-K // 32) + 1) * 2.0 ** -22 * magnitude.cpu()
    bound = bound + HALF_ULP[dtype] * (want.abs() + bound) + TINY[dtype]
    worst = ((got - want).abs() - bound).max()
    assert got.shape == want.shape and worst <= 0, f"off by {worst:.3g} more than the bound"


# ------------------------------------------------------------------------------- quantising

@pytest.mark.parametrize("how", ["rows", "columns", "aligned slice", "odd slice"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_all_forms(shape, dtype, how):
    x = activations(*shape, dtype)
    g = layout(x, how)
    for tile in (False, True):
        want, want_t = ob.quantize(x, tile), ob.quantize(x.T, tile)
        same(quantize(g, tile=tile), *want)
        same(quantize(g, tile=tile, transpose=True), *want_t)
        q, qt, sums = quantize_both(g, tile=tile, col_sums=True)
        same(q, *want)
        same(qt, *want_t)
        # fp32 sums of n addends, each addition rounding a partial sum of at most sum |x|
        bound = shape[0] * 2.0 ** -24 * x.double().abs().sum(0)
        assert ((sums.cpu().double() - x.double().sum(0)).abs() <= bound).all()
        if tile:
            assert torch.equal(q.scales, qt.scales.T)


@pytest.mark.parametrize("tile", [False, True])
def test_quantize_scale_edges(tile):
    """One block each: amax at, just above and just below 448 2^k, subnormal, the largest float, zero,
    non-finite entries beside finite ones and alone, and ties of the e4m3 grid."""
    inf, nan = float("inf"), float("nan")
    up = torch.nextafter(torch.tensor(448.0), torch.tensor(500.0)).item()
    down = torch.nextafter(torch.tensor(448.0), torch.tensor(0.0)).item()
    rows = [[448.0], [up], [down], [448.0 * 2 ** -100], [up * 2.0 ** 100], [3.4028234663852886e38], [1e-45], [2e-39],
            [0.0], [-0.0], [inf, 1.0, -2.0], [nan, 1e-30], [inf, -inf, nan], [1.0, 2.0 ** -17, 3 * 2.0 ** -19],
            [448.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, 17.0, 19.0, 21.0, -17.0, 2.0 ** -9 * 1.5]]
    for values in rows:
        x = torch.zeros(2, 130)
        x[1, :len(values)] = torch.tensor(values)
        same(quantize(x.cuda(), tile=tile), *ob.quantize(x, tile))
        same(quantize(x.cuda(), tile=tile, transpose=True), *ob.quantize(x.T, tile))


# ------------------------------------------------------------------------------- the store

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 16, 100, 128, 777, 2304])
def test_store_write_and_read(d, dtype):
    cap, T = 400, 150
    store = ActivationStore(cap, d)
    x = activations(T, d, dtype)
    slots = torch.randperm(cap)[:T]
    slots[::7] = -1
    store.write(x.cuda(), slots.cuda())
    q, s = torch.zeros(cap, d, dtype=torch.float64), torch.zeros(cap, -(-d // 128), dtype=torch.int64)
    wq, ws = ob.quantize(x)
    kept = slots >= 0
    q[slots[kept]], s[slots[kept]] = wq[kept], ws[kept]
    same(store.blocks, q, s)  # dropped rows wrote nothing
    rows = torch.cat([torch.randint(0, cap, (200,)), torch.tensor([-1, 0, cap - 1, -5])])
    want = ob.dequantize(q, s)[rows.clamp(min=0)]
    want[rows < 0] = 0
    for out_dtype in DTYPES:
        got = store.read(rows.cuda(), out_dtype)
        assert got.dtype == out_dtype and torch.equal(got.cpu(), want.float().to(out_dtype))
    assert torch.equal(store.read(rows.int().cuda(), torch.float32).cpu(), want.float())  # int32 rows
    wide = torch.full((len(rows), d + 5), 7.0, device="cuda")
    store.read(rows.cuda(), out=wide[:, 2:2 + d])  # a slice of a wider tensor, nothing beside it touched
    assert torch.equal(wide[:, 2:2 + d].cpu(), want.float())
    assert (wide[:, :2] == 7).all() and (wide[:, 2 + d:] == 7).all()
    taken = store.take(rows.cuda())
    same(taken, torch.where((rows < 0)[:, None], 0.0, q[rows.clamp(min=0)]),
         torch.where((rows < 0)[:, None], 0, s[rows.clamp(min=0)]))


def test_store_slice_of_wider_memory_is_left_alone():
    """A store over columns of a wider buffer: writes stay inside its columns, tails included."""
    data = torch.full((8, 64), 5, dtype=torch.uint8, device="cuda")
    scales = torch.full((8, 8), 9, dtype=torch.uint8, device="cuda")
    store = ActivationStore.wrap(data.view(torch.float8_e4m3fn)[:, 16:16 + 13], scales[:, :1])
    x = torch.randn(8, 13)
    store.write(x.cuda(), torch.arange(8).cuda())
    same(store.blocks, *ob.quantize(x))
    assert (data[:, :16] == 5).all() and (data[:, 29:] == 5).all() and (scales[:, 1:] == 9).all()


def test_store_append_wraps_and_keeps_the_newest():
    store = ActivationStore(100, 40)
    x = activations(370, 40, torch.float32)
    for a, b in [(0, 0), (0, 60), (60, 130), (130, 131), (131, 370)]:  # the last overwrites the store twice
        store.append(x[a:b].cuda())
        assert len(store) == min(b, 100) and store.written == b
    order = torch.arange(270, 370)
    want = ob.round_trip(x[order])
    assert torch.equal(store.read((order % 100).cuda(), torch.float32).cpu(), want.float())
    same(store.view(10, 20), *ob.quantize(x[310:320]))


def test_store_empty_calls():
    store = ActivationStore(10, 64)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    store.write(torch.zeros(0, 64, device="cuda"), none)
    assert store.read(none).shape == (0, 64) and store.take(none).shape == (0, 64)
    assert quantize(torch.zeros(0, 64, device="cuda")).shape == (0, 64)
    assert quantize(torch.zeros(0, 64, device="cuda"), transpose=True).shape == (64, 0)


def test_store_indices_past_the_end_are_reported():
    store = ActivationStore(10, 64)
    x = activations(3, 64, torch.float32)
    store.write(x.cuda(), torch.tensor([10, 4, 1 << 40], device="cuda"))
    assert device_error() == 2
    want = torch.zeros(10, 64)
    want[4] = ob.round_trip(x)[1].float()
    assert torch.equal(store.blocks.dequantize().cpu(), want)
    got = store.read(torch.tensor([4, 10, 1 << 40], device="cuda"), torch.float32)
    assert device_error() == 2
    assert torch.equal(got.cpu(), torch.stack([want[4], want[0], want[0]]))
    taken = store.take(torch.tensor([10, 4], device="cuda"))
    assert device_error() == 2
    assert torch.equal(taken.dequantize().cpu(), want[[0, 4]])


def test_store_offsets_past_32_bits():
    cap, d = 2_000_000, 2304  # 4.6 GB of numbers
    store = ActivationStore(cap, d)
    x = activations(300, d, torch.bfloat16)
    slots = torch.cat([torch.arange(cap - 200, cap), torch.arange(100)])
    store.write(x.cuda(), slots.cuda())
    want = ob.round_trip(x)
    assert torch.equal(store.read(slots.cuda(), torch.float32).cpu(), want.float())
    assert torch.equal(store.take(slots.cuda()).dequantize().cpu(), want.float())
    W = torch.randn(64, d)
    got = block_matmul(store.view(cap - 200, cap), quantize(W.cuda(), tile=True), out_dtype=torch.float32)
    y, mag = ob.matmul(want[:200], ob.round_trip(W, True))
    close(got, y, mag, d, torch.float32)


# ------------------------------------------------------------------------------- the product

def operands(M, N, K, a_tile=False, b_tile=True):
    a, b = activations(M, K, torch.float32), torch.randn(N, K) * 0.3
    b[:, :K // 2] *= 2.0 ** -7  # scales that differ along K
    return a, b, quantize(a.cuda(), tile=a_tile), quantize(b.cuda(), tile=b_tile)


@pytest.mark.parametrize("a_tile,b_tile", [(False, True), (False, False), (True, True), (True, False)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 513, 129), (5, 128, 128), (33, 300, 31), (64, 640, 512),
                                   (100, 70, 513), (129, 257, 1000), (300, 1030, 640), (520, 1100, 2304)])
def test_block_matmul(M, N, K, a_tile, b_tile):
    a, b, a8, b8 = operands(M, N, K, a_tile, b_tile)
    want, mag = ob.matmul(ob.round_trip(a, a_tile), ob.round_trip(b, b_tile))
    for dtype in DTYPES:
        got = block_matmul(a8, b8, out_dtype=dtype)
        assert got.dtype == dtype
        close(got, want, mag, K, dtype)


@pytest.mark.parametrize("M", [1, 2, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("N", [1, 127, 128, 129, 255, 257, 511])
def test_block_matmul_ragged_tiles(M, N):
    K = 384
    a, b, a8, b8 = operands(M, N, K)
    bias = torch.randn(N)
    want, mag = ob.matmul(ob.round_trip(a), ob.round_trip(b, True), bias, "relu")
    got = block_matmul(a8, b8, bias.cuda(), "relu", out_dtype=torch.float32)
    close(got, want, mag + bias.abs(), K, torch.float32)


@pytest.mark.parametrize("M,N", [(1, 1000), (40, 1000), (300, 1000), (1000, 40)])
@pytest.mark.parametrize("K", [4000, 20000])
def test_block_matmul_long_sums(M, N, K):
    """Few tiles and a long K: the work is split along K and joined, the same bits each time."""
    a, b, a8, b8 = operands(M, N, K, False, False)
    bias = torch.randn(N)
    want, mag = ob.matmul(ob.round_trip(a), ob.round_trip(b), bias)
    got = block_matmul(a8, b8, bias.cuda(), out_dtype=torch.float32)
    close(got, want, mag + bias.abs(), K, torch.float32)
    for _ in range(3):
        assert torch.equal(got, block_matmul(a8, b8, bias.cuda(), out_dtype=torch.float32))


@pytest.mark.parametrize("M", [3, 200, 700])
def test_block_matmul_jumprelu(M):
    """Features whose sum lies within the bound of the cut may fall on either side of it."""
    N, K = 1000, 500
    a, b, a8, b8 = operands(M, N, K)
    bias, thr = torch.randn(N), torch.rand(N)
    pre, mag = ob.matmul(ob.round_trip(a), ob.round_trip(b, True), bias)
    want = torch.where((pre > thr.double()) & (pre > 0), pre, torch.zeros_like(pre))
    got = block_matmul(a8, b8, bias.cuda(), "jumprelu", thr.cuda(), out_dtype=torch.float32).cpu()
    bound = (-(-K // 32) + 1) * 2.0 ** -22 * (mag + bias.abs())
    sure = (pre - thr.double()).abs() > bound
    assert sure.double().mean() > 0.99
    assert ((got.double() - want).abs() <= 2 * bound)[sure].all()


@pytest.mark.parametrize("M,N,K", [(2, 300, 300), (300, 300, 300)])
def test_block_matmul_non_finite(M, N, K):
    """A NaN of a row of `a` reaches that row of the product and no other; ReLU keeps it."""
    a, b = torch.randn(M, K), torch.randn(N, K)
    a[1, 7] = float("inf")
    b[299, 3] = float("nan")
    a8, b8 = quantize(a.cuda()), quantize(b.cuda(), tile=True)
    for act in (None, "relu"):
        got = torch.isnan(block_matmul(a8, b8, activation=act).float()).cpu()
        want = torch.zeros(M, N, dtype=torch.bool)
        want[1], want[:, 299] = True, True
        assert torch.equal(got, want)


@pytest.mark.parametrize("M", [2, 200])
@pytest.mark.parametrize("scale", [2.0 ** -120, 2.0 ** -60, 2.0 ** 60, 2.0 ** 118])
def test_block_matmul_extreme_scales(M, scale):
    """Scale bytes at both ends of their range: the operands' scales multiply before the sum."""
    a, b = torch.randn(M, 200).clamp(-4, 4) * scale, torch.randn(300, 200).clamp(-4, 4) / scale
    want, mag = ob.matmul(ob.round_trip(a), ob.round_trip(b, True))
    got = block_matmul(quantize(a.cuda()), quantize(b.cuda(), tile=True), out_dtype=torch.float32)
    close(got, want, mag, 200, torch.float32)


@pytest.mark.parametrize("M", [7, 300])
def test_block_matmul_strided_out_and_views(M):
    """Rows and outputs that are parts of larger tensors; nothing beside them is touched."""
    N, K = 333, 260
    a, b, a8, b8 = operands(M + 9, N, K)
    want, mag = ob.matmul(ob.round_trip(a), ob.round_trip(b, True))
    for lead in (0, 3):
        wide = torch.full((M, N + 8), 7.0, device="cuda", dtype=torch.bfloat16)
        out = block_matmul(a8.rows(9, 9 + M), b8, out=wide[:, lead:lead + N])
        close(out, want[9:], mag[9:], K, torch.bfloat16)
        assert (wide[:, :lead] == 7).all() and (wide[:, lead + N:] == 7).all()


def test_block_matmul_empty():
    a, b = quantize(torch.zeros(0, 64, device="cuda")), quantize(torch.randn(5, 64, device="cuda"))
    assert block_matmul(a, b).shape == (0, 5) and block_matmul(b, a).shape == (5, 0)


def test_another_stream():
    """Every operator runs on the current stream: work queued behind a slow kernel of that stream
    sees its results."""
    side = torch.cuda.Stream()
    x, W = activations(300, 500, torch.float32), torch.randn(200, 500)
    gx, gW = x.cuda(), W.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        store = ActivationStore(300, 500)
        store.write(gx * 2, torch.arange(300, device="cuda"))
        y = block_matmul(store.view(0, 300), quantize(gW, tile=True), out_dtype=torch.float32)
        back = store.read(torch.arange(300, device="cuda"), torch.float32)
    side.synchronize()
    want = ob.round_trip(2 * x)
    assert torch.equal(back.cpu(), want.float())
    close(y, *ob.matmul(want, ob.round_trip(W, True)), 500, torch.float32)


# ------------------------------------------------------------------------------- training

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 16, 32), (37, 50, 129), (200, 130, 300), (513, 256, 640), (1500, 100, 70)])
def test_linear8_against_the_formulas(M, K, N, dtype):
    x, W = activations(M, K, dtype), (torch.randn(K, N) / K ** 0.5).to(dtype)
    b, dy = torch.randn(N), (torch.randn(M, N) * 0.1).to(dtype)
    g = [t.cuda().requires_grad_() for t in (x, W, b)]
    y = linear8(*g)
    got = (y.detach(), *torch.autograd.grad(y, g, dy.cuda()))
    want, mags = ob.linear(x, W, b, dy)
    for name, v, w, m, n, dt in zip(("y", "dx", "dW", "db"), got, want, mags, (K, N, M, 32 * M),
                                    (dtype, dtype, dtype, torch.float32)):
        assert v.dtype == dt, name
        close(v, w, m + (b.abs() if name == "y" else 0), n, dt)


def test_linear8_against_differences():
    """Small integers are exact in e4m3 under any scale they meet here, and so are their sums in fp32:
    the loss is linear in each entry, and a difference over a unit step is its gradient exactly."""
    M, K, N = 140, 20, 30
    x, W = torch.randint(-3, 4, (M, K)).float(), torch.randint(-3, 4, (K, N)).float()
    b, c = torch.randint(-3, 4, (N,)).float(), torch.randint(-3, 4, (M, N)).float()
    g = [t.cuda().requires_grad_() for t in (x, W, b)]
    loss = (linear8(*g) * c.cuda()).sum()
    grads = [t.cpu() for t in torch.autograd.grad(loss, g)]

    def value(x, W, b):
        return (linear8(x.cuda(), W.cuda(), b.cuda()).double() * c.cuda().double()).sum().item()

    base = value(x, W, b)
    assert base == loss.item()
    for which, t in enumerate((x, W, b)):
        for _ in range(10):
            at = tuple(torch.randint(0, n, ()).item() for n in t.shape)
            args = [x, W, b]
            args[which] = t.clone()
            args[which][at] += 1
            assert value(*args) - base == grads[which][at].item()


def test_linear8_needs_only_what_is_asked():
    x, W, b = torch.randn(40, 64), torch.randn(64, 96), torch.randn(96)
    dy = torch.randn(40, 96).cuda()
    full = [t.cuda().requires_grad_() for t in (x, W, b)]
    want = torch.autograd.grad(linear8(*full), full, dy)
    for which in range(3):
        g = [t.cuda().requires_grad_(i == which) for i, t in enumerate((x, W, b))]
        got, = torch.autograd.grad(linear8(*g), g[which], dy)
        assert torch.equal(got, want[which])
    g = [t.cuda().requires_grad_() for t in (x, W)]
    y = linear8(*g)  # no bias; a gradient that is one number broadcast
    y.sum().backward()
    dx, dW = g[0].grad, g[1].grad
    want, mags = ob.linear(x, W, torch.zeros(96), torch.ones(40, 96))
    close(dx, want[1], mags[1], 96, torch.float32)
    close(dW, want[2], mags[2], 40, torch.float32)


def test_linear8_without_gradients_and_twice():
    x, W, b = (torch.randn(*s, device="cuda").requires_grad_() for s in ((30, 64), (64, 40), (40,)))
    y = linear8(x, W, b)
    with torch.no_grad():
        assert torch.equal(linear8(x, W, b), y) and not linear8(x, W, b).requires_grad
    dx, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_linear8_on_another_stream():
    """Forward and backward on a side stream, behind a slow kernel there."""
    x, W, b, dy = torch.randn(200, 96), torch.randn(96, 150), torch.randn(150), torch.randn(200, 150)
    g = [t.cuda().requires_grad_() for t in (x, W, b)]
    gdy = dy.cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = torch.autograd.grad(linear8(*g), g, gdy)
    side.synchronize()
    want = torch.autograd.grad(linear8(*g), g, gdy)
    for a, w in zip(got, want):
        assert torch.equal(a, w)


def test_operators_in_a_graph():
    """Captured once, replayed on new values in the same memory."""
    x, W = torch.randn(300, 200, device="cuda"), torch.randn(500, 200, device="cuda")
    store = ActivationStore(400, 200)
    slots = torch.arange(300, device="cuda")
    w8 = quantize(W, tile=True)

    def step():
        store.write(x, slots)
        return block_matmul(store.view(0, 300), w8), store.read(slots, torch.float32), quantize_both(x, col_sums=True)[2]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for _ in range(2):
        x.normal_()
        graph.replay()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_linear8_without_rows():
    x, W, b = (torch.randn(*s, device="cuda").requires_grad_() for s in ((0, 64), (64, 32), (32,)))
    y = linear8(x, W, b)
    y.sum().backward()
    assert y.shape == (0, 32) and x.grad.shape == (0, 64)
    assert (W.grad == 0).all() and W.grad.shape == (64, 32) and (b.grad == 0).all()


# ------------------------------------------------------------------------------- the SAE on stored rows

@pytest.mark.parametrize("activation", ["relu", "jumprelu"])
def test_quantized_sae(activation):
    sae = saeflow_b200.SAE(200, 1000, activation, device="cuda", dtype=torch.bfloat16)
    sae.b_enc.normal_(0, 0.1)
    sae.b_dec.normal_(0, 0.1)
    if activation == "jumprelu":
        sae.threshold.uniform_(0.5, 1.0)
    store = ActivationStore(300, 200)
    store.append(torch.randn(300, 200, device="cuda"))
    rows = torch.randperm(300, device="cuda")[:77]
    q = saeflow_b200.QuantizedSAE(sae)
    x8 = store.take(rows)
    f = q.encode(x8, torch.float32)
    x = store.read(rows, torch.float32).cpu().double()
    W8 = ob.round_trip(sae.W_enc.cpu().T, tile=True)
    pre = (x - sae.b_dec.cpu().double()) @ W8.T + sae.b_enc.cpu().double()
    cut = sae.threshold.cpu().double() if activation == "jumprelu" else torch.zeros(1000, dtype=torch.float64)
    # the bias is a sum of 200 fp32 products, the pre-activation one of 200 more
    bound = 400 * 2.0 ** -22 * (x.abs() @ W8.abs().T + (sae.b_dec.cpu().double().abs() @ W8.abs().T) + 1)
    sure = (pre - cut).abs() > bound
    want = torch.where(pre > cut, pre, torch.zeros_like(pre))
    assert sure.double().mean() > 0.99
    assert ((f.cpu().double() - want).abs() <= bound)[sure].all()
    csr = q.encode_sparse(x8)
    dense = q.encode(x8)
    assert torch.equal(saeflow_b200.kernels.csr_to_dense(*csr, 1000), dense)
    assert torch.equal(q.forward(x8), saeflow_b200.decode_sparse(sae, csr))


# ------------------------------------------------------------------------------- refusals

def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    a = quantize(x)
    store = ActivationStore(8, 64)
    i = torch.arange(4, device="cuda")
    bad = [
        (lambda: quantize(x.double()), "dtype"),
        (lambda: quantize(x[0]), "2-D"),
        (lambda: BlockScaled(a.data, a.scales[:2]), "scales must be"),
        (lambda: BlockScaled(a.data[:, 1:], a.scales), "aligned"),
        (lambda: BlockScaled(a.data.view(torch.uint8), a.scales), "float8"),
        (lambda: BlockScaled(a.data, a.scales.int()), "uint8"),
        (lambda: BlockScaled(a.data, a.scales.cpu()), "CUDA"),
        (lambda: quantize(x, tile=True).rows(0, 2), "tiles"),
        (lambda: store.write(x[:, :32], i), "x must be"),
        (lambda: store.write(x, i[:3]), "slots must be"),
        (lambda: store.write(x, i.float()), "dtype"),
        (lambda: store.write(x, i.cpu()), "expected"),
        (lambda: store.read(i, torch.float64), "dtype"),
        (lambda: store.read(i[None]), "1-D"),
        (lambda: store.read(i, out=torch.empty(3, 64, device="cuda")), "out must be"),
        (lambda: write_rows(torch.randn(9, 64, device="cuda"), store.blocks), "more rows"),
        (lambda: write_rows(x, quantize(x, tile=True)), "row blocks"),
        (lambda: take_rows(quantize(x, tile=True), i), "row blocks"),
        (lambda: read_rows(a, i.cpu()), "expected"),
        (lambda: block_matmul(a, quantize(torch.randn(4, 65, device="cuda"))), "columns"),
        (lambda: block_matmul(a, a, activation="gelu"), "supports"),
        (lambda: block_matmul(a, a, activation="jumprelu"), "threshold"),
        (lambda: block_matmul(a, a, torch.zeros(5, device="cuda")), "bias must be"),
        (lambda: block_matmul(a, a, torch.zeros(4)), "bias must be"),
        (lambda: block_matmul(a, a, out_dtype=torch.float64), "dtype"),
        (lambda: block_matmul(a, a, out=torch.empty(4, 5, device="cuda")), "out must be"),
        (lambda: block_matmul(quantize(x[:, :0]), quantize(x[:, :0])), "no columns"),
        (lambda: linear8(x, x), "linear8 takes"),
        (lambda: linear8(x, x.T, torch.zeros(3, device="cuda")), "b must be"),
        (lambda: saeflow_b200.QuantizedSAE(saeflow_b200.SAE(64, 128, "topk", k=4, device="cuda")), "top-k"),
        (lambda: saeflow_b200.QuantizedSAE(saeflow_b200.SAE(64, 128, device="cuda")).encode(x), "BlockScaled"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()
    with pytest.raises(IndexError):
        store.view(3, 9)
    with pytest.raises(RuntimeError, match="unit column stride"):
        block_matmul(a, a, out=torch.empty(4, 4, device="cuda").T)


def test_example_trains_and_encodes_from_the_store():
    """examples/train_from_store.py at a small size: the loss falls, and the 8-bit encoder explains most of
    the stored activations."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "train_from_store.py"
    spec = importlib.util.spec_from_file_location("train_from_store", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    first, last, explained = example.main(["--rows", "8192", "--d-in", "192", "--d-sae", "1024", "--steps", "150"])
    assert last < 0.6 * first and explained > 0.5
