"""Plain 64-bit forms of the block-scaled 8-bit operators, from the format's definition.

A matrix [R, C] is e4m3 numbers q and scale bytes s, one per 128 columns of a row or per 128 x 128
tile; an element is worth q 2^(s - 127). s is the smallest byte whose scale brings the block's
largest finite magnitude to at most 448; q is the quotient by the scale rounded to the nearest e4m3,
ties to even; what is not finite becomes NaN.
"""

import torch

BLOCK = 128


def _spread(per_block, shape, tile):
    """[R, C] of each element's block value."""
    R, C = shape
    rows = torch.arange(R) // (BLOCK if tile else 1)
    return per_block[rows][:, torch.arange(C) // BLOCK]


def scale_bytes(x, tile=False):
    """int64 scale bytes of x [R, C]."""
    R, C = x.shape
    x = x.double()
    mag = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    top = torch.stack([b.amax(1) for b in mag.split(BLOCK, 1)], 1)
    if tile:
        top = torch.stack([b.amax(0) for b in top.split(BLOCK, 0)])
    s = torch.zeros(top.shape, dtype=torch.int64)
    for byte in range(254, -1, -1):  # the smallest byte that is enough
        s = torch.where(top <= 448.0 * 2.0 ** (byte - 127), torch.full_like(s, byte), s)
    return s


def e4m3_values():
    """All non-negative finite e4m3 numbers, ascending, and whether each has an even mantissa."""
    values = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)]
    values = values[:-1]  # the last code is NaN
    return torch.tensor(values, dtype=torch.float64), torch.arange(len(values)) % 2 == 0


def round_e4m3(t):
    """t in float64 rounded to the nearest e4m3 number by search, ties to the even mantissa."""
    grid, even = e4m3_values()
    a = t.abs().clamp(max=448.0)
    hi = torch.searchsorted(grid, a).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    take_hi = (up < down) | ((up == down) & even[hi])
    r = torch.where(take_hi, grid[hi], grid[lo])
    r = torch.copysign(r, t)
    return torch.where(torch.isfinite(t), r, torch.full_like(r, float("nan")))


def quantize(x, tile=False):
    """(q float64 [R, C], s int64) of x."""
    s = scale_bytes(x, tile)
    scale = torch.exp2(_spread(s, x.shape, tile).double() - 127)
    return round_e4m3(x.double() / scale), s


def dequantize(q, s, tile=False):
    """float64 values of numbers q (any float type) and bytes s."""
    return q.double() * torch.exp2(_spread(s.long(), q.shape, tile).double() - 127)


def round_trip(x, tile=False):
    return dequantize(*quantize(x, tile), tile)


def matmul(a, b, bias=None, activation=None, threshold=None):
    """(act(a @ b.T + bias), sum_k |a||b|) of float64 matrices."""
    y = a @ b.T
    if bias is not None:
        y = y + bias.double()
    if activation == "relu":
        y = torch.relu(y)
    elif activation == "jumprelu":
        y = torch.where((y > threshold.double()) & (y > 0), y, torch.zeros_like(y))
    return y, a.abs() @ b.abs().T


def linear(x, W, b, dy):
    """y, dx, dW, db of the 8-bit linear step in float64, each with the sum of its products' magnitudes."""
    xr, xc = round_trip(x), round_trip(x.T)
    dyr, dyc = round_trip(dy), round_trip(dy.T)
    W8 = round_trip(W, tile=True)
    y, my = matmul(xr, W8.T, b)
    dx, mx = matmul(dyr, W8)
    dW, mw = matmul(xc, dyc)
    return (y, dx, dW, dy.double().sum(0)), (my, mx, mw, dy.double().abs().sum(0))
