"""Block-scaled 8-bit matrices (libsaeflow_b200.so, csrc/blocks.cu and csrc/block_gemm.cu).

A BlockScaled matrix holds e4m3 numbers and one power-of-two scale per 128 columns of a row ("row
blocks": activations and gradients) or per 128 x 128 tile (weights, whose transpose then has the
same scales). Its blocks are the tensor cores' own operands: block_matmul reads them as they lie.
The reference has neither (it keeps activations in 16 or 32 bits).

- quantize / quantize_both: from fp32 / bf16 / fp16, x itself, its transpose, or both in one pass;
- write_rows / read_rows / take_rows: a store's rows by index, quantised in, dequantised out, or
  gathered as they are;
- block_matmul: act(a @ b.T + bias).
"""

from __future__ import annotations

import ctypes

import torch

from .. import _abi
from .encode import ACTIVATIONS

BLOCK = _abi.BLOCK
_F8 = torch.float8_e4m3fn


def _cdiv(a, b):
    return -(-a // b)


class BlockScaled:
    """An 8-bit matrix [rows, cols] on a CUDA device.

    data: float8_e4m3fn [rows, cols], unit column stride, base and row pitch 16-byte aligned.
    scales: uint8 [rows, ceil(cols / 128)], or [ceil(rows / 128), ceil(cols / 128)] with
      tile=True; unit column stride, base and row pitch 4-byte aligned. Byte s is worth
      2^(s - 127).
    """

    __slots__ = ("data", "scales", "tile", "shape", "device", "_ref", "_c")

    def __init__(self, data, scales, tile=False):
        if data.dim() != 2 or scales.dim() != 2:
            raise ValueError(f"data and scales must be 2-D, got {tuple(data.shape)} and {tuple(scales.shape)}")
        if data.dtype != _F8:
            raise ValueError(f"data has dtype {data.dtype}; expected float8_e4m3fn")
        if scales.dtype != torch.uint8:
            raise ValueError(f"scales has dtype {scales.dtype}; expected uint8")
        self.device = _abi.require_cuda(("data", data), ("scales", scales))
        R, K = data.shape
        want = (_cdiv(R, BLOCK) if tile else R, _cdiv(K, BLOCK))
        if tuple(scales.shape) != want:
            raise ValueError(f"scales must be {list(want)} for {'tiles' if tile else 'row blocks'} of {[R, K]}, "
                             f"got {list(scales.shape)}")
        for name, t, align in (("data", data, 16), ("scales", scales, 4)):
            if t.numel() and (t.stride(1) != 1 and t.shape[1] > 1 or t.shape[0] > 1 and t.stride(0) % align
                              or t.shape[0] > 1 and t.stride(0) < t.shape[1] or t.data_ptr() % align):
                raise ValueError(f"{name} needs a unit column stride and {align}-byte aligned rows, got strides "
                                 f"{t.stride()}")
        self.data, self.scales, self.tile, self.shape = data, scales, bool(tile), (R, K)
        # a single row's stride is never used; any covering multiple passes the library's checks
        dp = data.stride(0) if R > 1 else _cdiv(K, 16) * 16
        sp = scales.stride(0) if scales.shape[0] > 1 else _cdiv(want[1], 4) * 4
        self._c = _abi.SfBlocks(data.data_ptr(), scales.data_ptr(), R, K, dp, sp, int(self.tile), 0)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, rows, cols, tile=False, device=None):
        """Uninitialised, with the smallest aligned row pitches."""
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise ValueError(f"device is {dev}; saeflow_b200 runs on CUDA devices only")
        nb = _cdiv(cols, BLOCK)
        data = torch.empty(rows, _cdiv(cols, 16) * 16, dtype=_F8, device=dev)[:, :cols]
        # a product reads scale bytes four at a time; the padding's values are never used
        scales = torch.empty(_cdiv(rows, BLOCK) if tile else rows, _cdiv(nb, 4) * 4, dtype=torch.uint8,
                             device=dev)[:, :nb]
        return cls(data, scales, tile)

    def rows(self, start, stop):
        """Rows [start, stop) in place (row blocks only)."""
        if self.tile:
            raise ValueError("tiles cannot be sliced by rows")
        return BlockScaled(self.data[start:stop], self.scales[start:stop])

    def dequantize(self, dtype=torch.float32):
        """The matrix in `dtype` (fp32 / bf16 / fp16)."""
        return read_rows(self, None, dtype)

    def __repr__(self):
        return f"BlockScaled({list(self.shape)}, {'tiles' if self.tile else 'row blocks'}, {self.device})"


def _run(dev, fn, *args):
    """Call a library function on `dev`'s current stream."""
    if torch.cuda.current_device() == dev.index:
        _abi.check(fn(*args, _abi.stream_of(dev)))
    else:
        with torch.cuda.device(dev):
            _abi.check(fn(*args, _abi.stream_of(dev)))


def _index(t, name, n, dev):
    """`t` as a contiguous int64 tensor [n] on dev."""
    if t.dim() != 1 or n is not None and t.shape[0] != n:
        raise ValueError(f"{name} must be 1-D{'' if n is None else f' with {n} entries'}, got {tuple(t.shape)}")
    if t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} has dtype {t.dtype}; expected int64 or int32")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    return t.to(torch.int64).contiguous()


def quantize(x, *, tile=False, transpose=False):
    """x [R, C] as a BlockScaled matrix, or its transpose [C, R] with transpose=True: blocks run
    along the columns of the result."""
    q, qt, _ = quantize_both(x, tile=tile, want=(not transpose, transpose))
    return qt if transpose else q


def quantize_both(x, *, tile=False, want=(True, True), col_sums=False):
    """(x, x.T, column sums) from one pass over x [R, C]: both BlockScaled (None where `want`
    says so), and fp32 [C] sums of x's columns (None unless asked for), summed in a fixed order."""
    dev = _abi.require_cuda(("x", x))
    m = _abi.matrix(x, "x")
    R, C = x.shape
    q = BlockScaled.empty(R, C, tile, dev) if want[0] else None
    if q is not None and not tile and not want[1] and not col_sums:
        _run(dev, _abi.load().sf_blocks_write, ctypes.byref(m), None, q._ref)
        return q, None, None
    qt = BlockScaled.empty(C, R, tile, dev) if want[1] else None
    sums = torch.empty(C, dtype=torch.float32, device=dev) if col_sums else None
    n = _cdiv(R, BLOCK) * C if col_sums else 0
    ws = torch.empty(n, dtype=torch.float32, device=dev) if n else None
    _run(dev, _abi.load().sf_blocks_quantize, ctypes.byref(m), q._ref if q is not None else None,
         qt._ref if qt is not None else None, sums.data_ptr() if col_sums else None,
         ws.data_ptr() if n else None, 4 * n)
    return q, qt, sums


def write_rows(x, dst, slots=None):
    """Quantise the rows of x [T, cols] into the rows `slots` of dst (row blocks): slots int64 [T],
    distinct; a negative slot drops the row. slots=None: rows 0..T-1. A slot past the end is
    skipped and reported by device_error()."""
    dev = _abi.require_cuda(("x", x))
    if dst.device != dev:
        raise ValueError(f"x is on {dev}, the store on {dst.device}")
    m = _abi.matrix(x, "x")
    if slots is not None:
        slots = _index(slots, "slots", x.shape[0], dev)
    _run(dev, _abi.load().sf_blocks_write, ctypes.byref(m), slots.data_ptr() if slots is not None else None, dst._ref)


def read_rows(src, rows=None, dtype=torch.bfloat16, out=None):
    """The dequantised rows `rows` (int64 [n]; None: all) of src as [n, cols] in `dtype`. A negative
    row reads as zeros; so does one past the end, which device_error() reports."""
    dev = src.device
    if rows is not None:
        rows = _index(rows, "rows", None, dev)
    shape = (src.shape[0] if rows is None else rows.shape[0], src.shape[1])
    if out is None:
        _abi.dtype_code(dtype, "dtype")
        out = torch.empty(shape, dtype=dtype, device=dev)
    elif tuple(out.shape) != shape or out.device != dev or out.numel() and out.stride(1) != 1 and shape[1] > 1:
        raise ValueError(f"out must be {list(shape)} on {dev} with a unit column stride")
    m = _abi.matrix(out, "out")
    _run(dev, _abi.load().sf_blocks_read, src._ref, rows.data_ptr() if rows is not None else None, ctypes.byref(m))
    return out


def take_rows(src, rows):
    """The rows `rows` of src (row blocks) as a new BlockScaled matrix; rows as in read_rows."""
    rows = _index(rows, "rows", None, src.device)
    dst = BlockScaled.empty(rows.shape[0], src.shape[1], False, src.device)
    _run(src.device, _abi.load().sf_blocks_take, src._ref, rows.data_ptr(), dst._ref)
    return dst


def block_matmul(a, b, bias=None, activation=None, threshold=None, *, out_dtype=torch.bfloat16, out=None):
    """act(a @ b.T + bias) -> [M, N], products on the 8-bit tensor cores, accumulated in fp32.

    a [M, K], b [N, K]: BlockScaled, in row blocks or tiles each.
    bias: [N] or None. activation: None, "relu" or "jumprelu" (needs `threshold` [N]; 0 unless
      the sum is above it).
    out_dtype: fp32 / bf16 / fp16; out: a tensor to write into, unit column stride.
    """
    dev = a.device
    if b.device != dev:
        raise ValueError(f"b is on {b.device}, expected {dev}")
    (M, K), (N, K_b) = a.shape, b.shape
    if K != K_b:
        raise ValueError(f"a has {K} columns but b has {K_b}")
    if activation is not None and activation not in ACTIVATIONS:
        raise ValueError(f"block_matmul supports None and {list(ACTIVATIONS)}, got {activation!r}")
    if activation == "jumprelu" and threshold is None:
        raise ValueError("jumprelu needs a threshold")
    if activation != "jumprelu":
        threshold = None
    vectors = []
    for name, v in (("bias", bias), ("threshold", threshold)):
        if v is not None:
            if tuple(v.shape) != (N,) or v.device != dev:
                raise ValueError(f"{name} must be [{N}] on {dev}, got {list(v.shape)} on {v.device}")
            _abi.dtype_code(v.dtype, name)
            v = v.detach().to(torch.float32).contiguous()
        vectors.append(v)
    if out is None:
        _abi.dtype_code(out_dtype, "out_dtype")
        out = torch.empty(M, N, dtype=out_dtype, device=dev)
    elif tuple(out.shape) != (M, N) or out.device != dev:
        raise ValueError(f"out must be {[M, N]} on {dev}, got {list(out.shape)} on {out.device}")
    m = _abi.matrix(out, "out")
    lib = _abi.load()
    need = ctypes.c_size_t(0)
    _abi.check(lib.sf_block_matmul_workspace(a._ref, b._ref, ctypes.byref(m), ctypes.byref(need)))
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
    _run(dev, lib.sf_block_matmul, a._ref, b._ref, *(v.data_ptr() if v is not None else None for v in vectors),
         -1 if activation is None else ACTIVATIONS[activation], ctypes.byref(m),
         ws.data_ptr() if ws is not None else None, need.value)
    return out
