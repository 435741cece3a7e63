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
import functools

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

    __slots__ = ("_data", "_scales", "_tile", "_shape", "_device", "_ref", "_c")
    # What the library reads is in _c, with the tensors' addresses: a matrix is made anew, not changed.
    data = property(lambda self: self._data)
    scales = property(lambda self: self._scales)
    tile = property(lambda self: self._tile)
    shape = property(lambda self: self._shape)
    device = property(lambda self: self._device)

    def __init__(self, data, scales, tile=False):
        if data.dim() != 2 or scales.dim() != 2:
            raise ValueError(f"data and scales must be 2-D, got {tuple(data.shape)} and {tuple(scales.shape)}")
        if data.dtype != _F8:
            raise ValueError(f"data has dtype {data.dtype}; expected float8_e4m3fn")
        if scales.dtype != torch.uint8:
            raise ValueError(f"scales has dtype {scales.dtype}; expected uint8")
        self._device = _abi.require_cuda(("data", data), ("scales", scales))
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
        self._data, self._scales, self._tile, self._shape = data, scales, bool(tile), (R, K)
        # a single row's stride is never used; any covering multiple passes the library's checks
        dp = data.stride(0) if R > 1 else _cdiv(K, 16) * 16
        sp = scales.stride(0) if scales.shape[0] > 1 else _cdiv(want[1], 4) * 4
        self._c = _abi.SfBlocks(data.data_ptr(), scales.data_ptr(), R, K, dp, sp, int(self._tile), 0)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, rows, cols, tile=False, device=None):
        """Uninitialised, with the smallest aligned row pitches."""
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise ValueError(f"device is {dev}; saeflow_b200 runs on CUDA devices only")
        nb = _cdiv(cols, BLOCK)
        dp, sp, scale_rows = _cdiv(cols, 16) * 16, _cdiv(nb, 4) * 4, _cdiv(rows, BLOCK) if tile else rows
        data = torch.empty_strided((rows, cols), (dp, 1), dtype=_F8, device=dev)
        # a product reads scale bytes four at a time, so the padding is there; its values are never used
        scales = torch.empty(scale_rows, sp, dtype=torch.uint8, device=dev)
        self = cls.__new__(cls)
        self._data, self._scales = data, scales if sp == nb else scales[:, :nb]
        self._tile, self._shape, self._device = bool(tile), (rows, cols), data.device
        self._c = _abi.SfBlocks(data.data_ptr(), scales.data_ptr(), rows, cols, dp, sp, int(tile), 0)
        self._ref = ctypes.byref(self._c)
        return self

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


def _run(dev, fn, *args, retry=None):
    """Call a library function on `dev`'s current stream. True if it returned the status `retry`."""
    i = dev.index
    if torch._C._cuda_getDevice() == i:  # as torch.cuda.current_device, on an initialised device
        status = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _abi.stream_of(dev))
    if status and status != retry:
        _abi.check(status)
    return status != 0


def _index(t, name, n, dev):
    """`t` as a contiguous int64 tensor [n] on dev."""
    if t.dim() != 1 or n is not None and t.shape[0] != n:
        raise ValueError(f"{name} must be 1-D{'' if n is None else f' with {n} entries'}, got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if t.dtype != torch.int64:
        if t.dtype != torch.int32:
            raise ValueError(f"{name} has dtype {t.dtype}; expected int64 or int32")
        t = t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


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
    """act(a @ b.T + bias) -> [M, N], products on the 8-bit tensor cores, accumulated in fp32: truncated after
    every 32 products within ranges of K of at most 1024 (fp32 outputs) or 2560 (16-bit ones), rounded to
    nearest between the ranges.

    a [M, K], b [N, K]: BlockScaled, in row blocks or tiles each.
    bias: [N] or None. activation: None, "relu" or "jumprelu" (needs `threshold` [N]; 0 unless
      the sum is above it).
    out_dtype: fp32 / bf16 / fp16; out: a tensor to write into, unit column stride.

    ReLU keeps a NaN, JumpReLU makes it 0. The result has no gradient: bias and threshold are taken as they are,
    without their history (saeflow_b200.training.linear8 is the differentiable product).
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
    bias = _vector(bias, "bias", N, dev)
    threshold = _vector(threshold, "threshold", N, dev)
    if out is None:
        _abi.dtype_code(out_dtype, "out_dtype")
        out = torch.empty(M, N, dtype=out_dtype, device=dev)
    elif tuple(out.shape) != (M, N) or out.device != dev:
        raise ValueError(f"out must be {[M, N]} on {dev}, got {list(out.shape)} on {out.device}")
    _product(dev, a._ref, b._ref, bias, threshold, -1 if activation is None else ACTIVATIONS[activation], out)
    return out


def product_plan(a, b, out_dtype=torch.bfloat16):
    """How block_matmul computes a @ b.T: (rows, columns of a tile, splits of K, K of a sum in the tensor cores)."""
    plan = _abi.SfBlockPlan()
    out = _abi.SfMatrix(a._c.data, _abi.dtype_code(out_dtype, "out_dtype"), 0, a.shape[0], b.shape[0], b.shape[0], 1)
    with torch.cuda.device(a.device):
        _abi.check(_abi.load().sf_block_matmul_plan(a._ref, b._ref, ctypes.byref(out), ctypes.byref(plan)))
    return plan.tile_rows, plan.tile_cols, plan.splits, plan.range


def _vector(v, name, n, dev):
    """A [n] vector in contiguous fp32, or None."""
    if v is None:
        return None
    if tuple(v.shape) != (n,) or v.device != dev:
        raise ValueError(f"{name} must be [{n}] on {dev}, got {list(v.shape)} on {v.device}")
    if v.dtype != torch.float32:
        _abi.dtype_code(v.dtype, name)
        v = v.detach().to(torch.float32)
    return v if v.is_contiguous() else v.detach().contiguous()


def _product(dev, a, b, bias, threshold, activation, out):
    """sf_block_matmul on ctypes references. Most products need no scratch: it is asked for when one does."""
    lib = _abi.load()
    m = ctypes.byref(_abi.matrix(out, "out"))
    args = (a, b, bias.data_ptr() if bias is not None else None,
            threshold.data_ptr() if threshold is not None else None, activation, m)
    if _run(dev, lib.sf_block_matmul, *args, None, 0, retry=_abi.SF_ERR_WORKSPACE):
        need = ctypes.c_size_t(0)
        _abi.check(lib.sf_block_matmul_workspace(a, b, m, ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        _run(dev, lib.sf_block_matmul, *args, ws.data_ptr(), need.value)


@functools.lru_cache(maxsize=256)
def _linear8_bytes(M, K, N, x_code, W_code, needs, device_index):
    """Sizes of a step's buffers: they depend on the extents alone (and on the device's SM count)."""
    keep, temp, later = ctypes.c_size_t(0), ctypes.c_size_t(0), ctypes.c_size_t(0)
    with torch.cuda.device(device_index):
        _abi.check(_abi.load().sf_linear8_bytes(M, K, N, x_code, W_code, needs, ctypes.byref(keep), ctypes.byref(temp),
                                                ctypes.byref(later)))
    return keep.value, temp.value, later.value


def linear8_forward(x, W, b, needs):
    """(y, kept, backward's scratch bytes) of saeflow_b200.training.linear8: y = Q(x) @ Q(W) + b in x's dtype, and the
    buffer that its backward reads. needs: bits 1 dx, 2 dW, 4 db."""
    dev = _abi.require_cuda(("x", x), ("W", W), ("b", b))
    (M, K), N = x.shape, W.shape[1]
    xm, wm = _abi.matrix(x, "x"), _abi.matrix(W, "W")
    bias = _vector(b, "b", N, dev)
    lib = _abi.load()
    keep, temp, later = _linear8_bytes(M, K, N, xm.dtype, wm.dtype, needs, dev.index)
    y = torch.empty(M, N, dtype=x.dtype, device=dev)
    kept = torch.empty(keep, dtype=torch.uint8, device=dev) if keep else None
    scratch = torch.empty(temp, dtype=torch.uint8, device=dev)
    _run(dev, lib.sf_linear8_forward, ctypes.byref(xm), ctypes.byref(wm), bias.data_ptr() if bias is not None else None,
         ctypes.byref(_abi.matrix(y, "y")), needs, kept.data_ptr() if keep else None, scratch.data_ptr(), temp)
    return y, kept, later


def linear8_backward(dy, kept, K, x_dtype, W_dtype, needs, scratch_bytes):
    """(dx, dW, fp32 db) of linear8 from dy [M, N], M > 0, and its forward's buffer; None where not needed."""
    dev = _abi.require_cuda(("dy", dy))
    dm = _abi.matrix(dy, "dy")
    M, N = dy.shape
    dx = torch.empty(M, K, dtype=x_dtype, device=dev) if needs & 1 else None
    dW = torch.empty(K, N, dtype=W_dtype, device=dev) if needs & 2 else None
    db = torch.empty(N, dtype=torch.float32, device=dev) if needs & 4 else None
    scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=dev)
    _run(dev, _abi.load().sf_linear8_backward, ctypes.byref(dm), kept.data_ptr() if kept is not None else None, K, needs,
         ctypes.byref(_abi.matrix(dx, "dx")) if needs & 1 else None,
         ctypes.byref(_abi.matrix(dW, "dW")) if needs & 2 else None,
         db.data_ptr() if needs & 4 else None, scratch.data_ptr(), scratch_bytes)
    return dx, dW, db
