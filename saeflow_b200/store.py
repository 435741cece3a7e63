"""A GPU-resident store of activations in 8 bits: quantised as it is written, read back by row.

Training an SAE reads its activations shuffled, many times over, and a row of d_in = 2304 takes 4608
bytes in bf16 but 2322 here (e4m3 with one power-of-two scale per 128 columns), so a GPU holds twice
as many. The rows are also operands as they lie: `take` and `view` give batches that
saeflow_b200.quantized.QuantizedSAE encodes without dequantising them.

The on-disk cache (saeflow_b200.cache) keeps activations in 16 or 32 bits, as the reference's does
(saeflow/cache.py:70-137); `ActivationReader.iter_batches(device=...)` feeds `append`.
"""

from __future__ import annotations

import torch

from .kernels.blocks import BLOCK, BlockScaled, read_rows, take_rows, write_rows


class ActivationStore:
    """`capacity` rows of width d on a CUDA device, zeros until written.

    write(x, slots): rows of x into the given slots; append(x): into the next ones, around the end.
    read(rows): rows by index, dequantised; take(rows), view(start, stop): rows as held.
    """

    def __init__(self, capacity, d, device=None):
        if capacity < 1 or d < 1:
            raise ValueError(f"a store needs at least one row and column, got {capacity} x {d}")
        blocks = BlockScaled.empty(capacity, d, device=device)
        blocks.data.view(torch.uint8).zero_()
        blocks.scales.zero_()
        self._adopt(blocks)

    def _adopt(self, blocks):
        self.blocks = blocks
        self.written = 0  # rows appended so far, over all laps

    @classmethod
    def wrap(cls, data, scales):
        """A store over existing tensors (float8_e4m3fn [capacity, d] and uint8 [capacity,
        ceil(d / 128)], aligned as BlockScaled asks), e.g. of a store saved earlier."""
        store = cls.__new__(cls)
        store._adopt(BlockScaled(data, scales))
        return store

    @property
    def capacity(self):
        return self.blocks.shape[0]

    @property
    def d(self):
        return self.blocks.shape[1]

    @property
    def device(self):
        return self.blocks.device

    def __len__(self):
        """Rows that hold appended activations."""
        return min(self.written, self.capacity)

    @staticmethod
    def bytes_per_row(d):
        return -(-d // 16) * 16 + -(-d // (4 * BLOCK)) * 4

    def write(self, x, slots):
        """Quantise x [T, d] (fp32 / bf16 / fp16, any strides) into rows `slots` (int64 [T], distinct).
        A negative slot drops its row (padding, masked tokens)."""
        if x.dim() != 2 or x.shape[1] != self.d:
            raise ValueError(f"x must be [T, {self.d}], got {tuple(x.shape)}")
        write_rows(x, self.blocks, slots)

    def append(self, x):
        """Quantise x [T, d] into the next T rows, overwriting the oldest once the store is full."""
        if x.dim() != 2 or x.shape[1] != self.d:
            raise ValueError(f"x must be [T, {self.d}], got {tuple(x.shape)}")
        lost = max(0, x.shape[0] - self.capacity)  # rows that this very call would overwrite
        x = x[lost:]
        first = (self.written + lost) % self.capacity
        head = min(x.shape[0], self.capacity - first)
        if head:
            write_rows(x[:head], self.blocks.rows(first, first + head))
        if x.shape[0] > head:
            write_rows(x[head:], self.blocks.rows(0, x.shape[0] - head))
        self.written += lost + x.shape[0]

    def read(self, rows, dtype=torch.bfloat16, out=None):
        """Rows `rows` (int64 [n]) dequantised, [n, d] in `dtype`; a negative row reads as zeros."""
        return read_rows(self.blocks, rows, dtype, out)

    def take(self, rows):
        """Rows `rows` as a BlockScaled batch of their own."""
        return take_rows(self.blocks, rows)

    def view(self, start, stop):
        """Rows [start, stop) as a BlockScaled batch in place."""
        if not 0 <= start <= stop <= self.capacity:
            raise IndexError(f"rows [{start}, {stop}) outside the store's {self.capacity}")
        return self.blocks.rows(start, stop)
