"""Train a small SAE on activations held in 8 bits, then encode the store with it.

    python examples/train_from_store.py [--rows 65536] [--d-in 768] [--d-sae 4096] [--steps 200]

The operators together, as a training run uses them: batches are appended to an ActivationStore
(quantised as they are written, padded tokens dropped), shuffled rows are read back for each step, a
ReLU SAE with an L1 penalty is trained with 8-bit products in both directions (linear8), and the
trained SAE encodes rows of the store as they are held (QuantizedSAE), without dequantising them.
Activations are synthetic: sparse sums of unit-norm directions, with token norms that vary.
"""

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import saeflow_b200  # noqa: E402
from saeflow_b200.training import linear8  # noqa: E402


def activations(directions, rows):
    """`rows` sums of about eight of the directions, of varying norm."""
    n = directions.shape[0]
    code = torch.rand(rows, n, device=directions.device)
    code = torch.where(code < 8 / n, 1 + code, torch.zeros_like(code))
    return code @ directions * torch.exp(0.3 * torch.randn(rows, 1, device=directions.device))


def fill(store, directions, rows, batch=8192):
    """Harvest `rows` activations into the store; one token in 16 is padding, which is not kept."""
    kept = 0
    while kept < rows:
        x = activations(directions, batch)
        real = torch.rand(batch, device=x.device) >= 1 / 16
        slots = torch.where(real, kept + real.cumsum(0) - 1, -1)
        slots = torch.where(slots < rows, slots, -1)  # the store is full: drop the rest
        store.write(x, slots)
        kept += int(real.sum())


def train(store, sae, steps, batch=4096, lr=1e-3, l1=2e-3):
    """Adam on mean squared error + l1 |f|; returns the losses of the first and last step."""
    params = [sae.W_enc, sae.b_enc, sae.W_dec, sae.b_dec]
    for p in params:
        p.requires_grad_(True)
    opt = torch.optim.Adam(params, lr=lr)
    first = last = None
    for _ in range(steps):
        rows = torch.randint(store.capacity, (batch,), device=store.device)
        x = store.read(rows, torch.bfloat16)
        f = torch.relu(linear8(x - sae.b_dec.to(x.dtype), sae.W_enc, sae.b_enc))
        x_hat = linear8(f, sae.W_dec, sae.b_dec)
        loss = (x_hat.float() - x.float()).square().sum(1).mean() + l1 * f.float().sum(1).mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        last = loss.detach()
        first = last if first is None else first
    for p in params:
        p.requires_grad_(False)
    return float(first), float(last)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=65536)
    ap.add_argument("--d-in", type=int, default=768)
    ap.add_argument("--d-sae", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=200)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    directions = torch.nn.functional.normalize(torch.randn(a.d_sae // 4, a.d_in, device="cuda"), dim=1)
    store = saeflow_b200.ActivationStore(a.rows, a.d_in)
    fill(store, directions, a.rows)
    sae = saeflow_b200.SAE(a.d_in, a.d_sae, device="cuda")
    first, last = train(store, sae, a.steps)
    quantized = saeflow_b200.QuantizedSAE(sae)
    rows = torch.randint(a.rows, (4096,), device="cuda")
    csr = quantized.encode_sparse(store.take(rows), torch.float32)
    x = store.read(rows, torch.float32)
    x_hat = quantized.decode_sparse(csr)
    explained = 1 - float((x - x_hat).square().sum() / (x - x.mean(0)).square().sum())
    l0 = csr[1].numel() / len(rows)
    mb = store.blocks.data.numel() + store.blocks.scales.numel()
    print(f"store {a.rows} x {a.d_in}: {mb / 1e6:.1f} MB; loss {first:.4f} -> {last:.4f}; "
          f"8-bit encoder: explained variance {explained:.3f}, L0 {l0:.1f}")
    return first, last, explained


if __name__ == "__main__":
    main()
