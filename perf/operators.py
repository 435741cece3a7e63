"""What the 8-bit operators are measured on: quantised activation stores and block-scaled products.

Format. A matrix [R, K] is held as e4m3 numbers and power-of-two scales, one scale byte s (worth
2^(s - 127)) for each block of 128 columns of a row ("row blocks") or of 128 rows x 128 columns
("tiles"); the last blocks of a ragged matrix are smaller. s is the smallest byte whose scale
brings the block's largest finite magnitude to at most 448; each element is its quotient by the
scale, rounded once to e4m3 (nearest, ties to even).

Operators:
  write   quantise T rows of activations into the slots of a store (a slot below 0 drops the row)
  read    gather n rows of a store and dequantise them (a row below 0 reads as zeros)
  encode  act(a @ b^T + bias) of two quantised matrices: stored activations (row blocks) against
          encoder weights (tiles)
  train   y = x @ W + b with 8-bit operands and its gradients: x and the output's gradient are
          quantised along the axis that each product sums over, W in tiles

`run` computes them in plain torch where `own` is false, and with saeflow_b200's kernels where
it is true.
"""

import math

import torch

own = False

BLOCK = 128
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token of a generating model harvested at a 768-wide hook: launch latency
        {"name": "write 1x768", "op": "write", "rows": 1, "d": 768, "dtype": "bf16", "capacity": 4096,
         "slots": "run", "dropped": 0.0, "lead": 0},
        # a padded batch at a 2304-wide hook, one row in eight masked out, scattered over the store
        {"name": "write 4095x2304 masked", "op": "write", "rows": 4095, "d": 2304, "dtype": "bf16",
         "capacity": 16384, "slots": "spread", "dropped": 0.125, "lead": 0},
        # a large fp32 harvest appended to the store
        {"name": "write 65536x2304 fp32", "op": "write", "rows": 65536, "d": 2304, "dtype": "fp32",
         "capacity": 65536, "slots": "run", "dropped": 0.0, "lead": 0},
        # part of a wider hook (rows not 16-byte aligned) of odd width
        {"name": "write 5000x1001 slice", "op": "write", "rows": 5000, "d": 1001, "dtype": "fp16",
         "capacity": 8192, "slots": "spread", "dropped": 0.02, "lead": 3},
        # one row looked up for inspection
        {"name": "read 1x768", "op": "read", "rows": 1, "d": 768, "dtype": "fp32", "capacity": 4096},
        # a shuffled training batch out of a large store
        {"name": "read 16384x2304", "op": "read", "rows": 16384, "d": 2304, "dtype": "bf16", "capacity": 262144},
        # one token against a 65536-feature dictionary: the weights' bytes
        {"name": "encode 1x2304x65536", "op": "encode", "rows": 1, "d": 2304, "features": 65536, "dtype": "bf16",
         "activation": "relu"},
        # a short odd prompt
        {"name": "encode 100x768x16384", "op": "encode", "rows": 100, "d": 768, "features": 16384, "dtype": "bf16",
         "activation": "relu"},
        # ragged in every extent, no activation
        {"name": "encode 3001x1000x24577", "op": "encode", "rows": 3001, "d": 1000, "features": 24577,
         "dtype": "fp16", "activation": "none"},
        # the benchmark's batch
        {"name": "encode 16384x2304x65536", "op": "encode", "rows": 16384, "d": 2304, "features": 65536,
         "dtype": "bf16", "activation": "relu"},
        # a small ragged training step
        {"name": "train 1000x768x5000", "op": "train", "rows": 1000, "d": 768, "features": 5000, "dtype": "bf16"},
        # a training step of a large dictionary
        {"name": "train 8192x2304x16384", "op": "train", "rows": 8192, "d": 2304, "features": 16384,
         "dtype": "bf16"},
    ]


LARGEST_COST = 16384 * 2304 * 65536 * 2 / 4.0e15  # seconds of the largest listed case at a nominal rate


def _size(rng, low, high, multiple):
    """An extent spread over its logarithm: a multiple of `multiple` half of the time, any number otherwise."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5:
        n = max(multiple, n // multiple * multiple)
    return n + 1 if n == 3072 else n


def draw(rng):
    while True:
        op = rng.choice(["write", "read", "encode", "train"])
        case = {"op": op, "rows": _size(rng, 1, 65536 if op in ("write", "read") else 16384, 64)}
        case["d"] = _size(rng, 64, 4608, 128)
        case["dtype"] = rng.choice(["fp32", "bf16", "fp16"] if op in ("write", "read") else ["bf16", "bf16", "fp16"])
        if op == "write":
            case["capacity"] = int(case["rows"] * rng.choice([1, 2, 4])) + rng.randrange(1000)
            case["slots"] = rng.choice(["run", "spread"])
            case["dropped"] = rng.choice([0.0, 0.0, 0.1, 0.5])
            case["lead"] = rng.choice([0, 0, 1, 8, 16])
            small = case["rows"] * case["d"] <= 65536 * 2304 and case["capacity"] * case["d"] <= 1 << 29
        elif op == "read":
            case["capacity"] = 1000 + int(case["rows"] * rng.choice([1, 4, 16]))
            small = case["rows"] * case["d"] <= 65536 * 2304 and case["capacity"] * case["d"] <= 1 << 30
        else:
            if op == "train":
                case["rows"] = max(16, case["rows"])
            case["features"] = _size(rng, 256, 65536, 128)
            if op == "encode":
                case["activation"] = rng.choice(["relu", "none"])
            small = True
        w = work(case)
        if small and w["flops"] / 4.0e15 + w["bytes"] / 8.0e12 <= LARGEST_COST:
            return case


def work(case):
    M, K, es = case["rows"], case["d"], 4 if case["dtype"] == "fp32" else 2
    blocks = -(-K // BLOCK)
    if case["op"] == "write":
        kept = M - int(case["dropped"] * M)
        return {"bytes": M * K * es + 8 * M + kept * (K + blocks), "flops": 0}
    if case["op"] == "read":
        return {"bytes": M * (K + blocks) + 8 * M + M * K * es, "flops": 0}
    N = case["features"]
    if case["op"] == "encode":
        return {"bytes": M * (K + blocks) + N * K + -(-N // BLOCK) * blocks + 4 * N + M * N * es,
                "flops": 2 * M * N * K}
    return {"bytes": (2 * M * K + 2 * K * N + 2 * M * N) * es + 8 * N, "flops": 6 * M * N * K}


# ------------------------------------------------------------------------------- plain forms

def _padded(rows, cols, multiple, dtype, device):
    """[rows, cols] of zeros whose row pitch is a multiple of `multiple` elements."""
    return torch.zeros(rows, -(-cols // multiple) * multiple, dtype=dtype, device=device)[:, :cols]


def _blocks(x):
    """[R, K] in fp32 with zeros up to whole blocks: [R, K / 128, 128]."""
    R, K = x.shape
    nb = -(-K // BLOCK)
    return torch.nn.functional.pad(x.float(), (0, nb * BLOCK - K)).view(R, nb, BLOCK)


def _scale_byte(amax):
    """The smallest byte s with amax <= 448 * 2^(s - 127): 448 = 1.75 * 2^8, so the exponent
    field of amax less 8, one more where its mantissa is above 1.75."""
    return (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=0)


def _power(byte):
    """2^(byte - 127) in fp32 (byte 0 is a subnormal)."""
    return torch.where(byte > 0, byte << 23, torch.full_like(byte, 1 << 22)).view(torch.float32)


def _quantise(x, tile=False):
    """e4m3 [R, K] and scale bytes of row blocks [R, nb] or tiles [ceil(R / 128), nb]."""
    R, K = x.shape
    v = _blocks(x)
    amax = v.abs().amax(-1)
    if tile:
        nt = -(-R // BLOCK)
        amax = torch.nn.functional.pad(amax, (0, 0, 0, nt * BLOCK - R)).view(nt, BLOCK, -1).amax(1)
    byte = _scale_byte(amax)
    inverse = ((254 - byte) << 23).view(torch.float32)
    if tile:
        inverse = inverse.repeat_interleave(BLOCK, 0)[:R]
    q = (v * inverse[..., None]).view(R, -1)[:, :K].to(torch.float8_e4m3fn)
    return q, byte.to(torch.uint8)


def _dequantise(q, byte, tile=False):
    """fp32 [R, K] of a quantised matrix."""
    R, K = q.shape
    s = _power(byte.to(torch.int32))
    if tile:
        s = s.repeat_interleave(BLOCK, 0)[:R]
    return (_blocks(q) * s[..., None]).view(R, -1)[:, :K]


def _round_trip(x, tile=False):
    return _dequantise(*_quantise(x, tile), tile)


# ------------------------------------------------------------------------------- inputs

def _activations(g, rows, d, device="cuda"):
    """Rows as a language model's residual stream gives them: norms that vary from token to
    token and a few channels of far larger magnitude."""
    x = torch.randn(rows, d, device=device, generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device=device, generator=g))
    loud = torch.randint(0, d, (max(1, d // 256),), device=device, generator=g)
    x[:, loud] *= 30.0
    return x


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    M, K, dtype = case["rows"], case["d"], DTYPES[case["dtype"]]
    nb = -(-K // BLOCK)
    s = {"case": case, "dtype": dtype}
    if case["op"] in ("write", "read"):
        cap = case["capacity"]
        s["data"] = _padded(cap, K, 16, torch.float8_e4m3fn, "cuda")
        s["scales"] = _padded(cap, nb, 4, torch.uint8, "cuda")
        if case["op"] == "write":
            lead = case["lead"]
            s["x"] = _activations(g, M, K + lead).to(dtype)[:, lead:]
            if case["slots"] == "run":
                first = (cap - M) // 2
                slots = torch.arange(first, first + M, device="cuda")
            else:
                slots = torch.randperm(cap, device="cuda", generator=g)[:M]
            drop = torch.randperm(M, device="cuda", generator=g)[:int(case["dropped"] * M)]
            slots[drop] = -1
            s["slots"] = slots
        else:
            for r in range(0, cap, 65536):
                q, byte = _quantise(_activations(g, min(65536, cap - r), K))
                s["data"][r:r + 65536], s["scales"][r:r + 65536] = q, byte
            s["rows"] = torch.randint(0, cap, (M,), device="cuda", generator=g)
        if own:
            from saeflow_b200.store import ActivationStore

            s["store"] = ActivationStore.wrap(s["data"], s["scales"])
        return s
    N = case["features"]
    W = torch.randn(N, K, device="cuda", generator=g)
    W /= W.norm(dim=1, keepdim=True)
    s["b"] = torch.randn(N, device="cuda", generator=g) - 1.0
    x = _activations(g, M, K)
    if case["op"] == "train":
        s["x"] = x.to(dtype).requires_grad_()
        s["W"] = W.T.contiguous().to(dtype).requires_grad_()
        s["b"].requires_grad_()
        s["dy"] = (torch.randn(M, N, device="cuda", generator=g) * 1e-3).to(dtype)
        return s
    for name, v, tile in (("x", x, False), ("W", W, True)):
        q, byte = _quantise(v, tile)
        s[name] = _padded(*v.shape, 16, torch.float8_e4m3fn, "cuda")
        s[name + "s"] = _padded(byte.shape[0], nb, 4, torch.uint8, "cuda")
        s[name][:], s[name + "s"][:] = q, byte
    if own:
        from saeflow_b200.kernels import BlockScaled

        s["a8"] = BlockScaled(s["x"], s["xs"])
        s["b8"] = BlockScaled(s["W"], s["Ws"], tile=True)
    return s


# ------------------------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    op = s["case"]["op"]
    if op == "write":
        s["store"].write(s["x"], s["slots"])
        return {"data": s["data"], "scales": s["scales"]}
    if op == "read":
        return s["store"].read(s["rows"], dtype=s["dtype"])
    if op == "encode":
        from saeflow_b200.kernels import block_matmul

        act = s["case"]["activation"]
        return block_matmul(s["a8"], s["b8"], s["b"], activation=None if act == "none" else act,
                            out_dtype=s["dtype"])
    from saeflow_b200.training import linear8

    y = linear8(s["x"], s["W"], s["b"])
    dx, dW, db = torch.autograd.grad(y, (s["x"], s["W"], s["b"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dW": dW, "db": db}


@torch.no_grad()
def _run_plain(s):
    op, dtype = s["case"]["op"], s["dtype"]
    if op == "write":
        q, byte = _quantise(s["x"])
        kept = s["slots"] >= 0
        slots = s["slots"][kept]
        s["data"].view(torch.uint8)[slots] = q.view(torch.uint8)[kept]
        s["scales"][slots] = byte[kept]
        return {"data": s["data"], "scales": s["scales"]}
    if op == "read":
        q = s["data"].view(torch.uint8)[s["rows"]].view(torch.float8_e4m3fn)
        return _dequantise(q, s["scales"][s["rows"]]).to(dtype)
    if op == "encode":
        y = _dequantise(s["x"], s["xs"]) @ _dequantise(s["W"], s["Ws"], tile=True).T + s["b"]
        if s["case"]["activation"] == "relu":
            y = torch.relu(y)
        return y.to(dtype)
    x, W, dy = s["x"], s["W"], s["dy"]
    W8 = _round_trip(W, tile=True)
    y = (_round_trip(x) @ W8 + s["b"]).to(dtype)
    dx = (_round_trip(dy) @ W8.T).to(dtype)
    dW = (_round_trip(x.T) @ _round_trip(dy.T).T).to(dtype)
    return {"y": y, "dx": dx, "dW": dW, "db": dy.float().sum(0)}


# ------------------------------------------------------------------------------- in 64 bits

def _exact_numbers(x, tile=False):
    """(numbers, scales) of a matrix from the format's definition, both in 64 bits and of x's
    shape: the exponent of the largest magnitude by frexp, the e4m3 grid as multiples of its step."""
    R, K = x.shape
    x = x.double()
    # largest magnitude of each block, by indices of the blocks that the elements fall into
    col = (torch.arange(K, device=x.device) // BLOCK).expand(R, K)
    top = torch.zeros(R, -(-K // BLOCK), dtype=torch.float64, device=x.device).scatter_reduce(
        1, col, x.abs(), "amax")
    if tile:
        row = torch.arange(R, device=x.device) // BLOCK
        top = torch.stack([t.amax(0) for t in top.split(BLOCK)])[row]
    m, e = torch.frexp(top)  # top = m 2^e with m in [1/2, 1); 448 = 0.875 * 2^9
    e = e.double() - 9 + (m > 0.875).double()
    e = torch.where(top > 0, e, torch.full_like(e, -127.0)).clamp(min=-127)
    scale = torch.exp2(e).gather(1, col)
    t = x / scale
    _, te = torch.frexp(t)
    step = torch.exp2((te.double() - 1).clamp(min=-6) - 3)  # 3 bits after the leading one, subnormal below 2^-6
    return torch.round(t / step) * step, scale


def _exact_values(x, tile=False):
    n, scale = _exact_numbers(x, tile)
    return n * scale


def _exact_of_stored(q, byte, tile=False):
    R, K = q.shape
    row = torch.arange(R, device=q.device) // (BLOCK if tile else 1)
    col = torch.arange(K, device=q.device) // BLOCK
    return q.double() * torch.exp2(byte.double() - 127)[row][:, col]


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":
        kept = s["slots"] >= 0
        data = torch.zeros(s["data"].shape, dtype=torch.float64, device="cuda")
        for first in range(0, case["rows"], 8192):  # in parts, for the sake of memory
            part = slice(first, first + 8192)
            data[s["slots"][part][kept[part]]] = _exact_numbers(s["x"][part])[0][kept[part]]
        return {"data": data, "scales": None}
    if case["op"] == "read":
        q = s["data"].float()[s["rows"]]
        return _exact_of_stored(q, s["scales"][s["rows"]])
    if case["op"] == "encode":
        y = _exact_of_stored(s["x"], s["xs"]) @ _exact_of_stored(s["W"], s["Ws"], tile=True).T
        y += s["b"].double()
        return y.clamp_(min=0) if case["activation"] == "relu" else y
    x, W, dy = s["x"], s["W"], s["dy"]
    W8 = _exact_values(W, tile=True)
    return {"y": _exact_values(x) @ W8 + s["b"].double(), "dx": _exact_values(dy) @ W8.T,
            "dW": _exact_values(x.T) @ _exact_values(dy.T).T, "db": dy.double().sum(0)}
