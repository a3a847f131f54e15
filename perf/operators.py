"""The 8-bit projections of a decoder layer, as they are timed: the plain forms and the calls of the kernels.

Rows and weights are held in e4m3 (`torch.float8_e4m3fn`) with one fp32 scale for every 128 consecutive inputs of a row and
for every 128 x 128 block of a weight matrix; a value is its e4m3 number times its scale.

    rmsnorm_fp8         h = x + residual, then the root-mean-square norm of h in 8 bits (a decoder layer's two norms)
    swiglu_fp8          silu(gate) * up in 8 bits (between the gate/up and the down projection)
    quantize_rows_fp8   rows as they are in 8 bits (the attention output before its projection)
    linear_fp8          the projection itself: few rows (one token per sequence) to whole prompts, with a residual or SwiGLU behind

Sizes: hidden 4096, feed-forward 14336, QKV 6144 of the decoder shape that `bench.py` runs; batches 1 to 16; prompts of
thousands of tokens; and sizes that are no multiple of anything.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128
LARGEST = 448.0          # largest e4m3 value
SMALLEST = 2.0 ** -96    # a block whose largest magnitude is below this is scaled as if it were this
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def _ops():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hashattention-1.0_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from hashattention import _ops as ops
    return ops


def listed():
    return [
        # one new token for each of 4 sequences: the norm in front of a decode step's projections
        {"name": "norm decode 4x4096", "op": "norm", "m": 4, "k": 4096, "dtype": "bf16", "residual": True},
        # a prompt of 8192 tokens
        {"name": "norm prompt 8192x4096", "op": "norm", "m": 8192, "k": 4096, "dtype": "bf16", "residual": True},
        # a ragged chunk in fp32, width no multiple of the block, first norm of a model (nothing to add)
        {"name": "norm ragged 777x5000", "op": "norm", "m": 777, "k": 5000, "dtype": "fp32", "residual": False},
        # feed-forward activations: one token for each of 16 sequences, and a prompt
        {"name": "swiglu decode 16x14336", "op": "swiglu", "m": 16, "k": 14336, "dtype": "bf16"},
        {"name": "swiglu prompt 4096x14336", "op": "swiglu", "m": 4096, "k": 14336, "dtype": "bf16"},
        # attention output of a decode step, and an odd fp16 chunk
        {"name": "rows decode 4x4096", "op": "rows", "m": 4, "k": 4096, "dtype": "bf16"},
        {"name": "rows chunk 1001x4100", "op": "rows", "m": 1001, "k": 4100, "dtype": "fp16"},
        # down projection of a decode step, residual behind
        {"name": "linear 4x4096x14336", "op": "linear", "m": 4, "n": 4096, "k": 14336, "out": "bf16", "behind": "residual"},
        # gate/up projection of a decode step at 16 sequences, SwiGLU behind
        {"name": "linear 16x28672x4096 glu", "op": "linear", "m": 16, "n": 28672, "k": 4096, "out": "bf16", "behind": "swiglu"},
        # QKV projection of a short chunk of tokens
        {"name": "linear 128x6144x4096", "op": "linear", "m": 128, "n": 6144, "k": 4096, "out": "bf16", "behind": "none"},
        # sizes that divide by nothing, fp32 out
        {"name": "linear 333x1000x1111", "op": "linear", "m": 333, "n": 1000, "k": 1111, "out": "fp32", "behind": "none"},
        # gate/up projection of a prompt of 4096 tokens
        {"name": "linear 4096x28672x4096", "op": "linear", "m": 4096, "n": 28672, "k": 4096, "out": "bf16", "behind": "none"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "swiglu", "rows", "linear", "linear"])
    m = log(1, 8192)
    k = log(64, 14336)
    if rng.random() < 0.5:
        k = max(128, k // 128 * 128)
    if op == "norm":
        return {"op": op, "m": m, "k": k, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "residual": rng.random() < 0.6}
    if op in ("swiglu", "rows"):
        return {"op": op, "m": m, "k": k, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    n = log(16, 28672)
    if rng.random() < 0.5:
        n = max(128, n // 128 * 128)
    while m * n * k > 4096 * 28672 * 4096:
        m //= 2
    behind = rng.choice(["none", "residual", "swiglu"])
    if behind == "swiglu":
        n += n % 2
    return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "behind": behind}


def _blocks(k):
    return -(-k // BLOCK)


def _quantise(y):
    """fp32 [m, k] -> (e4m3 [m, k], scales fp32 [m, blocks]): every block of 128 scaled so that its largest magnitude is 448."""
    m, k = y.shape
    kb = _blocks(k)
    y = torch.nn.functional.pad(y, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    top = y.abs().amax(dim=-1)
    floor = top.clamp(min=SMALLEST)
    q = (y * (LARGEST / floor).unsqueeze(-1)).to(torch.float8_e4m3fn).view(m, kb * BLOCK)[:, :k]
    scale = torch.where(top == 0, torch.ones_like(top), floor / LARGEST)
    return q, scale


def _quantise_weight(w):
    """fp32 [n, k] -> (e4m3 [n, k], scales fp32 [row blocks, column blocks])."""
    n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    t = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    scale = t.abs().amax(dim=(1, 3)).clamp(min=SMALLEST) / LARGEST
    q = (t / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous()
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def noise(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op, m, k = case["op"], case["m"], case["k"]
    s = dict(case)
    if own:
        s["ops"] = _ops()
    if op in ("norm", "rows", "swiglu"):
        dtype = TYPES[case["dtype"]]
        width = 2 * k if op == "swiglu" else k
        # the magnitudes of a residual stream and of projections: a few channels far above the rest
        channel = torch.exp(0.5 * noise(1, width))
        s["x"] = (noise(m, width) * channel).to(dtype)
        if op == "norm":
            s["weight"] = (1.0 + 0.2 * noise(k)).to(dtype)
            s["residual"] = (noise(m, k) * 2.0).to(dtype) if case["residual"] else None
        if own:
            s["q"], s["scales"] = s["ops"].fp8_rows(m, k, s["x"].device)
            if op == "norm" and case["residual"]:
                s["sum"] = torch.empty(m, k, dtype=dtype, device="cuda")
        return s
    n = case["n"]
    # rows as one of the operators above leaves them, zero beyond column k; weights of a projection, scaled per block
    q, s["scales"] = _quantise(noise(m, k) * torch.exp(0.5 * noise(1, k)))
    s["q"] = torch.nn.functional.pad(q.view(torch.uint8), (0, _blocks(k) * BLOCK - k)).view(torch.float8_e4m3fn)
    if case["behind"] == "swiglu":       # gate rows, then up rows, each matrix with blocks of its own
        halves = [_quantise_weight(noise(n // 2, k) * k ** -0.5) for _ in range(2)]
        s["wq"], s["ws"] = torch.cat([h[0].view(torch.uint8) for h in halves]).view(torch.float8_e4m3fn), torch.cat([h[1] for h in halves])
    else:
        s["wq"], s["ws"] = _quantise_weight(noise(n, k) * k ** -0.5)
    dtype = TYPES[case["out"]]
    s["residual"] = noise(m, n).to(dtype) if case["behind"] == "residual" else None
    if own:
        glu = case["behind"] == "swiglu"
        s["w"] = s["ops"].pack_weight_fp8(s["wq"], scales=s["ws"], glu=glu)
        s["y"] = torch.empty(m, n // 2 if glu else n, dtype=dtype, device="cuda")
    return s


def run(s):
    if own:
        return _run_own(s)
    op, k = s["op"], s["k"]
    if op == "linear":
        x = s["q"].float() * s["scales"].repeat_interleave(BLOCK, dim=1)
        x = x[:, :k]
        n, dtype = s["n"], TYPES[s["out"]]
        if s["behind"] == "swiglu":
            f, nb = n // 2, _blocks(n // 2)
            rows = torch.cat([s["ws"][:nb].repeat_interleave(BLOCK, dim=0)[:f], s["ws"][nb:].repeat_interleave(BLOCK, dim=0)[:f]])
        else:
            rows = s["ws"].repeat_interleave(BLOCK, dim=0)[:n]
        w = s["wq"].float() * rows.repeat_interleave(BLOCK, dim=1)[:, :k]
        y = x @ w.t()
        if s["behind"] == "swiglu":
            gate, up = y[:, :n // 2], y[:, n // 2:]
            y = gate / (1.0 + torch.exp(-gate)) * up
        elif s["behind"] == "residual":
            y = y + s["residual"].float()
        return y.to(dtype)
    x = s["x"].float()
    if op == "swiglu":
        gate, up = x[:, :k], x[:, k:]
        q, scale = _quantise(gate / (1.0 + torch.exp(-gate)) * up)
        return {"q": q, "scales": scale}
    if op == "rows":
        q, scale = _quantise(x)
        return {"q": q, "scales": scale}
    out = {}
    if s["residual"] is not None:
        out["sum"] = (x + s["residual"].float()).to(s["x"].dtype)
        x = out["sum"].float()
    y = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * s["weight"].float()
    out["q"], out["scales"] = _quantise(y)
    return out


def _run_own(s):
    ops = s["ops"]
    op, k = s["op"], s["k"]
    if op == "linear":
        return ops.linear_fp8(s["q"], s["scales"], s["w"], s["y"], residual=s["residual"], swiglu=s["behind"] == "swiglu")
    if op == "norm":
        out = {"q": s["q"][:, :k], "scales": s["scales"]}
        if s["residual"] is not None:
            out["sum"] = s["sum"]
        ops.rmsnorm_fp8(s["x"], s["weight"], EPS, s["q"], s["scales"], residual=s["residual"], sum_out=out.get("sum"))
        return out
    if op == "swiglu":
        ops.swiglu_fp8(s["x"], s["q"], s["scales"])
    else:
        ops.quantize_rows_fp8(s["x"], s["q"], s["scales"])
    return {"q": s["q"][:, :k], "scales": s["scales"]}


def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    if op == "linear":
        n, size = case["n"], 4 if case["out"] == "fp32" else 2
        cols = n // 2 if case["behind"] == "swiglu" else n
        moved = m * k + 4 * m * _blocks(k) + n * k + 4 * _blocks(n) * _blocks(k) + size * m * cols
        if case["behind"] == "residual":
            moved += size * m * n
        return {"bytes": moved, "flops": 2 * m * n * k}
    size = 4 if case["dtype"] == "fp32" else 2
    written = m * k + 4 * m * _blocks(k)
    if op == "swiglu":
        return {"bytes": 2 * size * m * k + written, "flops": 8 * m * k}
    if op == "rows":
        return {"bytes": size * m * k + written, "flops": 3 * m * k}
    return {"bytes": size * (m * k * (3 if case["residual"] else 1) + k) + written, "flops": 7 * m * k}


def _e4m3(v):
    """fp64 -> the nearest e4m3 number, ties to even, as fp64 (|v| at most 448 up to rounding)."""
    _, e = torch.frexp(v)                                   # |v| = f 2^e, 1/2 <= f < 1
    step = ((e.long().clamp(min=-5) - 4 + 1023) << 52).view(torch.float64)   # an exact power of two
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    op, m, k = case["op"], case["m"], case["k"]
    kb = _blocks(k)
    if op == "linear":
        n, f = case["n"], case["n"] // 2
        x = torch.nn.functional.pad(s["q"].double()[:, :k], (0, kb * BLOCK - k)).view(m, kb, BLOCK) * s["scales"].double()[:, :, None]
        row = torch.arange(n, device="cuda")
        if case["behind"] == "swiglu":
            block = torch.where(row < f, row // BLOCK, _blocks(f) + (row - f) // BLOCK)
        else:
            block = row // BLOCK
        w = torch.nn.functional.pad(s["wq"].double(), (0, kb * BLOCK - k)).view(n, kb, BLOCK) * s["ws"].double()[block][:, :, None]
        y = torch.mm(x.view(m, -1), w.view(n, -1).t().contiguous())
        if case["behind"] == "swiglu":
            y = y[:, :f] * torch.sigmoid(y[:, :f]) * y[:, f:]
        elif case["behind"] == "residual":
            y += s["residual"].double()
        return y
    x, out = s["x"].double(), {}
    if op == "swiglu":
        y = x[:, :k] * torch.sigmoid(x[:, :k]) * x[:, k:]
    elif op == "rows":
        y = x
    else:
        if s["residual"] is not None:
            x = x + s["residual"].double()
            out["sum"] = x
            x = x.to(s["x"].dtype).double()                 # the norm is that of the sum as it is stored
        y = x / torch.sqrt((x * x).sum(dim=1, keepdim=True) / k + EPS) * s["weight"].double()
    y = torch.nn.functional.pad(y, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    top = y.abs().max(dim=2).values
    scale = torch.where(top > 0, top.clamp(min=SMALLEST) / LARGEST, 1.0)
    out["q"] = _e4m3(y / scale[:, :, None]).view(m, -1)[:, :k]
    out["scales"] = scale
    return out
