"""The staged kernels over many blocks of K, where every buffer is refilled many times, with scales of neighbouring blocks and rows
several powers of two apart: a scale or a buffer of another block is off by the order of the result."""
import pytest
import torch

from hashattention import _ops
from tests import fp8_util as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def noise(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV, dtype=torch.float64)


def apart(*shape):
    """Powers of two, 1 to 16, that change with every row and every column."""
    a, b = (torch.arange(n, device=DEV) for n in shape)
    return torch.exp2((a[:, None] * 3 + b[None, :] * 2) % 5.0)


def make(m, n, k, glu):
    q, s = ref.quantise(noise(m, k))
    parts = [ref.quantise_weight(noise(n // 2 if glu else n, k, seed=1 + i) * k ** -0.5) for i in range(2 if glu else 1)]
    wq = torch.cat([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
    ws = torch.cat([p[1] for p in parts])
    return q, s * apart(*s.shape).float(), wq, ws * apart(*ws.shape).float()


def values(q, s, wq, ws, k, glu):
    x = q[:, :k].double() * ref.spread(s, k)
    n = wq.shape[0]
    if glu:
        f, nb = n // 2, ref.blocks(n // 2)
        return x, [wq[:f].double() * ref.weight_spread(ws[:nb], f, k), wq[f:].double() * ref.weight_spread(ws[nb:], f, k)]
    return x, [wq.double() * ref.weight_spread(ws, n, k)]


# 256 x 256 tiles (16-bit results, 200 and more of them), 128 x 128 tiles, K cut over workgroups
@pytest.mark.parametrize("m,n,k", [(2100, 6200, 4096), (1000, 2000, 4200), (300, 515, 8192)])
@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_error_over_many_blocks(m, n, k, glu, dtype):
    """2-norm of the error against 64 bits.  The 8-bit instructions are off by 1.5e-5 of a block's sum on normally distributed numbers,
    whatever the block's scales: with v the root of the sum of the squared products, an output is off by 1.5e-5 v, taken twice here
    (fp32 sums: 1e-6 v).  SwiGLU: |d silu| <= 1.1 |d gate|.  Then half a step of the output's type."""
    n += n % 2
    q, s, wq, ws = make(m, n, k, glu)
    x, w = values(q, s, wq, ws, k, glu)
    scale = 2.0 ** -8 if glu and dtype == torch.float16 else 1.0          # gate x up stays below fp16's largest number
    s, x = s * scale, x * scale
    out = _ops.linear_fp8(q, s, _ops.pack_weight_fp8(wq, scales=ws, glu=glu), torch.empty(m, n // 2 if glu else n, dtype=dtype, device=DEV),
                          swiglu=glu)
    off = 1e-6 if dtype == torch.float32 else 3e-5
    y = [torch.mm(x, p.t().contiguous()) for p in w]
    d = [off * torch.mm(x.square(), p.square().t().contiguous()).sqrt() for p in w]
    if glu:
        silu = y[0] * torch.sigmoid(y[0])
        want, most = silu * y[1], (1.1 * d[0] * y[1]).square() + (silu * d[1]).square()
    else:
        want, most = y[0], d[0].square()
    assert torch.isfinite(out).all()
    assert float((out.double() - want).norm()) <= float(most.sum().sqrt() + torch.finfo(dtype).eps / 2 * want.norm())
