"""`Fp8Linear` with a bias: the sum is rounded once, as `nn.Linear` rounds it."""
import pytest
import torch

from hashattention import _ops, fp8
from tests import fp8_util as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(m, n, k, bias_dtype):
    """Whole numbers in x and weights (every sum exact in fp32 and in the 8-bit instructions' 13 bits), one place of each block held by
    448 in x and 0 in the weights (scale 1), a bias in steps of 1/8."""
    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    x = torch.randint(-3, 4, (m, k), generator=g, device=DEV).float()
    w = torch.randint(-2, 3, (n, k), generator=g, device=DEV).float()
    x[:, ::128], w[:, ::128] = 448.0, 0.0
    bias = (torch.randint(-200, 201, (n,), generator=g, device=DEV).float() / 8).to(bias_dtype)
    packed = _ops.pack_weight_fp8(w.to(torch.float8_e4m3fn), scales=torch.ones(ref.blocks(n), ref.blocks(k), device=DEV))
    return x, w, bias, fp8.Fp8Linear(packed, bias)


SIZES = [(1, 129, 512), (3, 129, 4200), (3, 256, 4000), (40, 130, 1000), (40, 257, 4300), (300, 515, 8192), (700, 3000, 640)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype,bias_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32),
                                              (torch.bfloat16, torch.float32), (torch.float32, torch.float16), (torch.float16, torch.bfloat16)])
def test_bias_is_added_before_the_one_rounding(m, n, k, dtype, bias_dtype):
    x, w, bias, mod = make(m, n, k, bias_dtype)
    with torch.no_grad():
        got = mod(x.to(dtype))
    want = (x.double() @ w.double().t() + bias.double()).to(dtype)
    assert got.dtype == dtype and torch.equal(got, want)


def test_one_row_added_to_every_row():
    """The residual's rows may be one and the same."""
    x, w, bias, mod = make(37, 200, 900, torch.bfloat16)
    q, s = _ops.fp8_rows(37, 900, DEV)
    _ops.quantize_rows_fp8(x, q, s)
    out = torch.empty(37, 200, dtype=torch.bfloat16, device=DEV)
    _ops.linear_fp8(q, s, mod.packed, out, residual=bias.expand(37, 200))
    full = _ops.linear_fp8(q, s, mod.packed, torch.empty_like(out), residual=bias.expand(37, 200).contiguous())
    assert torch.equal(out, full)
