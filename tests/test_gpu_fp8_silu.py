"""SwiGLU to 8 bits of gates so far out that the exponential nears the largest fp32 number (exp(88.72))."""
import pytest
import torch

from hashattention import _ops
from tests import fp8_util as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("low,high", [(-88.7, -88.0), (-88.0, -87.3), (-87.5, -87.5), (-88.5, -88.5), (-87.3, -80.0), (-80.0, -40.0), (-50.0, -20.0)])
def test_far_gates_keep_their_precision(low, high):
    """up as large as the activations are small, so that every value of the block counts.  Exponential to 2 ulp, reciprocal to 1 ulp,
    three products: below 2^-20."""
    gate = torch.linspace(low, high, 128, device=DEV)
    up = (torch.linspace(0.5, 1.0, 128, device=DEV).double() / torch.sigmoid(gate.double()) / gate.double()).clamp(-3e38, 3e38).float()
    x = torch.cat([gate, up]).view(1, 256)
    q, s = _ops.fp8_rows(1, 128, DEV)
    _ops.swiglu_fp8(x, q, s)
    g, u = gate.double(), up.double()
    ref.assert_rows(q, s, (g * torch.sigmoid(g) * u).view(1, 128), 2.0 ** -20)


def test_far_gates_behind_the_product():
    """The same function behind a projection: gates of -87.5 and -88.5, up of 2^118, results around -0.2, in fp32."""
    q = torch.zeros(2, 128, device=DEV)
    q[:, 0] = 1.0
    w = torch.zeros(16, 128, device=DEV)
    w[:8, 0] = w[8:, 0] = 1.0
    for gate in (-87.5, -88.5):
        pack = _ops.pack_weight_fp8(w.to(torch.float8_e4m3fn), scales=torch.tensor([[gate], [2.0 ** 118]], device=DEV), glu=True)
        out = _ops.linear_fp8(q.to(torch.float8_e4m3fn), torch.ones(2, 1, device=DEV), pack, torch.empty(2, 8, device=DEV), swiglu=True)
        g = torch.tensor(gate, dtype=torch.float64)
        want = float(g * torch.sigmoid(g)) * 2.0 ** 118
        assert ((out.double() - want).abs() <= abs(want) * 2.0 ** -20).all()
