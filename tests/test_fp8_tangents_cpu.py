"""`Fp8Linear` is for inference: forward-mode derivatives are refused (host side)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from hashattention import fp8
from tests.test_fp8_convert_cpu import fake_weight


def test_tangents_are_refused():
    """Forward-mode derivatives would be lost without a word."""
    mod = fp8.Fp8Linear(fake_weight(16, 128))
    x = torch.zeros(2, 128)
    with torch.no_grad(), fwd.dual_level():
        with pytest.raises(RuntimeError, match="inference"):
            mod(fwd.make_dual(x, torch.ones_like(x)))
        with pytest.raises(ValueError, match="GPU"):         # no tangent: as far as the device check
            mod(x)


def test_tangents_of_torch_func_are_refused():
    mod = fp8.Fp8Linear(fake_weight(16, 128))
    x = torch.zeros(2, 128)
    with pytest.raises(RuntimeError, match="inference"):
        torch.func.jvp(mod, (x,), (torch.ones_like(x),))
