"""Weights stacked under `torch.inference_mode` (a first step there) stay ordinary tensors."""
import torch
from torch import nn

from hashattention import fp8
from tests.test_fp8_convert_cpu import fake_weight


def test_stacked_under_inference_mode_and_loaded_afterwards():
    owner = nn.Module()
    owner.parts = nn.ModuleList([fp8.Fp8Linear(fake_weight(n, 128, 1)) for n in (128, 32)])
    with torch.inference_mode():
        w = fp8.stacked_weight(owner, "_stack", list(owner.parts))
    state = {k: torch.zeros_like(v) for k, v in owner.state_dict().items()}
    owner.load_state_dict(state)
    assert not w.tiles.any() and not w.scales.any()
    assert fp8.stacked_weight(owner, "_stack", list(owner.parts)) is w


def test_parts_made_under_inference_mode():
    owner = nn.Module()
    with torch.inference_mode():
        owner.parts = nn.ModuleList([fp8.Fp8Linear(fake_weight(n, 128, 1)) for n in (128, 32)])
    w = fp8.stacked_weight(owner, "_stack", list(owner.parts))
    assert w.tiles.numel() == 2048 * 10 and owner.parts[1].tiles.data_ptr() == w.tiles.data_ptr() + 8 * 2048
