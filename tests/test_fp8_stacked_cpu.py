"""What a stacked 8-bit weight holds on to (host side, packing stubbed)."""
import copy
import gc
import weakref

import pytest
import torch
from torch import nn

from hashattention import _ops, fp8
from tests.test_fp8_convert_cpu import fake_weight


def stacked():
    owner = nn.Module()
    owner.parts = nn.ModuleList([fp8.Fp8Linear(fake_weight(n, 128, fill)) for n, fill in ((256, 1), (32, 2))])
    w = fp8.stacked_weight(owner, "_stack", list(owner.parts))
    assert fp8.stacked_weight(owner, "_stack", list(owner.parts)) is w
    return owner, weakref.ref(w.tiles), weakref.ref(w.scales)


def replace_state(owner):
    new = fp8.Fp8Linear(fake_weight(256, 128, 5)), fp8.Fp8Linear(fake_weight(32, 128, 6))
    owner.load_state_dict({f"parts.{i}.{k}": v for i, m in enumerate(new) for k, v in m.state_dict().items()}, assign=True)


def set_buffers(owner):
    for m in owner.parts:
        m.tiles, m.tile_scales = m.tiles.clone(), m.tile_scales.clone()


@pytest.mark.parametrize("move", [lambda o: o.to("meta"), replace_state, set_buffers], ids=["device", "state dict", "buffers"])
def test_nothing_is_held_once_the_parts_are_elsewhere(move):
    owner, tiles, scales = stacked()
    move(owner)
    gc.collect()
    assert tiles() is None and scales() is None


def test_casts_keep_the_stacked_weight():
    owner, tiles, _ = stacked()
    owner.half()
    owner.to(torch.bfloat16)
    assert fp8.stacked_weight(owner, "_stack", list(owner.parts)).tiles is tiles()
    state = {k: v.clone() for k, v in owner.state_dict().items()}
    owner.load_state_dict(state)
    assert fp8.stacked_weight(owner, "_stack", list(owner.parts)).tiles is tiles()


def test_a_copy_and_its_original_go_their_own_ways():
    owner, tiles, _ = stacked()
    twin = copy.deepcopy(owner)
    w = fp8.stacked_weight(twin, "_stack", list(twin.parts))
    assert w.tiles is not tiles() and torch.equal(w.tiles, tiles())
    twin.to("meta")
    assert fp8.stacked_weight(owner, "_stack", list(owner.parts)).tiles is tiles()
