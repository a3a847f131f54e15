"""Sizes that pass 32 bits, at the bindings of the 8-bit operators (tensors without memory, launches caught)."""
import pytest
import torch

from hashattention import _ops

BIG = 2 ** 32 + 128
META = dict(device="meta")


@pytest.fixture
def caught(monkeypatch):
    calls = []
    monkeypatch.setattr(_ops, "_same_device", lambda *t: 0)
    monkeypatch.setattr(_ops, "_launch_on", lambda dev, fn, where, args: calls.append((where, args)))
    return calls


def rows(m, k):
    return _ops.fp8_rows(m, k, "meta")


def test_sizes_beyond_32_bits_are_refused(caught):
    """They would reach the C entry as their lowest 32 bits: 128 elements instead of 2^32 + 128."""
    bf16, e4m3 = torch.bfloat16, torch.float8_e4m3fn
    small = _ops.Fp8Weight(torch.empty(2048, dtype=torch.uint8, **META), torch.empty(2, **META), 16, 128, False)
    bad = [
        lambda: _ops.quantize_rows_fp8(torch.empty(1, BIG, dtype=bf16, **META), *rows(1, BIG)),
        lambda: _ops.quantize_rows_fp8(torch.empty(BIG, 1, dtype=bf16, **META), *rows(BIG, 1)),
        lambda: _ops.swiglu_fp8(torch.empty(1, 2 * BIG, dtype=bf16, **META), *rows(1, BIG)),
        lambda: _ops.rmsnorm_fp8(torch.empty(1, BIG, dtype=bf16, **META), torch.empty(BIG, dtype=bf16, **META), 1e-5, *rows(1, BIG)),
        lambda: _ops.pack_weight_fp8(torch.empty(1, BIG, dtype=bf16, **META)),
        lambda: _ops.pack_weight_fp8(torch.empty(BIG, 1, dtype=bf16, **META)),
        lambda: _ops.pack_weight_fp8(torch.empty(1, BIG, dtype=e4m3, **META), scales=torch.empty(1, _ops.fp8_blocks(BIG), **META)),
        lambda: _ops.linear_fp8(*rows(BIG, 128), small, torch.empty(BIG, 16, dtype=bf16, **META)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken: {caught[-1]}")
    assert not caught


def test_sizes_within_32_bits_pass(caught):
    _ops.quantize_rows_fp8(torch.empty(1, 2 ** 31 - 129, dtype=torch.bfloat16, **META), *rows(1, 2 ** 31 - 129))
    _ops.quantize_rows_fp8(torch.empty(2 ** 31 - 1, 1, dtype=torch.bfloat16, **META), *rows(2 ** 31 - 1, 1))
    assert [c[0] for c in caught] == ["ha_quantize_rows_fp8"] * 2
