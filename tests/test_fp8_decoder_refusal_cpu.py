"""The decoder on a model that `convert_fp8` has converted (host side, packing stubbed)."""
import types

import pytest

from hashattention import fp8
from hashattention.decoder import LlamaShapedDecoder
from tests.test_fp8_convert_cpu import small_model, stub  # noqa: F401


def test_decoder_of_a_converted_model_is_refused_by_name(stub):  # noqa: F811
    """The decoder copies 16-bit weights, which `convert_fp8` has freed."""
    model = fp8.convert_fp8(small_model(1))
    usa = types.SimpleNamespace(rehash_every_step=False, num_layers=3, int_dim=128, lth_final_dim=32, num_heads=1)
    for k, v in dict(init_budget=8, heavy_budget=1.0, recent_budget=8).items():
        setattr(model.config, k, v)
    with pytest.raises(ValueError, match="convert_fp8"):
        LlamaShapedDecoder.from_hf(model, [usa], batch=1, cache_len=16, device="cpu", fp8_projections=True)
    with pytest.raises(ValueError, match="convert_fp8"):
        LlamaShapedDecoder.load_hf_llama(types.SimpleNamespace(layers=[{}]), model)
