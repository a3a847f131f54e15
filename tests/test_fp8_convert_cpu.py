"""Which layers `convert_fp8` takes (host side: packing needs a GPU and is stubbed, nothing is launched)."""
import warnings

import pytest
import torch
from torch import nn
from torch.nn.utils import parametrize
from transformers import LlamaConfig, LlamaForCausalLM

from hashattention import _ops, fp8

NAMES = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")


def fake_weight(n, k, fill=0):
    count = -(-n // 16) * -(-k // 128)
    return _ops.Fp8Weight(torch.full((2048 * count,), fill, dtype=torch.uint8), torch.full((2 * count,), float(fill)), n, k, False)


@pytest.fixture
def stub(monkeypatch):
    monkeypatch.setattr(_ops, "pack_weight_fp8", lambda w, scales=None, glu=False: fake_weight(*w.shape))


def small_model(layers=2):
    torch.manual_seed(0)
    return LlamaForCausalLM(LlamaConfig(hidden_size=64, intermediate_size=96, num_hidden_layers=layers, num_attention_heads=2,
                                        num_key_value_heads=1, head_dim=32, vocab_size=32))


def kinds(layer):
    return [type(layer.get_submodule(n)) for n in NAMES]


class LowRank(nn.Linear):
    """nn.Linear with a term of its own, as an adapter subclasses it."""

    def __init__(self, old):
        super().__init__(old.in_features, old.out_features, bias=False)
        self.a, self.b = nn.Parameter(torch.ones(2, old.in_features)), nn.Parameter(torch.ones(old.out_features, 2))

    def forward(self, x):
        return super().forward(x) + x @ self.a.t() @ self.b.t()


def _subclass(layer):
    layer.self_attn.q_proj = LowRank(layer.self_attn.q_proj)


def _hook(layer):
    layer.mlp.gate_proj.register_forward_hook(lambda m, a, out: out * 2)


def _pre_hook(layer):
    layer.mlp.down_proj.register_forward_pre_hook(lambda m, a: (a[0] * 2,))


def _own_forward(layer):
    lin = layer.self_attn.o_proj
    lin.forward = lambda x: nn.functional.linear(x, lin.weight) * 2


def _parametrized(layer):
    parametrize.register_parametrization(layer.mlp.up_proj, "weight", nn.Tanh())


@pytest.mark.parametrize("change", [_subclass, _hook, _pre_hook, _own_forward, _parametrized])
def test_layers_with_a_say_of_their_own_are_left_as_they_are(change, stub):
    """A projection that is a subclass of nn.Linear, has a hook, a forward or a parametrization of its own computes something else than
    x W^T: its layer is not converted, and the caller hears of it."""
    model = small_model()
    change(model.model.layers[0])
    before = kinds(model.model.layers[0])
    modules = [model.model.layers[0].get_submodule(n) for n in NAMES]
    with pytest.warns(UserWarning, match="1 decoder layer"):
        fp8.convert_fp8(model)
    assert kinds(model.model.layers[0]) == before
    assert all(model.model.layers[0].get_submodule(n) is m for n, m in zip(NAMES, modules))
    assert kinds(model.model.layers[1]) == [fp8.Fp8Linear] * 7


def test_a_model_of_such_layers_only_is_refused(stub):
    model = small_model(1)
    _subclass(model.model.layers[0])
    with pytest.raises(ValueError):
        fp8.convert_fp8(model)
    assert type(model.model.layers[0].mlp.up_proj) is nn.Linear


def test_plain_layers_are_taken_in_silence(stub):
    model = small_model()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        fp8.convert_fp8(model)
    assert all(kinds(layer) == [fp8.Fp8Linear] * 7 for layer in model.model.layers)


def test_a_prefill_module_with_a_say_of_its_own(stub):
    """The attention module that a converted one prefills through counts too."""
    model = small_model()
    attn = model.model.layers[0].self_attn
    twin = type(attn)(model.config, 0)
    twin.v_proj = LowRank(twin.v_proj)
    attn.flash_forward = twin.forward
    with pytest.warns(UserWarning):
        fp8.convert_fp8(model)
    assert type(attn.v_proj) is nn.Linear and type(twin.v_proj) is LowRank


def test_modules_that_accelerate_placed_are_taken(stub):
    """accelerate's placement hooks (a model spread over devices) move inputs and compute nothing."""
    hooks = pytest.importorskip("accelerate.hooks")
    model = small_model(1)
    hooks.add_hook_to_module(model.model.layers[0].mlp.gate_proj, hooks.AlignDevicesHook(execution_device="cpu"))
    fp8.convert_fp8(model)
    assert kinds(model.model.layers[0]) == [fp8.Fp8Linear] * 7
