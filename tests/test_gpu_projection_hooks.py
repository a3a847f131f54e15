"""Forward hooks on an attention module's projections: a step that calls none of them must not be taken past them."""
import pytest
import torch
from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

from hashattention import fp8
from hashattention import hashattention_llama as hl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("name", ["q_proj", "k_proj", "v_proj", "o_proj"])
def test_hooks_on_projections_fire_in_single_token_steps(name, eight_bit):
    cfg = LlamaConfig(hidden_size=256, intermediate_size=384, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, head_dim=128,
                      vocab_size=64, max_position_embeddings=1024)
    for k, v in dict(lth_init_dim=128, lth_final_dim=32, lth_thold=0, lth_num_layers=3, init_budget=8, heavy_budget=1.0, recent_budget=8,
                     usa_retrieve_depth=6, usa_eval_mode="simple").items():
        setattr(cfg, k, v)
    torch.manual_seed(0)
    model = hl.convert_usa(LlamaForCausalLM(cfg).bfloat16().to(DEV), cfg, hl.load_usa(cfg, None), collect_stats=False, train_usa=False)
    if eight_bit:
        fp8.convert_fp8(model)
    ids = torch.randint(1, 64, (2, 12), generator=torch.Generator().manual_seed(1)).to(DEV)
    cache, seen = DynamicCache(), []
    with torch.no_grad():
        model(ids[:, :10], past_key_values=cache, use_cache=True)
        hook = getattr(model.model.layers[1].self_attn, name).register_forward_hook(lambda m, a, out: seen.append(out.shape[1]))
        model(ids[:, 10:11], past_key_values=cache, use_cache=True)
        assert seen == [1]
        hook.remove()
        pre = getattr(model.model.layers[0].self_attn, name).register_forward_pre_hook(lambda m, a: seen.append("pre"))
        model(ids[:, 11:12], past_key_values=cache, use_cache=True)
        assert seen == [1, "pre"]
        pre.remove()
