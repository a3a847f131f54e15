"""Stacked 8-bit weights (`fp8.stacked_weight`) in every kernel of the product: parts whose rows are no whole blocks of 128, neighbouring
blocks whose magnitudes differ by powers of two."""
import pytest
import torch
from torch import nn
from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

from hashattention import _ops, fp8
from hashattention import hashattention_llama as hl
from tests import fp8_util as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def noise(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV, dtype=torch.float64)


def make_parts(rows, k, seed=0):
    """[(e4m3 weight, scales)], every part with blocks of its own, neighbours eight and more times apart."""
    parts = []
    for i, n in enumerate(rows):
        wq, ws = ref.quantise_weight(noise(n, k, seed=seed + i) * k ** -0.5)
        nb, kb = ws.shape
        power = (torch.arange(nb, device=DEV)[:, None] + torch.arange(kb, device=DEV)[None, :] + i) % 2 * 3 + 4 * i
        parts.append((wq, ws * torch.exp2(power.float())))
    return parts


# rows of x, rows of the parts, inputs: x in registers, the stream of few rows, K cut (17 and 40 rows of 4224), tiles of 128 x 128 over
# the whole of K, tiles of 256 x 256; parts of whole blocks next to others
SIZES = [(5, (1040, 1040), 512), (16, (144, 272, 96), 4224), (24, (144, 80), 700), (100, (144, 272, 96), 4096),
         (17, (1040, 1040), 4224), (40, (144, 272, 96), 4224), (40, (64, 192, 130), 4224),
         (1000, (1040, 1040), 700), (1000, (1088, 2048), 1300), (2100, (3040, 3040), 1000), (2100, (2944, 3200), 1000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,rows,k", SIZES)
def test_stacked_parts_in_every_kernel(m, rows, k, dtype):
    parts = make_parts(rows, k)
    owner = nn.Module()
    mods = [fp8.Fp8Linear(_ops.pack_weight_fp8(wq, scales=ws)) for wq, ws in parts]
    w = fp8.stacked_weight(owner, "_stack", mods)
    q, s = ref.quantise(noise(m, k, seed=9))
    r = noise(m, sum(rows), seed=10).to(dtype)
    wide = torch.full((m + 1, sum(rows) + 6), 9.0, dtype=dtype, device=DEV)
    out = wide[:m, 3:-3]
    assert _ops.linear_fp8(q, s, w, out, residual=r) is out
    at = 0
    for wq, ws in parts:
        n = wq.shape[0]
        ref.assert_linear(out[:, at:at + n], *ref.linear(q, s, wq, ws, k, residual=r[:, at:at + n],
                                                         eight_bit_sums=m > 16 and dtype != torch.float32))
        at += n
    assert (wide[:, :3] == 9.0).all() and (wide[:, -3:] == 9.0).all() and (wide[m] == 9.0).all()
    need = _ops.linear_fp8_workspace_bytes(m, w)
    mem = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device=DEV)
    again = _ops.linear_fp8(q, s, w, torch.empty_like(out), residual=r, ws=mem[:need] if need else None)
    assert torch.equal(again, out) and (mem[need:] == 0x5a).all()


@pytest.mark.parametrize("batch", [3, 20])
def test_layer_whose_gate_and_up_are_no_whole_blocks(batch):
    """A single-token step of a layer with 4224 hidden elements (K is cut at 20 sequences) and 1040 feed-forward ones, up's blocks eight
    times apart: the layer's launches against its modules called one by one.  Rows rounded to 8 bits on either way differ by at most
    2^-3 of their norm."""
    cfg = LlamaConfig(hidden_size=4224, intermediate_size=1040, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                      vocab_size=64, max_position_embeddings=1024)
    for k, v in dict(lth_init_dim=128, lth_final_dim=32, lth_thold=0, lth_num_layers=3, init_budget=8, heavy_budget=1.0, recent_budget=8,
                     usa_retrieve_depth=6, usa_eval_mode="simple").items():
        setattr(cfg, k, v)
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).bfloat16().to(DEV)
    mlp = model.model.layers[0].mlp
    with torch.no_grad():
        mlp.gate_proj.weight.mul_(4.0)
        mlp.up_proj.weight.mul_(torch.exp2(torch.arange(1040, device=DEV) // 128 % 2 * 3.0 + 5)[:, None])
    model = fp8.convert_fp8(hl.convert_usa(model, cfg, hl.load_usa(cfg, None), collect_stats=False, train_usa=False))
    ids = torch.randint(1, 64, (batch, 21), generator=torch.Generator().manual_seed(1)).to(DEV)
    outs = []
    for fast in (False, True):
        model.model.layers[0].self_attn.fast_layer = fast
        hl.reset_usa(model)
        cache = DynamicCache()
        with torch.no_grad():
            model(ids[:, :20], past_key_values=cache, use_cache=True)
            outs.append(model(ids[:, 20:], past_key_values=cache, use_cache=True).logits[:, 0].double())
    assert "_fast_fp8" in model.model.layers[0].self_attn.__dict__
    assert float((outs[1] - outs[0]).norm() / outs[0].norm()) < 2.0 ** -3
