"""8-bit projections in the framework's models: `Fp8Linear`, `convert_fp8` on transformers models (with and without `convert_usa`) and the
decoder with `fp8_projections`."""
import pytest
import torch
from torch import nn
from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

from hashattention import _ops, fp8
from hashattention import hashattention_llama as hl
from hashattention.decoder import LlamaShapedDecoder
from tests import fp8_util as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _config(**kw):
    shape = dict(hidden_size=512, intermediate_size=1040, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                 vocab_size=512, max_position_embeddings=4096, rope_theta=500000.0, rms_norm_eps=1e-5)
    cfg = LlamaConfig(**{**shape, **kw})
    # every cached token is selected: what a rounding changes in a code cannot change what is attended to
    for k, v in dict(lth_init_dim=128, lth_final_dim=32, lth_thold=0, lth_num_layers=3, init_budget=8, heavy_budget=1.0, recent_budget=8,
                     usa_retrieve_depth=6, usa_eval_mode="simple").items():
        setattr(cfg, k, v)
    return cfg


def _converted(cfg, seed=0):
    torch.manual_seed(seed)
    model = LlamaForCausalLM(cfg).bfloat16().to(DEV)
    usa = hl.load_usa(cfg, None)
    return fp8.convert_fp8(hl.convert_usa(model, cfg, usa, collect_stats=False, train_usa=False)), usa


def _tokens(cfg, b, n, seed=1):
    return torch.randint(1, cfg.vocab_size, (b, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


# Two ways through the same 8-bit projections differ where one rounds to bf16 before the 8-bit rounding and the other does not.  Rounding a
# row to e4m3 moves it by at most 2^-4 of its norm (half a step of 3 mantissa bits), so two roundings of nearly equal rows
# differ by at most 2^-3 of it; a misplaced operand, residual or norm is off by the order of 1.
SAME = 2.0 ** -3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,n", [((1, 1, 512), 300), ((2, 3, 500), 64), ((40, 384), 129), ((300, 256), 257)])
def test_fp8_linear_against_the_linear_it_replaces(dtype, shape, n):
    """Both factors are off by at most half an e4m3 step (2^-4 relative, 2^-10 of the block's scale below the smallest normal
    number): every output lies within what those errors can add up to."""
    torch.manual_seed(3)
    k = shape[-1]
    lin = nn.Linear(k, n, bias=n % 2 == 1).to(DEV).to(dtype)
    x = torch.randn(*shape, device=DEV).to(dtype)
    mod = fp8.Fp8Linear.from_linear(lin)
    with torch.no_grad():
        got = mod(x)
        assert got.shape == (*shape[:-1], n) and got.dtype == dtype
        xd, wd = x.reshape(-1, k).double(), lin.weight.double()
        want = xd @ wd.t()
        ex = xd.abs() * 2.0 ** -4 + ref.spread(ref.block_scales(xd), k) * 2.0 ** -10
        _, ws = ref.quantise_weight(wd)
        ew = wd.abs() * 2.0 ** -4 + ref.weight_spread(ws, n, k) * 2.0 ** -10
        bound = (xd.abs() + ex) @ (wd.abs() + ew).t() - xd.abs() @ wd.abs().t()
        if lin.bias is not None:
            want = want + lin.bias.double()
        bound = bound * (1 + 2.0 ** -9) + (want.abs() + bound) * 2 * torch.finfo(dtype).eps     # the sums, two roundings of the result
        assert ((got.reshape(-1, n).double() - want).abs() <= bound).all()
        wide = torch.zeros(*shape[:-1], k + 5, device=DEV, dtype=dtype)
        wide[..., 2:k + 2] = x
        assert torch.equal(mod(wide[..., 2:k + 2]), got)
        assert mod(x[:0]).shape == (0, *shape[1:-1], n)
    with pytest.raises(RuntimeError):
        mod(x.clone().requires_grad_())


def test_convert_fp8_replaces_the_projections_and_nothing_else():
    cfg = _config()
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).bfloat16().to(DEV)
    ids = _tokens(cfg, 2, 150)
    with torch.no_grad():
        before = model(ids).logits
        assert fp8.convert_fp8(model) is model
        after = model(ids).logits
    kinds = {n: type(m) for n, m in model.named_modules()}
    assert sum(t is fp8.Fp8Linear for t in kinds.values()) == 14
    assert [n for n, t in kinds.items() if t is nn.Linear] == ["lm_head"]
    # two layers of four projections in a row: each off by at most 2^-3 of its norm (rows and weights), added to the residual stream
    assert torch.isfinite(after).all() and _rel(after, before) < 0.5
    with pytest.raises(ValueError):
        fp8.convert_fp8(model)                       # nothing left to convert
    state = {k: v.clone() for k, v in model.state_dict().items()}
    model.load_state_dict(state)
    with torch.no_grad():
        assert torch.equal(model(ids).logits, after)


@pytest.mark.parametrize("batch", [1, 3, 9, 20, 40])
def test_single_token_steps_of_a_converted_layer(batch):
    """The launches of a single-token step against the same modules called one by one by the library's layer (hash attention through
    the general path), several steps in a row, and against the attention module alone on the few-launch path."""
    cfg = _config()
    model, _ = _converted(cfg)
    ids = _tokens(cfg, batch, 203)
    outs = {}
    for name, fast, layer_path in (("modules", False, False), ("attention", True, False), ("layer", True, True)):
        for layer in model.model.layers:
            layer.self_attn.fast_decode, layer.self_attn.fast_layer = fast, layer_path
        hl.reset_usa(model)
        cache = DynamicCache()
        with torch.no_grad():
            model(ids[:, :200], past_key_values=cache, use_cache=True)
            outs[name] = [model(ids[:, 200 + t:201 + t], past_key_values=cache, use_cache=True).logits[:, 0] for t in range(3)]
    assert "_qkv_fp8" in model.model.layers[0].self_attn.__dict__ and "_fast_fp8" in model.model.layers[1].self_attn.__dict__
    for t in range(3):
        assert _rel(outs["attention"][t], outs["modules"][t]) < SAME
        assert _rel(outs["layer"][t], outs["modules"][t]) < SAME


def test_stacked_weights_share_the_modules_memory_and_follow_them():
    cfg = _config()
    model, _ = _converted(cfg)
    attn = model.model.layers[0].self_attn
    parts = (attn.q_proj, attn.k_proj, attn.v_proj)
    w = fp8.stacked_weight(attn, "_qkv_fp8", parts)
    assert w.N == 1024 and w.tiles.data_ptr() == attn.q_proj.tiles.data_ptr()
    assert attn.v_proj.tiles.data_ptr() == w.tiles.data_ptr() + attn.q_proj.tiles.numel() + attn.k_proj.tiles.numel()
    assert fp8.stacked_weight(attn, "_qkv_fp8", parts).tiles is w.tiles
    x = torch.randn(5, 512, device=DEV).bfloat16()
    q, s = _ops.fp8_rows(5, 512, DEV)
    _ops.quantize_rows_fp8(x, q, s)
    with torch.no_grad():
        want = torch.cat([p(x) for p in parts], dim=1)
        assert torch.equal(_ops.linear_fp8(q, s, w, torch.empty(5, 1024, dtype=torch.bfloat16, device=DEV)), want)
        attn.k_proj.tiles = attn.k_proj.tiles.clone()            # as a move to another device and back leaves it
        w2 = fp8.stacked_weight(attn, "_qkv_fp8", parts)
        assert w2.tiles is not w.tiles
        assert torch.equal(_ops.linear_fp8(q, s, w2, torch.empty(5, 1024, dtype=torch.bfloat16, device=DEV)), want)
        assert torch.equal(torch.cat([p(x) for p in parts], dim=1), want)
    odd = [fp8.Fp8Linear.from_linear(nn.Linear(64, n, bias=False).to(DEV)) for n in (24, 16)]
    with pytest.raises(ValueError):
        fp8.stacked_weight(attn, "_odd", odd)


@pytest.mark.parametrize("batch", [2, 12, 40])
def test_decoder_with_8_bit_projections_against_the_converted_model(batch):
    """`LlamaShapedDecoder(fp8_projections=True)` and a model of the same 16-bit weights after `convert_fp8`: the same 8-bit weights, other
    launches (SwiGLU inside the gate/up product against behind it)."""
    cfg = _config()
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).bfloat16().to(DEV)
    usa = hl.load_usa(cfg, None)
    model = hl.convert_usa(model, cfg, usa, collect_stats=False, train_usa=False)
    dec = LlamaShapedDecoder.from_hf(model, usa, batch=batch, cache_len=256, device=DEV, fp8_projections=True)
    assert all(isinstance(p["w13_8"], _ops.Fp8Weight) and "w13" not in p for p in dec.layers)
    fp8.convert_fp8(model)
    ids = _tokens(cfg, batch, 203)
    cache = DynamicCache()
    with torch.no_grad():
        model(ids[:, :200], past_key_values=cache, use_cache=True)
        dec.load_cache([cache.layers[l].keys.clone() for l in range(2)], [cache.layers[l].values.clone() for l in range(2)])
        for t in range(3):
            want = model(ids[:, 200 + t:201 + t], past_key_values=cache, use_cache=True).logits[:, 0]
            got = dec.decode_step(ids[:, 200 + t])
            assert _rel(got, want) < SAME
    assert dec.seq_len == 203


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decoder_with_8_bit_projections_generates_from_one_graph(dtype):
    """The captured step replayed for successive tokens against eager steps: the same tokens and logits, from two decoders over the
    same weights, and a second allocation of the same decoder keeps its 8-bit weights."""
    kw = dict(n_layers=2, hidden=512, ffn=1040, n_heads=4, n_kv_heads=2, head_dim=128, vocab=512, n_code_heads=2, init_budget=8, recent_budget=8,
              heavy_budget=1.0, dtype=dtype, device=DEV, seed=3, fp8_projections=True)
    runs = []
    for use_graph in (True, False):
        dec = LlamaShapedDecoder(**kw)
        dec.allocate(3, 400)
        dec.fill_cache_synthetic(300)
        with torch.no_grad():
            toks = dec.generate(torch.tensor([5, 17, 99], device=DEV), 6, use_graph=use_graph)
            runs.append((toks, dec._gen_logits.clone()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    tiles = dec.layers[0]["wo_8"].tiles
    dec.allocate(5, 300)
    assert dec.layers[0]["wo_8"].tiles is tiles
    dec.fill_cache_synthetic(100)
    with torch.no_grad():
        assert torch.isfinite(dec.decode_step(torch.arange(5, device=DEV))).all()


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.float(), lambda m: m.to(torch.bfloat16), lambda m: m.cpu().to(DEV).half()])
def test_casting_a_model_keeps_the_packed_weights(cast):
    """The scales stay fp32, and the same rows give the same product."""
    torch.manual_seed(4)
    model = nn.Sequential(nn.Linear(300, 200), nn.Linear(200, 40)).to(DEV)
    model[0] = fp8.Fp8Linear.from_linear(model[0])
    tiles, scales = model[0].tiles.clone(), model[0].tile_scales.clone()
    x = torch.randn(3, 300, device=DEV).half().float()
    with torch.no_grad():
        want = model[0](x) - model[0].bias
        cast(model)
        assert model[0].tile_scales.dtype == torch.float32 and torch.equal(model[0].tile_scales, scales) and torch.equal(model[0].tiles, tiles)
        assert model[0].bias.dtype == model[1].weight.dtype
        model[0].bias.zero_()
        want2 = model[0](x)
    assert torch.allclose(want2, want, rtol=0, atol=2.0 ** -20 * float(want.abs().max() + 1))     # the bias came off with two roundings


def test_stacked_weights_follow_copies_and_replacements():
    """A deep copy of a model has its own stacked weight; buffers put in place of others are taken up, also where memory is reused."""
    import copy
    torch.manual_seed(5)
    parts = nn.ModuleList([fp8.Fp8Linear.from_linear(nn.Linear(256, n, bias=False).to(DEV)) for n in (64, 32)])
    q, s = _ops.fp8_rows(3, 256, DEV)
    _ops.quantize_rows_fp8(torch.randn(3, 256, device=DEV), q, s)

    def product(owner):
        return _ops.linear_fp8(q, s, fp8.stacked_weight(owner, "_stack", list(owner)), torch.empty(3, 96, device=DEV))

    def single(owner):
        return torch.cat([_ops.linear_fp8(q, s, m.packed, torch.empty(3, m.out_features, device=DEV)) for m in owner], dim=1)

    assert torch.equal(product(parts), single(parts))
    twin = copy.deepcopy(parts)
    with torch.no_grad():
        parts[0].tiles.zero_()
    assert torch.equal(product(parts), single(parts)) and torch.equal(product(twin), single(twin))
    assert not torch.equal(product(parts), product(twin))
    del parts
    new = fp8.Fp8Linear.from_linear(nn.Linear(256, 64, bias=False).to(DEV))
    twin[0].load_state_dict(new.state_dict(), assign=True)
    assert torch.equal(product(twin), single(twin))
    assert torch.equal(product(twin)[:, :64], _ops.linear_fp8(q, s, new.packed, torch.empty(3, 64, device=DEV)))


def test_stacking_inside_a_capture_is_refused():
    parts = [fp8.Fp8Linear.from_linear(nn.Linear(128, 16, bias=False).to(DEV)) for _ in range(2)]
    owner, x = nn.Module(), torch.zeros(4, device=DEV)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x.add_(1)
        with pytest.raises(RuntimeError, match="before capturing"):
            fp8.stacked_weight(owner, "_stack", parts)
    w = fp8.stacked_weight(owner, "_stack", parts)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x.add_(1)
        assert fp8.stacked_weight(owner, "_stack", parts) is w


def test_rows_of_another_width_are_refused():
    mod = fp8.Fp8Linear.from_linear(nn.Linear(128, 16).to(DEV))
    with pytest.raises(ValueError):
        mod(torch.zeros(4, 64, device=DEV))
