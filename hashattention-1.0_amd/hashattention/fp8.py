"""Projections in 8 bits for `transformers` models: e4m3 weights with one scale per 128 x 128 block, activations quantised per row and
128 inputs on their way into each projection (`ha_linear_fp8` and the row operators in front of it).

    model = convert_usa(model, config, usa, False, False)      # optional, and first
    model = convert_fp8(model)                                 # every decoder layer's seven projections
    model.generate(...)

`convert_fp8` replaces the projections of every decoder layer of the Llama shape (q, k, v, o, gate, up, down) by `Fp8Linear` and frees
the 16-bit weights: half the memory, half the bytes a decode step streams, and prompts on the 8-bit matrix instructions.  Norms,
embeddings and the lm_head stay as they are.  A converted layer's single-token steps run as a fixed set of launches around
`HeavyHitterMixin._fast_decode` (see `_patched.fast_decoder_layer_forward`).  Inference only.
"""
from __future__ import annotations

import warnings
from typing import Optional, Sequence

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _ops

__all__ = ["Fp8Linear", "convert_fp8", "stacked_weight"]


class Fp8Linear(nn.Module):
    """`nn.Linear` for inference with its weight in 8 bits.  `tiles` and `tile_scales` are buffers (`_ops.pack_weight_fp8`), so the
    module moves and is saved like any other.  Casts of the model to another type leave both as they are."""

    def __init__(self, weight: _ops.Fp8Weight, bias: Optional[torch.Tensor] = None):
        super().__init__()
        if weight.glu:
            raise ValueError("interleaved gate/up weights have no plain product")
        self.in_features, self.out_features = weight.K, weight.N
        self.register_buffer("tiles", weight.tiles)
        self.register_buffer("tile_scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().contiguous())

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Fp8Linear":
        return cls(_ops.pack_weight_fp8(linear.weight.detach()), linear.bias)

    @property
    def packed(self) -> _ops.Fp8Weight:
        return _ops.Fp8Weight(self.tiles, self.tile_scales, self.out_features, self.in_features, False)

    def __setattr__(self, name, value):
        if name in ("tiles", "tile_scales"):
            self._leave_stack()
        super().__setattr__(name, value)

    def _leave_stack(self):
        """The stacked weight this module's buffers are parts of (`stacked_weight`) is held no longer: it is out of date."""
        for holder in self.__dict__.pop("_stack", ()):
            holder.clear()

    def _apply(self, fn, recurse=True):
        # casts (`model.bfloat16()`, `model.to(dtype)`) skip integers: the scales pass as their bits and stay fp32
        own = self._buffers
        before = own["tiles"].data_ptr(), own["tile_scales"].data_ptr()
        own["tile_scales"] = own["tile_scales"].view(torch.int32)
        try:
            return super()._apply(fn, recurse)
        finally:
            own["tile_scales"] = own["tile_scales"].view(torch.float32)
            if before != (own["tiles"].data_ptr(), own["tile_scales"].data_ptr()):
                self._leave_stack()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1:] != (self.in_features,):
            raise ValueError(f"x has rows of {tuple(x.shape[-1:])}, the weight takes {self.in_features}")
        if torch.is_grad_enabled() and x.requires_grad or forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError("Fp8Linear is for inference: no gradient flows through the 8-bit product (use torch.no_grad())")
        rows = x.reshape(-1, self.in_features)
        if self.in_features > 1 and rows.stride(1) != 1:
            rows = rows.contiguous()
        q, scales = _ops.fp8_rows(rows.shape[0], self.in_features, x.device)
        _ops.quantize_rows_fp8(rows, q, scales)
        bias, dtype = self.bias, x.dtype
        # the bias is added in front of the result's one rounding; one of another type that x's does not hold, to sums in fp32
        if bias is not None and torch.promote_types(bias.dtype, dtype) != dtype:
            dtype = torch.float32
        out = torch.empty(rows.shape[0], self.out_features, dtype=dtype, device=x.device)
        _ops.linear_fp8(q, scales, self.packed, out, None if bias is None else bias.to(dtype).expand(out.shape))
        if dtype != x.dtype:
            out = out.to(x.dtype)
        return out.view(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, e4m3 per 128 x 128 block"


def _stacks(modules: Sequence[Fp8Linear]) -> bool:
    """Whether the modules' rows can lie behind each other in one packed matrix: whole tiles of 16 rows in front of the last."""
    return all(m.out_features % 16 == 0 for m in modules[:-1]) and len({m.in_features for m in modules}) == 1


def stacked_weight(owner: nn.Module, name: str, modules: Sequence[Fp8Linear]) -> _ops.Fp8Weight:
    """The modules' weights as one matrix, rows behind each other, kept on `owner` under `name`.  Packed tiles are ordered by row, so
    the modules' own buffers become parts of the stacked ones: nothing is held twice.  Each module's blocks of 128 rows begin at its
    own first row; where that is no multiple of 128 in the stacked matrix, the weight names its parts (`_ops.Fp8Weight`).  Rebuilt
    when a module's buffer is no longer that part (a move to another device, a loaded state dict): call it once before a graph is
    captured."""
    holder = owner.__dict__.get(name)       # [weight], emptied by the first module whose buffers move on
    if holder and _parts_of(holder[0], modules):
        return holder[0]
    if not _stacks(modules):
        raise ValueError("rows of packed weights stack in whole tiles of 16")
    if modules[0].tiles.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the projections' weights are not stacked yet: run one step before capturing a graph")
    with torch.inference_mode(False), torch.no_grad():      # ordinary tensors, which a state dict can be loaded into at any time
        tiles, scales = torch.cat([m.tiles for m in modules]), torch.cat([m.tile_scales for m in modules])
        at = s_at = 0
        for m in modules:
            n, ns = m.tiles.numel(), m.tile_scales.numel()
            m.tiles, m.tile_scales = tiles[at:at + n], scales[s_at:s_at + ns]
            at, s_at = at + n, s_at + ns
    rows = tuple(m.out_features for m in modules)
    weight = _ops.Fp8Weight(tiles, scales, sum(rows), modules[0].in_features, False,
                            rows if any(n % _ops.FP8_BLOCK for n in rows[:-1]) else ())
    holder = owner.__dict__[name] = [weight]
    for m in modules:
        m.__dict__["_stack"] = (holder,)
    return weight


def _parts_of(weight: _ops.Fp8Weight, modules: Sequence[Fp8Linear]) -> bool:
    """Whether the modules' buffers are the stacked weight's memory, in order (it is alive, so no other tensor can lie there)."""
    at, s_at = weight.tiles.data_ptr(), weight.scales.data_ptr()
    for m in modules:
        tiles, scales = m.tiles, m.tile_scales
        if tiles.data_ptr() != at or scales.data_ptr() != s_at:
            return False
        at, s_at = at + tiles.numel(), s_at + 4 * scales.numel()
    return True


_ATTENTION, _MLP = ("q_proj", "k_proj", "v_proj", "o_proj"), ("gate_proj", "up_proj", "down_proj")


def _is_plain(lin) -> bool:
    """Whether a projection computes x W^T (+ bias) and nothing else: no subclass (an adapter, a parametrization), no hook, no forward of
    its own.  accelerate's placement of a model spread over devices only moves inputs, which the layer's own hook does too."""
    if type(lin) is not nn.Linear or lin._forward_hooks or lin._forward_pre_hooks:
        return False
    return "forward" not in lin.__dict__ or type(getattr(lin, "_hf_hook", None)).__name__ == "AlignDevicesHook"


def _projections(layer: nn.Module) -> list:
    """The (owner, name) of a decoder layer's seven projections, and of the four of the module a converted attention module prefills
    through, which holds weights of its own; empty if the module is no such layer."""
    attn, mlp = getattr(layer, "self_attn", None), getattr(layer, "mlp", None)
    found = [(attn, n) for n in _ATTENTION] + [(mlp, n) for n in _MLP]
    if attn is None or mlp is None or not all(isinstance(getattr(o, n, None), nn.Linear) for o, n in found):
        return []
    twin = getattr(getattr(attn, "flash_forward", None), "__self__", None)
    return found + [(twin, n) for n in _ATTENTION if isinstance(getattr(twin, n, None), nn.Linear)]


def convert_fp8(model: nn.Module) -> nn.Module:
    """Replace the seven projections of every decoder layer in place by `Fp8Linear`.  The model is on the GPU; `convert_usa`, where it
    is used, comes first (it copies 16-bit weights).  A layer with a projection that is more than an nn.Linear - a subclass with a
    forward of its own, a hook - is left as it is, with a warning."""
    layers = {m: p for m in model.modules() if (p := _projections(m))}
    plain = {m: p for m, p in layers.items() if all(_is_plain(getattr(o, n)) for o, n in p)}
    if not plain:
        raise ValueError("no decoder layer with q/k/v/o and gate/up/down projections of type nn.Linear, without hooks, in this model")
    if len(plain) < len(layers):
        warnings.warn(f"{len(layers) - len(plain)} decoder layer(s) keep their projections: subclasses of nn.Linear, hooks or a forward of their own")
    for layer, projections in plain.items():
        attn = layer.self_attn
        for owner, name in projections[:7]:
            setattr(owner, name, Fp8Linear.from_linear(getattr(owner, name)))
        for owner, name in projections[7:]:
            setattr(owner, name, getattr(attn, name))
        for copy in ("_qkv_fused", "_qkv_tiles", "_o_tiles", "_gate_up_fused", "_gate_up_tiles", "_down_tiles"):
            attn.__dict__.pop(copy, None)        # stacked and tiled copies of the 16-bit weights, if steps ran before
    return model
