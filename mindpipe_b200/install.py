"""Model-level installers: put the real-quant twins where the reference puts its pseudo-quant modules.

Two entry points with the reference's names, arguments and error behaviour:

* :func:`quantize_model` -- SmoothQuant's installer
  (``ptq/smoothquant/source/smoothquant/fake_quant.py:441-458`` -> ``quantize_llama_like`` ``:227-437``):
  walks the decoder layers of a llama-like model, replaces the attention and MLP projections by
  :class:`~mindpipe_b200.modules.SmoothQuantLinear` and packed MoE experts by
  :class:`~mindpipe_b200.modules.SmoothQuantPackedMoeExperts`, and returns the qualified names it replaced.
* :func:`real_quantize_model_weight` -- the real-int counterpart of AWQ's ``pseudo_quantize_model_weight``
  (``ptq/awq/source/awq/quantize/quantizer.py:109-130``): instead of writing fake-quant fp16 weights back into
  every ``nn.Linear`` of every block it replaces the linear by a
  :class:`~mindpipe_b200.modules.VllmPackedInt4Linear` holding the same codes, scales and zero points packed.

:func:`load_exported_state_dict` fills installed twins from a checkpoint in the reference's export formats
(``exporters/vllm.py:224-327``: ``*.weight_packed / weight_scale / weight_shape``; the W8A8 exporter
``scripts/repro/export_fp16_to_ascend_w8a8_dynamic_probe.py:175-195``: ``*.weight / weight_scale / weight_offset``).

:func:`install_paged_attention` replaces the layers' ``self_attn`` by :class:`~mindpipe_b200.attention.PagedSelfAttention`
around the projections that are there, quantised or not.

The twins quantise on the GPU, so the model's linears must already live on a CUDA device.
"""
from __future__ import annotations

from typing import Iterable

import torch
from torch import nn

from .attention import PagedKVCache, PagedSelfAttention, rotary_table
from .attention_check import check_attention, check_config, check_table
from .modules import SmoothQuantLinear, SmoothQuantPackedMoeExperts, VllmPackedInt4Linear

_ATTN_PROJ = ("q_proj", "k_proj", "v_proj")
_MLP_PROJ = ("gate_proj", "up_proj", "down_proj")


def _backbone(model: nn.Module) -> nn.Module:
    """The module that holds the decoder layers, found the way ``awq/quantize/pre_quant.py:47-76`` finds them."""
    if hasattr(model, "model") and hasattr(model.model, "language_model"):
        return model.model.language_model
    if hasattr(model, "language_model") and hasattr(model.language_model, "layers"):
        return model.language_model
    if hasattr(model, "model") and hasattr(model.model, "layers"):
        return model.model
    if hasattr(model, "layers") and isinstance(model.layers, (nn.ModuleList, list)):
        return model
    raise NotImplementedError(type(model))


def get_blocks(model: nn.Module):
    """The decoder layers (text backbones only)."""
    return _backbone(model).layers


def _blocks_prefix(model: nn.Module) -> str:
    layers = get_blocks(model)
    for name, mod in model.named_modules():
        if mod is layers:
            return name
    return "layers"


def get_named_linears(module: nn.Module) -> dict[str, nn.Linear]:
    """``awq/quantize/pre_quant.py:34-35``: every ``nn.Linear`` below ``module`` by its relative name."""
    return {name: m for name, m in module.named_modules() if isinstance(m, nn.Linear)}


def _set_submodule(root: nn.Module, name: str, new: nn.Module) -> None:
    parent = root
    parts = name.split(".")
    for part in parts[:-1]:
        parent = getattr(parent, part)
    setattr(parent, parts[-1], new)


def _require_cuda(linear: nn.Linear, name: str) -> None:
    if linear.weight.device.type != "cuda":
        raise ValueError(f"{name}: the real-quant modules quantise on the GPU; move the model to a CUDA device first")


@torch.no_grad()
def real_quantize_model_weight(model: nn.Module, w_bit: int, q_config: dict, skip: Iterable[str] = ()) -> list[str]:
    """Replace every ``nn.Linear`` of every block by a packed int4 linear.

    ``q_config`` is AWQ's dictionary (``{"zero_point": bool, "q_group_size": int}``).  Only ``w_bit == 4`` and
    positive group sizes exist as kernels; anything else raises ``ValueError`` (the reference would fake-quantise
    it, a real-int format for it does not exist here).  Returns the qualified names that were replaced.
    """
    if w_bit != 4:
        raise ValueError(f"only w_bit=4 has a packed format and kernels, got {w_bit}")
    group = int(q_config.get("q_group_size", 128))
    if group <= 0:
        raise ValueError("per-channel (q_group_size <= 0) int4 has no packed kernel format; use a positive group size")
    zero_point = bool(q_config.get("zero_point", True))
    skip = tuple(skip)
    prefix = _blocks_prefix(model)
    replaced = []
    for i, block in enumerate(get_blocks(model)):
        for name, linear in get_named_linears(block).items():
            if any(s in name for s in skip):
                continue
            qualified = f"{prefix}.{i}.{name}"
            _require_cuda(linear, qualified)
            _set_submodule(block, name, VllmPackedInt4Linear.from_float(linear, w_bit=4, group_size=group,
                                                                         zero_point=zero_point))
            replaced.append(qualified)
    return replaced


def _replace_linear_with_smoothquant(module, proj_name, names, qualified, *, weight_bits, activation_bits, act_quant,
                                     quantize_output=False):
    linear = getattr(module, proj_name)
    _require_cuda(linear, qualified)
    setattr(module, proj_name, SmoothQuantLinear.from_float(linear, weight_bits=weight_bits,
                                                            activation_bits=activation_bits, act_quant=act_quant,
                                                            quantize_output=quantize_output))
    names.append(qualified)


@torch.no_grad()
def quantize_llama_like(model, weight_bits=8, activation_bits=8, act_quant="per_token", quantize_bmm_input=True):
    """``fake_quant.py:227-437`` for the standard attention + (dense | MoE) MLP layer layout: q/k/v (output
    re-quantised when ``quantize_bmm_input``), o, gate/up/down, shared expert, expert lists and packed experts.
    Models without ``config.model_type`` are accepted (the reference needs the type to pick a layout; this
    walker reads the layout off the modules), unsupported layouts raise ``ValueError``."""
    layers = get_blocks(model)
    prefix = _blocks_prefix(model)
    names: list[str] = []
    kw = dict(weight_bits=weight_bits, activation_bits=activation_bits, act_quant=act_quant)
    for i, layer in enumerate(layers):
        lp = f"{prefix}.{i}"
        attn = getattr(layer, "self_attn", None)
        mlp = getattr(layer, "mlp", None)
        if attn is None or mlp is None:
            raise ValueError(f"Unsupported layer layout at {lp}: expected .self_attn and .mlp")
        for proj in _ATTN_PROJ:
            _replace_linear_with_smoothquant(attn, proj, names, f"{lp}.self_attn.{proj}",
                                             quantize_output=quantize_bmm_input, **kw)
        _replace_linear_with_smoothquant(attn, "o_proj", names, f"{lp}.self_attn.o_proj", **kw)
        experts = getattr(mlp, "experts", None)
        if experts is None:
            for proj in _MLP_PROJ:
                _replace_linear_with_smoothquant(mlp, proj, names, f"{lp}.mlp.{proj}", **kw)
            continue
        shared = getattr(mlp, "shared_expert", None)
        if shared is not None:
            for proj in _MLP_PROJ:
                _replace_linear_with_smoothquant(shared, proj, names, f"{lp}.mlp.shared_expert.{proj}", **kw)
        if isinstance(experts, nn.ModuleList):
            for e, expert in enumerate(experts):
                for proj in _MLP_PROJ:
                    _replace_linear_with_smoothquant(expert, proj, names, f"{lp}.mlp.experts.{e}.{proj}", **kw)
        else:
            mlp.experts = SmoothQuantPackedMoeExperts.from_float(experts, weight_bits=weight_bits,
                                                                 activation_bits=activation_bits)
            names.append(f"{lp}.mlp.experts.gate_up_proj")
            names.append(f"{lp}.mlp.experts.down_proj")
    return names


def quantize_model(model, weight_bits=8, activation_bits=8, weight_quant="per_channel", act_quant="per_token",
                   quantize_bmm_input=True):
    """``fake_quant.py:441-458``: same arguments, same ``ValueError`` for anything but per-channel weights."""
    if weight_quant != "per_channel":
        raise ValueError(f"Invalid weight_quant: {weight_quant}")
    return quantize_llama_like(model, weight_bits=weight_bits, activation_bits=activation_bits, act_quant=act_quant,
                               quantize_bmm_input=quantize_bmm_input)


def install_paged_attention(model: nn.Module, cache: PagedKVCache, *, cos_sin: torch.Tensor | None = None,
                            max_positions: int | None = None) -> list[str]:
    """Run the attention of every decoder layer on ``cache``; returns the qualified names that were replaced.

    Works before or after the installers of the linears; ``install_paged_attention`` does not touch them.  The rotation's
    table is ``cos_sin`` (fp32 ``[positions, rotated]``, cosines then sines) or made from the ``rotary_emb`` beside the layers
    (``inv_freq`` and ``attention_scaling``) for ``max_positions`` positions (default: the config's
    ``max_position_embeddings``).  Layers whose attention does anything but project, rotate in halves and attend causally --
    normalised queries or keys, windows smaller than the table, capped scores, clamped values, rotation of neighbours or none,
    positions of several parts, whatever else changes its results (:mod:`mindpipe_b200.attention_check`) -- or that carry
    another state from token to token raise ``ValueError`` before anything is replaced.  A model that pairs neighbours, or whose
    attention cannot be asked, is put together from :class:`PagedSelfAttention` by hand.
    """
    backbone, prefix = _backbone(model), _blocks_prefix(model)
    layers = backbone.layers
    if len(layers) != cache.pool.shape[0]:
        raise ValueError(f"the model has {len(layers)} layers, the cache {cache.pool.shape[0]}")
    if cos_sin is None:
        cos_sin = _model_table(model, backbone, max_positions, cache.pool.device)
    if cos_sin.dim() != 2 or cos_sin.shape[0] < 1 or cos_sin.shape[1] % 2 or not 2 <= cos_sin.shape[1] <= cache.pool.shape[-1]:
        raise ValueError(f"cos_sin must be [positions, rotated] with an even number of rotated values up to the cache's heads of "
                         f"{cache.pool.shape[-1]}, got {tuple(cos_sin.shape)}")
    made = []
    for i, layer in enumerate(layers):
        attn, name = getattr(layer, "self_attn", None), f"{prefix}.{i}.self_attn"
        if attn is None:
            raise ValueError(f"Unsupported layer layout at {prefix}.{i}: expected .self_attn")
        config = next((c for c in (getattr(m, "config", None) for m in (attn, backbone, model)) if c is not None), None)
        check_config(config, name, i, cos_sin.shape[0])
        if isinstance(attn, PagedSelfAttention):                  # installed already: it keeps its own scale and pairs
            made.append((layer, name, PagedSelfAttention(attn, cache, i, cos_sin, scale=attn.scale, interleaved=attn.interleaved)))
            continue
        for extra in ("q_norm", "k_norm", "sliding_window", "attn_logit_softcapping", "sinks"):
            if getattr(attn, extra, None) is not None:
                raise ValueError(f"{name}: {extra} is not part of the paged attention")
        if getattr(attn, "is_causal", True) is False:
            raise ValueError(f"{name}: the paged attention is causal")
        if any(isinstance(m, nn.Conv1d) for m in layer.modules()):
            raise ValueError(f"{prefix}.{i}: a convolution over tokens has a state of its own, which the cache does not hold")
        new = PagedSelfAttention(attn, cache, i, cos_sin, head_dim=getattr(attn, "head_dim", None), scale=getattr(attn, "scaling", None))
        check_attention(attn, name, head_dim=new.head_dim, rotated=cos_sin.shape[1], scale=new.scale)
        made.append((layer, name, new))
    for layer, _, new in made:
        layer.self_attn = new
    return [name for _, name, _ in made]


def _model_table(model: nn.Module, backbone: nn.Module, max_positions: int | None, device) -> torch.Tensor:
    """The table of the rotary module that serves ``backbone`` (a vision tower beside it may have one of its own)."""
    rotary = [m for m in backbone.modules() if hasattr(m, "inv_freq")] or [m for m in model.children() if hasattr(m, "inv_freq")]
    if not rotary:
        raise ValueError("the model has no rotary_emb with inv_freq: pass cos_sin")
    for m in rotary:
        kind = getattr(m, "rope_type", "default")
        if kind in ("dynamic", "longrope"):
            raise ValueError(f"the frequencies of rope type {kind!r} depend on the length: pass cos_sin")
        if not torch.equal(m.inv_freq.to(rotary[0].inv_freq.device), rotary[0].inv_freq):
            raise ValueError("the model's layers rotate by different frequencies")
    limit = max_positions or next((n for n in (getattr(getattr(m, "config", None), "max_position_embeddings", None) for m in (backbone, model))
                                   if n is not None), None)
    if limit is None:
        raise ValueError("pass max_positions")
    table = rotary_table(rotary[0].inv_freq.to(device), int(limit), float(getattr(rotary[0], "attention_scaling", 1.0)))
    check_table(rotary[0], table)
    return table


_W4_KEYS = ("weight_packed", "weight_scale", "weight_zero_point", "weight_shape", "bias")
_W8_KEYS = ("weight", "weight_scale", "weight_offset", "bias")


@torch.no_grad()
def load_exported_state_dict(model: nn.Module, state_dict: dict) -> list[str]:
    """Copy an exported real-quant checkpoint into the installed twins; returns the module names it filled.

    W4 modules take ``weight_packed`` / ``weight_scale`` / ``weight_shape`` (+ ``weight_zero_point`` when the
    export is asymmetric); W8A8 modules take ``weight`` (int8) / ``weight_scale`` and check that
    ``weight_offset`` is zero (the kernels are symmetric, as the exporter's dynamic-W8A8 format is).  A module
    whose tensors are missing or mis-shaped raises ``KeyError`` / ``ValueError`` naming it.
    """
    filled = []
    for name, mod in model.named_modules():
        pre = f"{name}." if name else ""
        if isinstance(mod, VllmPackedInt4Linear):
            for key in ("weight_packed", "weight_scale"):
                if pre + key not in state_dict:
                    raise KeyError(f"{pre}{key} is missing from the checkpoint")
            shape = state_dict.get(pre + "weight_shape")
            if shape is not None and [int(v) for v in shape] != [mod.out_features, mod.in_features]:
                raise ValueError(f"{name}: checkpoint weight_shape {list(map(int, shape))} != "
                                 f"[{mod.out_features}, {mod.in_features}]")
            for key in ("weight_packed", "weight_scale", "weight_zero_point", "bias"):
                src = state_dict.get(pre + key)
                dst = getattr(mod, key, None)
                if src is None:
                    if key == "weight_zero_point" and dst is not None:
                        raise KeyError(f"{pre}{key} is missing: the module was built for an asymmetric export")
                    continue
                if dst is None:
                    raise ValueError(f"{name}: the checkpoint has {key} but the module was built without it")
                if tuple(dst.shape) != tuple(src.shape):
                    raise ValueError(f"{name}.{key}: checkpoint shape {tuple(src.shape)} != {tuple(dst.shape)}")
                dst.copy_(src.to(dst.dtype))
            mod._scale_zero = None
            mod.process_weights_after_loading()
            filled.append(name)
        elif isinstance(mod, SmoothQuantLinear):
            for key in ("weight", "weight_scale"):
                if pre + key not in state_dict:
                    raise KeyError(f"{pre}{key} is missing from the checkpoint")
            off = state_dict.get(pre + "weight_offset")
            if off is not None and bool(torch.any(off != 0)):
                raise ValueError(f"{name}: non-zero weight_offset; the W8A8 kernels are symmetric")
            w = state_dict[pre + "weight"]
            if w.dtype != torch.int8 or tuple(w.shape) != tuple(mod.weight.shape):
                raise ValueError(f"{name}.weight: expected int8 {tuple(mod.weight.shape)}, got {w.dtype} {tuple(w.shape)}")
            mod.weight.copy_(w)
            mod.weight_scale.copy_(state_dict[pre + "weight_scale"].reshape(mod.weight_scale.shape).to(mod.weight_scale.dtype))
            b = state_dict.get(pre + "bias")
            if b is not None and getattr(mod, "bias", None) is not None:
                mod.bias.copy_(b.to(mod.bias.dtype))
            mod.process_weights_after_loading()
            filled.append(name)
    return filled
