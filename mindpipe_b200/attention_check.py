"""Whether a model's attention is the one that :class:`~mindpipe_b200.attention.PagedSelfAttention` computes.

Model code keeps what it does between the projections in many places: child modules and attributes of any name, the config that
a forward reads, the function that rotates.  So the module itself is asked.  :func:`check_attention` runs its forward on the CPU
for a few tokens, with projections that return known queries, keys and values in fp32, and compares what reaches ``o_proj``
with the formula in 64 bits; the model's weights take no part and may be quantised, on any device or on none.  What a few tokens
cannot show -- windows, chunks, bidirectional attention -- is read from the config, and parameters that the replacement would
drop are refused.  :func:`check_table` compares the rotation's table with what the model's rotary module returns.

Everything here raises ``ValueError`` with the module's name, before anything of the model has changed.
"""
from __future__ import annotations

import copy
import inspect
from contextlib import contextmanager

import torch
from torch import nn

PROJECTIONS = ("q_proj", "k_proj", "v_proj", "o_proj")
_TOKENS = 7


class _Given(nn.Module):
    """In a projection's place: returns the same values whatever comes in, and keeps what came in."""

    def __init__(self, of: nn.Module, values: torch.Tensor):
        super().__init__()
        self.in_features, self.out_features, self.bias = getattr(of, "in_features", None), getattr(of, "out_features", None), None
        self.weight = nn.Parameter(torch.empty(0), requires_grad=False)
        self.values, self.seen = values, []

    def forward(self, x, *args, **kwargs):
        self.seen.append(x)
        return self.values.view(*x.shape[:-1], -1)


@contextmanager
def _plain_torch():
    """fp32 on the CPU, whatever the caller's defaults are."""
    dtype = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    try:
        with torch.no_grad(), torch.device("cpu"), torch.autocast("cpu", enabled=False):
            yield
    finally:
        torch.set_default_dtype(dtype)


def has_forward(module: nn.Module) -> bool:
    return type(module).forward is not nn.Module.forward


def _formula(q, k, v, cos_sin, scale):
    """Rotated in halves, causal, grouped: ``[tokens, heads * dim]`` in 64 bits."""
    half = cos_sin.shape[1] // 2
    c, s = cos_sin.double()[:, None, :half], cos_sin.double()[:, None, half:]

    def turn(x):
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)

    q, k, v = turn(q.double()), turn(k.double()), v.double()
    k, v = (x.repeat_interleave(q.shape[1] // x.shape[1], 1) for x in (k, v))
    scores = torch.einsum("qhd,khd->hqk", q, k) * scale
    scores = scores.masked_fill(torch.ones(scores.shape[1:], dtype=torch.bool).triu(1), -torch.inf)
    return torch.einsum("hqk,khd->qhd", scores.softmax(-1), v).flatten(1)


def _arguments(forward, cos_sin):
    """What the forward gets beside the hidden states, by the names of its parameters."""
    half = cos_sin.shape[1] // 2
    mask = torch.zeros(1, 1, _TOKENS, _TOKENS).masked_fill(torch.ones(_TOKENS, _TOKENS, dtype=torch.bool).triu(1),
                                                           torch.finfo(torch.float32).min)
    ids = torch.arange(_TOKENS)
    given = {"position_embeddings": tuple(torch.cat([x, x], -1)[None] for x in (cos_sin[:, :half], cos_sin[:, half:])),
             "attention_mask": mask, "position_ids": ids[None], "cache_position": ids, "past_key_value": None,
             "past_key_values": None, "use_cache": False, "output_attentions": False}
    parameters = list(inspect.signature(forward).parameters.values())[2:]            # behind self and the hidden states
    if not any(p.name == "position_embeddings" or p.kind is p.VAR_KEYWORD for p in parameters):
        raise TypeError("forward takes no position_embeddings")
    missing = [p.name for p in parameters if p.default is p.empty and p.kind not in (p.VAR_POSITIONAL, p.VAR_KEYWORD) and p.name not in given]
    if missing:
        raise TypeError(f"forward wants {', '.join(missing)}")
    names = {p.name for p in parameters}
    return {n: x for n, x in given.items() if n in names or n == "position_embeddings"}


def _clone(attention: nn.Module, projections: dict[str, nn.Module]) -> nn.Module:
    """The module's own code and attributes around other projections, in evaluation mode and with plain attention."""
    clone = copy.copy(attention)
    clone._parameters, clone._buffers = dict(attention._parameters), dict(attention._buffers)
    clone._modules = dict(attention._modules) | projections
    clone.training = False
    for name, child in attention.named_children():
        if name not in projections:                               # (without parameters: dropout, a rotation of its own)
            clone._modules[name] = copy.deepcopy(child).cpu().eval()
    config = getattr(attention, "config", None)
    if config is not None:
        clone.config = copy.deepcopy(config)                      # (setting it reaches the configs inside)
        if hasattr(config, "_attn_implementation"):
            clone.config._attn_implementation = "eager"
    return clone


def check_attention(attention: nn.Module, name: str, *, head_dim: int, rotated: int, scale: float | None) -> None:
    """``attention`` computes ``o_proj(softmax(scale rot(q) rot(k)^T, causal) v)`` of its own projections, heads in groups."""
    dropped = [n for n, p in attention._parameters.items() if p is not None] + \
        [n for n, c in attention.named_children() if n not in PROJECTIONS and next(c.parameters(), None) is not None]
    if dropped:
        raise ValueError(f"{name}: {', '.join(dropped)} is not part of the paged attention")
    if not has_forward(attention):
        return                                                    # projections and nothing else: there is no code to differ
    with _plain_torch():
        _compare(attention, name, head_dim, rotated, head_dim ** -0.5 if scale is None else float(scale))


def _compare(attention, name, head_dim, rotated, scale):
    g = torch.Generator().manual_seed(0)
    # scores of a few units, so that caps and norms show; large values, so that clamps do
    size = (4.0 / max(abs(scale) * head_dim ** 0.5, 1e-6)) ** 0.5
    q, k, v = (torch.randn(_TOKENS, getattr(attention, n).out_features // head_dim, head_dim, generator=g) * x
               for n, x in (("q_proj", size), ("k_proj", size), ("v_proj", 1000.0)))
    angle = torch.rand(_TOKENS, rotated // 2, generator=g) * 6
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1)
    want = _formula(q, k, v, cos_sin, scale)
    hidden = torch.randn(1, _TOKENS, attention.q_proj.in_features, generator=g)
    result = torch.randn(_TOKENS, attention.o_proj.out_features, generator=g)
    stand = {n: _Given(getattr(attention, n), x) for n, x in zip(PROJECTIONS, (q, k, v, result))}
    try:
        forward = type(attention).forward
        out = forward(_clone(attention, stand), hidden, **_arguments(forward, cos_sin))
        out = out[0] if isinstance(out, (tuple, list)) else out
        seen = {n: m.seen for n, m in stand.items()}
        reached = seen["o_proj"][0].reshape(_TOKENS, -1).double()
        same = all(len(x) == 1 for x in seen.values()) and all(torch.equal(seen[n][0].reshape(hidden.shape), hidden) for n in PROJECTIONS[:3])
        same = same and torch.equal(out.reshape(result.shape), result)
        off = ((reached - want).abs().max() / want.abs().max()).item()
    except Exception as e:
        raise ValueError(f"{name}: {type(attention).__name__} cannot be compared with the paged attention ({type(e).__name__}: {e}); "
                         "where it is the same, put PagedSelfAttention in its place by hand") from e
    if not same or not off <= 1e-4:
        raise ValueError(f"{name}: {type(attention).__name__} does not compute what the paged attention does "
                         "(projections, rotation in halves, causal softmax, nothing else)")


def check_table(rotary: nn.Module, cos_sin: torch.Tensor) -> None:
    """``cos_sin`` holds what ``rotary(x, position_ids)`` returns: cosines and sines, each twice in halves."""
    if not has_forward(rotary):
        return
    rows, half = cos_sin.shape[0], cos_sin.shape[1] // 2
    ids = torch.tensor(sorted(p for p in {0, 1, 2, 3, rows // 2, rows - 1} if p < rows), device="cpu")
    table = cos_sin[ids.to(cos_sin.device)].cpu()
    want = [torch.cat([x, x], -1)[None] for x in (table[:, :half], table[:, half:])]
    try:
        with _plain_torch():
            got = type(rotary).forward(copy.deepcopy(rotary).cpu(), torch.zeros(1, len(ids), 1), ids[None])
        # (the model's angles are taken in 32 bits)
        same = len(got) == 2 and all(g.shape == w.shape and bool(((g.double() - w).abs() <= 1e-4 + ids[None, :, None] * 2.0 ** -22).all())
                                     for g, w in zip(got, want))
    except Exception as e:
        raise ValueError(f"{type(rotary).__name__} cannot be compared with a table ({type(e).__name__}: {e}): pass cos_sin") from e
    if not same:
        raise ValueError(f"{type(rotary).__name__} does not rotate by a table of inv_freq in halves: pass cos_sin")


def check_config(config, name: str, layer: int, positions: int) -> None:
    """No window or chunk is smaller than ``positions``, attention is causal, positions are single numbers."""
    get = lambda key, default=None: getattr(config, key, default)
    kinds = get("layer_types")
    kind = kinds[layer] if kinds and layer < len(kinds) else None
    if kind not in (None, "full_attention", "sliding_attention", "chunked_attention"):
        raise ValueError(f"{name}: attention of the kind {kind!r} is not the paged attention")
    if kind != "full_attention":
        windows = {key: get(key) for key in ("sliding_window", "attention_chunk_size") if get(key) is not None}
        if kind is None and get("use_sliding_window", True) is False:
            windows.pop("sliding_window", None)
        if kind is not None and not windows:
            raise ValueError(f"{name}: {kind} without its size in the config")
        for key, size in windows.items():
            if not isinstance(size, int) or size < positions:
                raise ValueError(f"{name}: {key} of {size} is less than the table's {positions} positions, and not part of the paged "
                                 "attention (max_positions up to it is)")
    if get("use_bidirectional_attention", False) or get("is_causal", True) is False:
        raise ValueError(f"{name}: the paged attention is causal")
    for key in ("rope_parameters", "rope_scaling"):
        if "mrope_section" in (get(key) or {}):
            raise ValueError(f"{name}: positions of several parts (mrope_section) are not part of the paged attention")
