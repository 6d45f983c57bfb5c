"""What ``install_paged_attention`` takes and refuses, on models of real classes and on plain trees, without a GPU."""
import pytest
import torch
from torch import nn

from mindpipe_b200 import install
from mindpipe_b200.attention import PagedKVCache, PagedSelfAttention, rotary_table
from tests._tiny_llama import TinyLlama


def make_cache(layers=2, heads=2, dim=64, pages=20, page=8):
    cache = PagedKVCache(layers, pages, page, heads, dim, device="cpu")
    cache.pool = cache.pool.float()                               # (plain forms of the operators have no types to keep)
    return cache


def test_installing_again_keeps_scale_and_pairs():
    model, table = TinyLlama(), rotary_table(torch.ones(32), 8)
    attn = model.model.layers[0].self_attn
    attn.scaling = 0.25
    install.install_paged_attention(model, make_cache(), cos_sin=table)
    model.model.layers[1].self_attn.interleaved = True
    cache = make_cache()
    assert len(install.install_paged_attention(model, cache, cos_sin=table)) == 2
    first, second = (layer.self_attn for layer in model.model.layers)
    assert first.scale == 0.25 and first.interleaved is False and second.scale is None and second.interleaved is True
    assert first.cache is cache and first.q_proj is attn.q_proj and isinstance(first, PagedSelfAttention)


class _Rotary(nn.Module):
    def __init__(self, inv_freq):
        super().__init__()
        self.register_buffer("inv_freq", inv_freq)


def test_the_table_is_that_of_the_layers_rotation():
    """A tower beside the language model, in front of it in the tree, has frequencies of its own."""
    class Tree(nn.Module):
        def __init__(self):
            super().__init__()
            self.model = nn.Module()
            self.model.visual = _Rotary(torch.ones(4))
            self.model.language_model = TinyLlama().model
            self.model.language_model.rotary_emb = _Rotary(inv)

    inv = 100.0 ** (-torch.arange(32) / 32)
    model = Tree()
    install.install_paged_attention(model, make_cache(), max_positions=50)
    assert torch.equal(model.model.language_model.layers[1].self_attn.cos_sin, rotary_table(inv, 50))
    model = Tree()
    del model.model.language_model.rotary_emb
    with pytest.raises(ValueError, match="pass cos_sin"):
        install.install_paged_attention(model, make_cache(), max_positions=50)
    model = Tree()
    model.model.language_model.layers[1].rotary_emb = _Rotary(inv * 2)
    with pytest.raises(ValueError, match="different frequencies"):
        install.install_paged_attention(model, make_cache(), max_positions=50)
