"""What ``install_paged_attention`` takes and refuses, on models of real classes and on plain trees, without a GPU."""
import pytest
import torch
from torch import nn

from mindpipe_b200 import install
from mindpipe_b200.attention import PagedKVCache, PagedSelfAttention, rotary_table
from tests import _attention_cpu
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


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return x * cos[:, None] + torch.cat([-b, a], -1) * sin[:, None]


def _rotate_neighbours(x, cos, sin):
    half = cos.shape[-1] // 2
    c, s = cos[:, None, :, :half], sin[:, None, :, :half]
    a, b = x[..., ::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)


class _Attention(nn.Module):
    """Two heads of keys, four of queries, 64 values each, with one thing done differently."""

    def __init__(self, of, kind):
        super().__init__()
        for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
            setattr(self, name, getattr(of, name))
        self.kind, self.head_dim, self.dropout = kind, 64, nn.Dropout(0.5)
        if kind == "norm of another name":
            self.pre_rotation = nn.RMSNorm(64)
        if kind == "bias of its own":
            self.offset = nn.Parameter(torch.zeros(64))
        if kind == "scale of another name":
            self.softmax_scale = 0.3
        if kind == "scale":
            self.scaling = 0.3

    def forward(self, hidden_states, position_embeddings, attention_mask=None, **kwargs):
        lead, kind = hidden_states.shape[:-1], self.kind
        x = hidden_states * 2 if kind == "input scaled" else hidden_states
        q, k, v = (p(x).view(*lead, -1, 64).transpose(1, 2) for p in (self.q_proj, self.k_proj, self.v_proj))
        if kind == "norm of another name":
            q, k = self.pre_rotation(q), self.pre_rotation(k)
        if kind == "norm without weights":
            q, k = (nn.functional.rms_norm(y, (64,)) for y in (q, k))
        if kind == "clamp":
            v = v.clamp(-8, 8)
        turn = _rotate_neighbours if kind == "neighbours" else _rotate
        if kind != "no rotation":
            q, k = (turn(y, *position_embeddings) for y in (q, k))
        k, v = (y.repeat_interleave(2, 1) for y in (k, v))
        s = q @ k.transpose(-1, -2) * (getattr(self, "softmax_scale", None) or getattr(self, "scaling", None) or 64 ** -0.5)
        if kind == "cap":
            s = 50 * torch.tanh(s / 50)
        if kind != "no mask":
            s = s + attention_mask
        if kind == "heads in turn":
            k, v = k[:, [0, 2, 1, 3]], v[:, [0, 2, 1, 3]]
        p = s.softmax(-1)
        if kind == "off by one":
            p = s.exp() / (1 + s.exp().sum(-1, keepdim=True))
        out = self.o_proj((self.dropout(p) @ v).transpose(1, 2).flatten(-2))
        return out * 0.5 if kind == "output scaled" else out, None


class _Bare(_Attention):
    def forward(self, hidden_states, cos, sin):
        raise AssertionError("not called")


@pytest.mark.parametrize("kind", ["plain", "scale"])
def test_a_module_that_computes_the_same_is_taken(kind):
    model = TinyLlama()
    for layer in model.model.layers:
        layer.self_attn = _Attention(layer.self_attn, kind)
    before = {n: x.clone() for n, x in model.state_dict().items()}
    assert len(install.install_paged_attention(model, make_cache(), cos_sin=rotary_table(torch.ones(32), 8))) == 2
    assert model.model.layers[0].self_attn.scale == (0.3 if kind == "scale" else None)
    assert all(torch.equal(x, before[n]) for n, x in model.state_dict().items())


@pytest.mark.parametrize("kind", ["norm of another name", "norm without weights", "bias of its own", "clamp", "neighbours", "no rotation",
                                  "scale of another name", "cap", "no mask", "heads in turn", "off by one", "input scaled", "output scaled"])
def test_a_module_that_computes_something_else_is_refused(kind):
    model = TinyLlama()
    model.model.layers[1].self_attn = _Attention(model.model.layers[1].self_attn, kind)
    with pytest.raises(ValueError, match="layers.1.self_attn"):
        install.install_paged_attention(model, make_cache(), cos_sin=rotary_table(torch.ones(32), 8))
    assert not isinstance(model.model.layers[0].self_attn, PagedSelfAttention)


def test_a_module_that_cannot_be_asked_is_refused():
    model = TinyLlama()
    model.model.layers[1].self_attn = _Bare(model.model.layers[1].self_attn, "plain")
    with pytest.raises(ValueError, match="cannot be compared"):
        install.install_paged_attention(model, make_cache(), cos_sin=rotary_table(torch.ones(32), 8))
    model = TinyLlama()
    model.model.layers[0].mixer = nn.Conv1d(4, 4, 3)
    with pytest.raises(ValueError, match="state of its own"):
        install.install_paged_attention(model, make_cache(), cos_sin=rotary_table(torch.ones(32), 8))


# ---- real classes, small
SMALL = dict(vocab_size=128, hidden_size=128, intermediate_size=96, num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=2,
             head_dim=32, max_position_embeddings=128, pad_token_id=0, bos_token_id=1, eos_token_id=2)
EXPERTS = dict(num_experts=4, num_local_experts=4, num_experts_per_tok=2, moe_intermediate_size=64)
LLAMA3 = dict(rope_type="llama3", rope_theta=10000.0, factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=64)
YARN = dict(rope_type="yarn", rope_theta=10000.0, factor=4.0, original_max_position_embeddings=64)


def build(kind, **settings):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(0)
    config = transformers.AutoConfig.for_model(kind, **(SMALL | settings))
    model = transformers.AutoModelForCausalLM.from_config(config, attn_implementation="eager").eval().float()
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() > 1:
                p.mul_(3)                                         # so that attention counts
    return model


@pytest.mark.parametrize("kind,settings,positions", [
    ("llama", {}, None), ("llama", dict(rope_parameters=LLAMA3), None), ("llama", dict(rope_parameters=YARN), None),
    ("llama", dict(attention_bias=True), None), ("mistral", dict(sliding_window=None), None), ("mistral", dict(sliding_window=70), 70),
    ("mixtral", dict(sliding_window=None) | EXPERTS, None), ("qwen2", {}, None), ("granite", dict(attention_multiplier=0.03), None),
    ("nemotron", dict(partial_rotary_factor=0.5), None), ("starcoder2", dict(sliding_window=None), None), ("gemma", {}, None),
    ("stablelm", {}, None), ("olmo", dict(clip_qkv=None), None)])
@torch.no_grad()
def test_real_models_give_the_same_on_the_cache(monkeypatch, kind, settings, positions):
    """Two prompts packed, then tokens of both, against the model by itself on each sequence."""
    _attention_cpu.use(monkeypatch)
    model = build(kind, **settings)
    g = torch.Generator().manual_seed(1)
    sequences = [torch.randint(3, 128, (n,), generator=g) for n in (66, 9)]
    want = [model(s[None], use_cache=False).logits[0] for s in sequences]
    cache = make_cache(4, 2, 32)
    cache.pool.fill_(float("nan"))
    install.install_paged_attention(model, cache, max_positions=positions)
    first = [60, 3]
    step = cache.prompts(first)
    got = [[], []]
    while True:
        begin = [cache.length(s) - (f if step.cu_seqlens is not None else 1) for s, f in zip(step.sequences, first)]
        tokens = torch.cat([s[b:cache.length(i)] for s, b, i in zip(sequences, begin, step.sequences)])
        with cache.running(step):
            logits = model(tokens[None], position_ids=step.positions.long()[None], use_cache=False).logits[0]
        for mine, part in zip(got, logits.split([cache.length(i) - b for i, b in zip(step.sequences, begin)])):
            mine.append(part)
        if cache.length(step.sequences[0]) == 66:
            break
        step = cache.next_token(step.sequences)
    for mine, w in zip(got, want):
        mine = torch.cat(mine)
        assert ((mine - w[:len(mine)]).norm() / w[:len(mine)].norm()).item() < 1e-4


@pytest.mark.parametrize("kind,settings,why", [
    ("mistral", dict(sliding_window=64), "sliding_window of 64"), ("mixtral", dict(sliding_window=64) | EXPERTS, "sliding_window of 64"),
    ("starcoder2", dict(sliding_window=64), "sliding_window of 64"), ("phimoe", dict(sliding_window=64) | EXPERTS, "sliding_window of 64"),
    ("qwen2", dict(use_sliding_window=True, sliding_window=64, max_window_layers=2), "sliding_window"),
    ("cohere", {}, "in halves"), ("glm", {}, "does not compute"), ("ernie4_5", {}, "does not compute"), ("helium", {}, "does not compute"),
    ("hunyuan_v1_dense", {}, "query_layernorm"), ("stablelm", dict(qk_layernorm=True), "q_layernorm"),
    ("smollm3", dict(no_rope_layer_interval=2), "layers.1"), ("olmo", dict(clip_qkv=0.5), "does not compute"),
    ("olmo", dict(clip_qkv=30.0), "does not compute"), ("bitnet", {}, "attn_sub_norm"), ("diffllama", {}, "lambda"),
    ("falcon_h1", {}, "hybrid|state of its own"), ("qwen3", {}, "q_norm")])
def test_real_models_whose_attention_is_another_are_refused(kind, settings, why):
    model = build(kind, **settings)
    with pytest.raises(ValueError, match=why):
        install.install_paged_attention(model, make_cache(4, 2, 32))
    assert not any(isinstance(layer.self_attn, PagedSelfAttention) for layer in install.get_blocks(model))
    if kind in ("cohere", "glm"):                                 # with a table of the caller's, too
        with pytest.raises(ValueError, match="does not compute"):
            install.install_paged_attention(model, make_cache(4, 2, 32), cos_sin=rotary_table(torch.ones(16 if kind == "cohere" else 8), 128))


def test_positions_of_several_parts_are_refused():
    transformers = pytest.importorskip("transformers")
    text = dict(vocab_size=128, hidden_size=128, intermediate_size=96, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=2,
                max_position_embeddings=64, rope_scaling=dict(type="mrope", mrope_section=[8, 12, 12]))
    vision = dict(depth=1, hidden_size=32, intermediate_size=32, num_heads=2, out_hidden_size=128)
    model = transformers.Qwen2_5_VLForConditionalGeneration(transformers.Qwen2_5_VLConfig(text_config=text, vision_config=vision))
    for table in (None, rotary_table(torch.ones(32), 64)):
        with pytest.raises(ValueError, match="mrope_section|in halves|cannot be compared"):
            install.install_paged_attention(model, make_cache(2, 2, 64), cos_sin=table)


def test_a_move_that_fails_leaves_the_table():
    model = TinyLlama()
    install.install_paged_attention(model, make_cache(), cos_sin=rotary_table(torch.ones(32), 8))
    attn = model.model.layers[0].self_attn

    def fails(t):
        raise RuntimeError("out of memory")
    with pytest.raises(RuntimeError):
        attn._apply(fails)
    assert attn.cos_sin.shape == (8, 64) and [n for n, _ in attn.named_buffers()] == ["cos_sin"]


def test_sequences_beyond_the_rotations_table_are_refused(monkeypatch):
    """The kernels would store nothing of their tokens and say so at the next look for errors only."""
    _attention_cpu.use(monkeypatch)
    model, cache = TinyLlama().float(), make_cache()
    install.install_paged_attention(model, cache, cos_sin=rotary_table(torch.ones(32), 8))
    attn, x = model.model.layers[0].self_attn, torch.randn(40, 256)
    cache.pool.zero_()
    step = cache.prompts([9, 2])
    with cache.running(step), pytest.raises(ValueError, match="8 positions"):
        attn(x[:11])
    assert not cache.pool.any()
    step = cache.prompts([7, 8])
    with cache.running(step):
        attn(x[:15])
    with cache.running(cache.next_token(step.sequences[:1])):
        attn(x[:1])                                               # the eighth
    step = cache.next_token(step.sequences[:1])
    with cache.running(step), pytest.raises(ValueError, match="9 tokens"):
        attn(x[:1])
    # a step that is refilled, as a captured forward reads it
    ids = cache.prompts([6, 5]).sequences
    refilled = cache.reserve(2, 16)
    with cache.running(refilled):
        attn(x[:2])
    for _ in range(2):
        cache.next_token(ids, into=refilled)
    free = cache.free_pages
    with pytest.raises(ValueError, match="8 positions"):
        cache.next_token(ids, into=refilled)
    assert [cache.length(i) for i in ids] == [8, 7] and cache.free_pages == free and refilled.longest == 8


def test_a_second_thread_does_not_take_over_the_running_step():
    import copy
    import threading
    cache, seen = make_cache(), []
    one, two = cache.prompts([3]), cache.prompts([4])

    def other():
        try:
            with cache.running(two):
                seen.append("ran")
        except RuntimeError as e:
            seen.append(str(e))

    def run():
        thread = threading.Thread(target=other)
        thread.start()
        thread.join()

    with cache.running(one):
        run()
        assert cache.step is one
        with cache.running(two):                                  # within one thread steps nest
            assert cache.step is two
        assert cache.step is one
        run()
    run()
    assert ["another thread" in s for s in seen] == [True, True, False] and cache.step is None
    assert copy.deepcopy(cache).free_pages == cache.free_pages


@pytest.mark.parametrize("default", [torch.float16, torch.float64, "meta"])
def test_the_callers_defaults_do_not_enter(default):
    model = build("llama")
    before = torch.get_default_dtype()
    try:
        if default == "meta":
            with torch.device("meta"):
                cache = make_cache(4, 2, 32)
                install.install_paged_attention(model, cache, cos_sin=rotary_table(torch.ones(16, device="cpu"), 128))
        else:
            torch.set_default_dtype(default)
            install.install_paged_attention(model, make_cache(4, 2, 32))
            assert torch.get_default_dtype() == default
    finally:
        torch.set_default_dtype(before)
    assert isinstance(model.model.layers[3].self_attn, PagedSelfAttention)
    assert model.config._attn_implementation == "eager"


def test_the_models_config_is_left_alone():
    transformers = pytest.importorskip("transformers")
    config = transformers.AutoConfig.for_model("llama", **SMALL)
    model = transformers.AutoModelForCausalLM.from_config(config, attn_implementation="sdpa").eval()
    install.install_paged_attention(model, make_cache(4, 2, 32))
    assert model.config._attn_implementation == "sdpa"


def test_a_table_that_does_not_fit_the_heads_is_refused():
    for bad in (torch.ones(8, 66), torch.ones(8, 63), torch.ones(8, 0), torch.ones(0, 64), torch.ones(64)):
        model = build("llama", head_dim=64)
        with pytest.raises(ValueError, match="cos_sin must be"):
            install.install_paged_attention(model, make_cache(4, 2, 64), cos_sin=bad)
