"""The paged cache's host bookkeeping, the installer's refusals and the entries' checks, without a GPU."""
import ctypes
import math

import pytest
import torch
from torch import nn

from mindpipe_b200 import _lib, install, ops
from mindpipe_b200.attention import PagedKVCache, PagedSelfAttention, rotary_table
from tests._tiny_llama import TinyLlama


def make(pages=10, page=4, layers=2, heads=2, dim=64):
    return PagedKVCache(layers, pages, page, heads, dim, device="cpu")


def test_prompts_and_tokens_own_their_pages():
    cache = make()
    step = cache.prompts([5, 4, 1])
    assert step.cu_seqlens.tolist() == [0, 5, 9, 10] and step.tokens == 10
    assert step.positions.tolist() == [0, 1, 2, 3, 4, 0, 1, 2, 3, 0]
    assert len(set(step.slots.tolist())) == 10 and cache.free_pages == 6
    owner = {s // 4: q for s, q in zip(step.slots.tolist(), [0] * 5 + [1] * 4 + [2])}
    assert len(owner) == 4                                        # no page of two sequences
    nxt = cache.next_token(step.sequences)
    assert nxt.positions.tolist() == [5, 4, 1] and nxt.seq_lens.tolist() == [6, 5, 2]
    assert cache.free_pages == 5                                  # the second began a page
    for i, (row, slot, at) in enumerate(zip(nxt.page_table.tolist(), nxt.slots.tolist(), nxt.positions.tolist())):
        assert row[at // 4] * 4 + at % 4 == slot
        assert slot not in step.slots.tolist()
        assert all(p == -1 for p in row[-(-(at + 1) // 4):])
    cache.free(step.sequences[:2])
    assert cache.free_pages == 9
    again = cache.prompts([36])
    assert cache.free_pages == 0 and not set(s // 4 for s in again.slots.tolist()) & {nxt.page_table[2, 0].item()}


def test_running_out_of_pages_changes_nothing():
    cache = make(pages=2)
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.prompts([4, 5])
    step = cache.prompts([4, 4])
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.next_token(step.sequences)
    assert [cache.length(s) for s in step.sequences] == [4, 4] and cache.free_pages == 0
    cache.free(step.sequences[:1])
    assert cache.next_token(step.sequences[1:]).seq_lens.tolist() == [5]


def test_a_step_is_refilled_in_place():
    cache = make()
    ids = cache.prompts([3, 2]).sequences
    step = cache.reserve(2, 8)
    assert step.seq_lens.tolist() == [0, 0] and step.slots.tolist() == [-1, -1] and step.page_table.shape == (2, 2)
    held = step.page_table.data_ptr()
    for i in range(5):
        assert cache.next_token(ids, into=step) is step
    assert step.seq_lens.tolist() == [8, 7] and step.page_table.data_ptr() == held
    with pytest.raises(ValueError, match="pages"):
        cache.next_token(ids, into=step)
    assert [cache.length(s) for s in ids] == [8, 7]
    with pytest.raises(ValueError):
        cache.next_token(ids[:1], into=step)
    for bad in ([], [ids[0], ids[0]]):
        with pytest.raises(ValueError):
            cache.next_token(bad)
    with pytest.raises(ValueError):
        cache.prompts([3, 0])


def test_constructor_refusals():
    for kw, error in ((dict(dim=60), ValueError), (dict(dim=136), ValueError), (dict(pages=0), ValueError), (dict(pages=2**30, page=4), ValueError)):
        with pytest.raises(error):
            make(**kw)
    with pytest.raises(TypeError):
        PagedKVCache(1, 1, 1, 1, 64, dtype=torch.float32, device="cpu")


def test_rotary_table_far_positions():
    inv = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    t = rotary_table(inv.float(), 131072, 1.5)
    assert t.shape == (131072, 64) and t.dtype == torch.float32
    for p in (0, 1, 131071):
        for i in (0, 7, 31):
            f = float(inv.float()[i])
            assert abs(t[p, i].item() - 1.5 * math.cos(p * f)) < 2e-7 and abs(t[p, 32 + i].item() - 1.5 * math.sin(p * f)) < 2e-7


def test_installer_refuses_what_it_does_not_do():
    table = rotary_table(torch.ones(32), 8)
    model = TinyLlama()                                           # 256 wide, 128 of keys
    assert install.install_paged_attention(model, make(), cos_sin=table) == ["model.layers.0.self_attn", "model.layers.1.self_attn"]
    assert all(isinstance(layer.self_attn, PagedSelfAttention) for layer in model.model.layers)
    with pytest.raises(RuntimeError, match="no step"):
        model.model.layers[0].self_attn(torch.zeros(1, 256))
    for cache, kw, edit in ((make(layers=3), dict(cos_sin=table), None), (make(heads=4), dict(cos_sin=table), None), (make(), {}, None),
                            (make(), dict(cos_sin=table), "q_norm"), (make(), dict(cos_sin=table), "sliding_window")):
        model = TinyLlama()
        if edit:
            setattr(model.model.layers[1].self_attn, edit, nn.Identity() if edit == "q_norm" else 128)
        with pytest.raises(ValueError):
            install.install_paged_attention(model, cache, **kw)
        assert not any(isinstance(layer.self_attn, PagedSelfAttention) for layer in model.model.layers)


def test_casting_a_model_keeps_the_table():
    model = TinyLlama()
    install.install_paged_attention(model, make(), cos_sin=rotary_table(torch.ones(32), 8))
    model.bfloat16()
    attn = model.model.layers[0].self_attn
    assert attn.cos_sin.dtype == torch.float32 and attn.q_proj.weight.dtype == torch.bfloat16
    assert not any("cos_sin" in name for name in model.state_dict())


def test_attention_ops_reject_cpu_tensors():
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda q: ops.rotary_append_paged(q, x, x, torch.zeros(4, 64), i, i, x[None], x[None]),
                 lambda q: ops.paged_attention_decode(q, x[None], x[None], i[None], i), lambda q: ops.attention_prefill(q, x, x, i)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call(x)
        with pytest.raises(TypeError):
            call([1, 2])


def test_the_c_entries_check_before_they_touch_a_device():
    lib = _lib.load()
    OK_ARG, INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE = 4096, -1, -2, -3, -4      # an address that is never used

    def rows(data=OK_ARG, token=256, head=64):
        return ctypes.byref(_lib.HeadRows(data, token, head))

    def cache(k=OK_ARG, v=OK_ARG, pages=4, heads=2, page=16, **strides):
        c = _lib.PagedCache(k, v, pages, heads, page, 2048, 1024, 64, 2048, 1024, 64)
        for name, value in strides.items():
            setattr(c, name, value)
        return ctypes.byref(c)

    def append(dtype=0, q=None, k=None, v=None, table=OK_ARG, limit=8, rotated=64, pos=OK_ARG, slots=OK_ARG, t=3, hq=4, d=64, c=None,
               out=OK_ARG, k_out=None):
        return lib.mp_rotary_append_paged(dtype, q or rows(), k or rows(), v or rows(), table, limit, rotated, 0, pos, slots, t, hq, d,
                                          c or cache(), out, k_out, None, None)

    for kw, status in ((dict(q=rows(None)), INVALID), (dict(t=0), INVALID), (dict(pos=None), INVALID), (dict(out=None), INVALID),
                       (dict(table=None), INVALID), (dict(limit=0), INVALID), (dict(rotated=0), INVALID), (dict(c=cache(pages=0)), INVALID),
                       (dict(c=cache(v=None)), INVALID), (dict(dtype=2), UNSUPPORTED), (dict(rotated=66), UNSUPPORTED),
                       (dict(rotated=31), UNSUPPORTED), (dict(d=60), UNSUPPORTED), (dict(d=136, rotated=8), UNSUPPORTED),
                       (dict(v=rows(token=-8)), UNSUPPORTED), (dict(k=rows(OK_ARG + 8)), ALIGNMENT), (dict(k=rows(head=60)), ALIGNMENT),
                       (dict(c=cache(k_page_stride=4)), ALIGNMENT), (dict(out=OK_ARG + 2), ALIGNMENT), (dict(k_out=OK_ARG + 2), ALIGNMENT)):
        assert append(**kw) == status, kw

    need = lib.mp_paged_attention_decode_workspace_bytes()

    def decode(dtype=0, q=None, b=3, hq=4, d=64, c=None, table=OK_ARG, pages=2, lens=OK_ARG, out=OK_ARG, ws=OK_ARG, nbytes=need):
        return lib.mp_paged_attention_decode(dtype, q or rows(), b, hq, d, c or cache(), table, pages, lens, 0.1, out, ws, nbytes, None, None)

    for kw, status in ((dict(b=0), INVALID), (dict(pages=0), INVALID), (dict(table=None), INVALID), (dict(lens=None), INVALID),
                       (dict(out=None), INVALID), (dict(hq=3), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED), (dict(d=4), UNSUPPORTED),
                       (dict(ws=None), WORKSPACE), (dict(nbytes=need - 1), WORKSPACE), (dict(out=OK_ARG + 8), ALIGNMENT)):
        assert decode(**kw) == status, kw

    def prefill(dtype=0, q=None, k=None, v=None, t=3, hq=4, hk=2, d=64, cu=OK_ARG, b=1, out=OK_ARG):
        return lib.mp_attention_prefill(dtype, q or rows(), k or rows(), v or rows(), t, hq, hk, d, cu, b, 0.1, out, None, None, None)

    for kw, status in ((dict(t=0), INVALID), (dict(b=0), INVALID), (dict(hk=0), INVALID), (dict(cu=None), INVALID), (dict(hk=3), UNSUPPORTED),
                       (dict(dtype=2), UNSUPPORTED), (dict(d=130), UNSUPPORTED), (dict(q=rows(token=12)), ALIGNMENT),
                       (dict(out=OK_ARG + 8), ALIGNMENT), (dict(k=rows(token=0)), UNSUPPORTED)):
        assert prefill(**kw) == status, kw


def test_bad_bookkeeping_calls_change_nothing():
    cache = make()
    a, b = cache.prompts([5, 9]).sequences
    free = cache.free_pages
    for bad in ([a, a], [a, 99]):
        with pytest.raises(KeyError):
            cache.free(bad)
        assert cache.free_pages == free and cache.length(a) == 5
    with pytest.raises(KeyError):
        cache.next_token([a, 99])
    assert cache.length(a) == 5
    for batch, longest in ((0, 10), (2, 0)):
        with pytest.raises(ValueError):
            cache.reserve(batch, longest)
    cache.free([a, b])


def test_installer_refuses_attention_that_looks_ahead_or_gates():
    table = rotary_table(torch.ones(32), 8)
    for edit in ("is_causal", "o_proj"):
        model = TinyLlama()
        attn = model.model.layers[1].self_attn
        setattr(attn, edit, False if edit == "is_causal" else nn.Linear(128, 256, bias=False))
        with pytest.raises(ValueError):
            install.install_paged_attention(model, make(), cos_sin=table)
        assert not any(isinstance(layer.self_attn, PagedSelfAttention) for layer in model.model.layers)


def test_custom_ops_give_shapes_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from mindpipe_b200.custom_ops import load_and_register
    ns = load_and_register()
    with FakeTensorMode():
        qkv = torch.empty(6, 8 * 64, dtype=torch.bfloat16)
        q, k, v = (x.view(6, -1, 64) for x in qkv.split([256, 128, 128], 1))
        cache, i = torch.empty(3, 2, 16, 64, dtype=torch.bfloat16), torch.empty(6, dtype=torch.int32)
        qr, kr = ns.rotary_append_paged(q, k, v, torch.empty(9, 64), i, i, cache, cache)
        assert qr.shape == q.shape and kr.shape == k.shape and qr.is_contiguous() and qr.dtype == q.dtype
        assert ns.attention_prefill(q, k, v, torch.empty(2, dtype=torch.int32)).shape == q.shape
        out = ns.paged_attention_decode(q, cache, cache, torch.empty(6, 2, dtype=torch.int32), i, 0.5)
        assert out.shape == q.shape and out.is_contiguous()
