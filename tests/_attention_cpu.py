"""The three attention operators in plain torch, for tests of what calls them on a machine without a GPU."""
import torch

from mindpipe_b200 import attention
from tests import _attention_ref as ref


class _Plain:
    @staticmethod
    def rotary_append_paged(q, k, v, cos_sin, positions, slots, k_cache, v_cache, *, interleaved=False, want_k=False):
        q, k = (ref.rotate(x, cos_sin, positions, interleaved)[0].to(x.dtype) for x in (q, k))
        page = k_cache.shape[2]
        for t, slot in enumerate(slots.tolist()):
            if slot >= 0:
                k_cache[slot // page, :, slot % page], v_cache[slot // page, :, slot % page] = k[t], v[t]
        return q, k if want_k else None

    @staticmethod
    def paged_attention_decode(q, k_cache, v_cache, page_table, seq_lens, *, scale=None, out=None):
        return ref.decode(q, k_cache, v_cache, page_table, seq_lens.tolist(), scale)[0].to(q.dtype)

    @staticmethod
    def attention_prefill(q, k, v, cu_seqlens, *, scale=None, out=None):
        return ref.prefill(q, k, v, cu_seqlens.tolist(), scale)[0].to(q.dtype)


def use(monkeypatch):
    monkeypatch.setattr(attention, "ops", _Plain)
