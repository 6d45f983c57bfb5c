"""A decoder layer's attention between its quantised linears: a paged cache and the module that runs on it.

* :class:`PagedKVCache` -- keys and values of all layers in pages of one pool, and the host's record of which pages belong
  to which sequence.  It turns "these prompts" or "one token more for these sequences" into a :class:`Step`: the index
  tensors that the kernels of :mod:`mindpipe_b200.ops` read.
* :class:`PagedSelfAttention` -- stands where a llama-like layer has its ``self_attn``: the layer's own projections
  (quantised or not), rotation and append in one launch, then attention over the prompts or over the pages.

The reference leaves this part to its runtime (``npu_fused_infer_attention_score``,
acceleration/runtime_patches/vllm_ascend.patch:141-291).  ``mindpipe_b200.install.install_paged_attention`` puts the module
into a model.
"""
from __future__ import annotations

import threading
from contextlib import contextmanager
from dataclasses import dataclass

import torch
from torch import nn

from . import ops

_entry = threading.Lock()        # of running(), for all caches: a cache can be copied with its model


def rotary_table(inv_freq: torch.Tensor, max_positions: int, scaling: float = 1.0) -> torch.Tensor:
    """``[max_positions, 2 * len(inv_freq)]`` fp32 table of :func:`ops.rotary_append_paged`: cosines, then sines.

    Angles are taken in 64 bits: in 32 a position beyond 10^5 is off by up to 0.008.
    """
    angle = torch.arange(max_positions, dtype=torch.float64, device=inv_freq.device)[:, None] * inv_freq.double()
    return torch.cat([angle.cos() * scaling, angle.sin() * scaling], dim=1).float().contiguous()


@dataclass
class Step:
    """One forward's tokens, in the order the model sees them: whole prompts (``cu_seqlens``), or one token of each
    sequence (``page_table``, ``seq_lens``)."""
    sequences: list[int]
    positions: torch.Tensor                  # int32 [tokens]
    slots: torch.Tensor                      # int32 [tokens]
    cu_seqlens: torch.Tensor | None = None   # int32 [sequences + 1]
    page_table: torch.Tensor | None = None   # int32 [sequences, pages]
    seq_lens: torch.Tensor | None = None     # int32 [sequences]
    longest: int = 0                         # tokens of the longest sequence, as the host knows it; 0: it does not
    positions_limit: int | None = None       # of the tables that forwards have used with this step

    @property
    def tokens(self) -> int:
        return self.positions.shape[0]


class PagedKVCache:
    """Pages of ``page_size`` tokens for the keys and values of ``num_layers`` layers.

    ``prompts(lengths)`` takes pages for new sequences and returns their :class:`Step`; ``next_token(sequences)`` adds one
    token to each; ``free(sequences)`` gives the pages back.  ``running(step)`` makes a step the one that the attached
    modules run::

        step = cache.prompts([len(a), len(b)])
        with cache.running(step):
            model(torch.cat([a, b])[None], position_ids=step.positions.long()[None], use_cache=False)
        step = cache.next_token(step.sequences)

    The bookkeeping is host code; running out of pages raises ``RuntimeError`` and changes nothing.  A step with a sequence
    longer than the rotation's table raises ``ValueError`` in the forward, before anything is stored.  A cache is one thread's:
    neither its bookkeeping nor its running step is shared (a second thread that runs a step meanwhile is refused).
    """

    def __init__(self, num_layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        if min(num_layers, num_pages, page_size, kv_heads) < 1:
            raise ValueError("layers, pages, page size and heads must be positive")
        if num_pages * page_size > 2**31 - 1:
            raise ValueError("slots are 32-bit: num_pages * page_size must be below 2^31")
        if head_dim % 8 or not 8 <= head_dim <= 128:
            raise ValueError("head_dim must be a multiple of 8 up to 128")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("the cache holds float16 or bfloat16")
        self.num_pages, self.page_size = num_pages, page_size
        self.pool = torch.empty((num_layers, 2, num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next_id = 0
        self.step: Step | None = None
        self._runner: int | None = None          # the thread whose step it is

    def layer(self, index: int) -> tuple[torch.Tensor, torch.Tensor]:
        """``k_cache, v_cache`` of a layer: ``[pages, kv_heads, page_size, head_dim]`` each."""
        return self.pool[index, 0], self.pool[index, 1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._length[sequence]

    def _take(self, wanted: int) -> list[int]:
        if wanted > len(self._free):
            raise RuntimeError(f"the cache is out of pages: {wanted} wanted, {len(self._free)} free")
        taken = [self._free.pop() for _ in range(wanted)]
        return taken

    def _tensor(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.pool.device)

    def prompts(self, lengths) -> Step:
        """New sequences of these many tokens, to be run packed one behind the other."""
        lengths = [int(n) for n in lengths]
        if not lengths or min(lengths) < 1:
            raise ValueError("a prompt has at least one token")
        need = [-(-n // self.page_size) for n in lengths]
        pages = self._take(sum(need))
        ids, positions, slots, ends = [], [], [], [0]
        for n, count in zip(lengths, need):
            own, pages = pages[:count], pages[count:]
            ids.append(self._next_id)
            self._pages[self._next_id], self._length[self._next_id] = own, n
            self._next_id += 1
            positions.extend(range(n))
            slots.extend(own[i // self.page_size] * self.page_size + i % self.page_size for i in range(n))
            ends.append(ends[-1] + n)
        return Step(ids, self._tensor(positions), self._tensor(slots), cu_seqlens=self._tensor(ends), longest=max(lengths))

    def next_token(self, sequences, into: Step | None = None) -> Step:
        """One token more for each of the sequences.

        ``into``: an earlier step of as many sequences, whose tensors are written instead of new ones, on the current stream -- a
        captured forward then runs the new step when replayed there.  Its table keeps its width: sequences that outgrow it raise ``ValueError``
        (:meth:`reserve` makes a wider one), and so do sequences that outgrow the rotation's table of the forward."""
        sequences = list(sequences)
        if len(set(sequences)) != len(sequences):
            raise ValueError("a sequence may appear once in a step")
        if not sequences:
            raise ValueError("a step has at least one sequence")
        grow = [s for s in sequences if self._length[s] % self.page_size == 0]
        width = max(len(self._pages[s]) + (s in grow) for s in sequences)
        if into is not None:
            if into.page_table is None or into.page_table.shape[0] != len(sequences):
                raise ValueError("into must be a step of as many sequences")
            if into.page_table.shape[1] < width:
                raise ValueError(f"a sequence has {width} pages, the step's table room for {into.page_table.shape[1]}")
            width = into.page_table.shape[1]
        longest = max(self._length[s] for s in sequences) + 1
        if into is not None and into.positions_limit is not None and longest > into.positions_limit:
            raise ValueError(f"a sequence has {longest} tokens, the rotation's table of the step's forwards {into.positions_limit} positions")
        for s, page in zip(grow, self._take(len(grow))):
            self._pages[s].append(page)
        positions, slots, lens, table = [], [], [], []
        for s in sequences:
            at = self._length[s]
            self._length[s] = at + 1
            positions.append(at)
            slots.append(self._pages[s][at // self.page_size] * self.page_size + at % self.page_size)
            lens.append(at + 1)
            table.append(self._pages[s] + [-1] * (width - len(self._pages[s])))
        if into is None:
            return Step(sequences, self._tensor(positions), self._tensor(slots), page_table=self._tensor(table),
                        seq_lens=self._tensor(lens), longest=longest)
        for name, values in (("positions", positions), ("slots", slots), ("page_table", table), ("seq_lens", lens)):
            getattr(into, name).copy_(torch.tensor(values, dtype=torch.int32))
        into.sequences, into.longest = sequences, longest
        return into

    def reserve(self, batch: int, longest: int) -> Step:
        """An empty step of ``batch`` sequences of up to ``longest`` tokens for :meth:`next_token`'s ``into``: no token of it
        is stored and its rows attend to nothing until it is filled."""
        if batch < 1 or longest < 1:
            raise ValueError("a step has at least one sequence, of at least one token")
        width = -(-longest // self.page_size)
        return Step([], self._tensor([0] * batch), self._tensor([-1] * batch), page_table=self._tensor([[-1] * width] * batch),
                    seq_lens=self._tensor([0] * batch))

    def free(self, sequences) -> None:
        sequences = list(sequences)
        if len(set(sequences)) != len(sequences) or not all(s in self._pages for s in sequences):
            raise KeyError(f"not all of {sequences} are sequences of this cache, each once")
        for s in sequences:
            self._free.extend(reversed(self._pages.pop(s)))
            del self._length[s]

    @contextmanager
    def running(self, step: Step):
        """The attached modules' forwards belong to ``step``.  One thread at a time: a second one raises ``RuntimeError``."""
        me = threading.get_ident()
        with _entry:
            if self._runner not in (None, me):
                raise RuntimeError("another thread is running a step of this cache")
            before, self.step, self._runner = (self.step, self._runner), step, me
        try:
            yield step
        finally:
            with _entry:
                self.step, self._runner = before


class PagedSelfAttention(nn.Module):
    """Self-attention of one layer on a :class:`PagedKVCache`, with the projections of the module it replaces.

    ``forward(hidden_states, ...)`` takes the packed tokens of the cache's running step, in any leading shape, and returns
    ``(output, None)`` as the replaced modules do; masks, position embeddings and caches that a model passes along are not
    used.
    """

    def __init__(self, attention: nn.Module, cache: PagedKVCache, layer: int, cos_sin: torch.Tensor, *,
                 head_dim: int | None = None, scale: float | None = None, interleaved: bool = False):
        super().__init__()
        for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
            if not hasattr(attention, name):
                raise ValueError(f"the attention module has no {name}")
            setattr(self, name, getattr(attention, name))
        self.head_dim = int(head_dim if head_dim is not None else cache.pool.shape[-1])
        if self.head_dim != cache.pool.shape[-1]:
            raise ValueError(f"heads of {self.head_dim} values, the cache holds {cache.pool.shape[-1]}")
        for name in ("k_proj", "v_proj"):
            width = getattr(self, name).out_features
            if width != cache.pool.shape[3] * self.head_dim:
                raise ValueError(f"{name} gives {width} values, the cache holds {cache.pool.shape[3]} heads of {self.head_dim}")
        if self.o_proj.in_features != self.q_proj.out_features:
            raise ValueError(f"q_proj gives {self.q_proj.out_features} values, o_proj takes {self.o_proj.in_features}")
        if self.q_proj.out_features % (cache.pool.shape[3] * self.head_dim):
            raise ValueError("the query heads are not a multiple of the key heads")
        self.layer_idx, self.scale, self.interleaved = layer, scale, interleaved
        self.cache = cache
        self.register_buffer("cos_sin", cos_sin, persistent=False)

    def _apply(self, fn, *args, **kwargs):
        table = self._buffers.pop("cos_sin")             # moved with the module, never cast
        try:
            super()._apply(fn, *args, **kwargs)
        finally:
            self._buffers["cos_sin"] = table
        self._buffers["cos_sin"] = table.to(fn(torch.empty(0, dtype=torch.float32, device=table.device)).device)
        return self

    @torch.no_grad()
    def forward(self, hidden_states: torch.Tensor, *args, **kwargs):
        step = self.cache.step
        if step is None:
            raise RuntimeError("no step is running: call the model within cache.running(step)")
        lead = hidden_states.shape[:-1]
        tokens = hidden_states.numel() // hidden_states.shape[-1]
        if tokens != step.tokens:
            raise ValueError(f"the running step has {step.tokens} tokens, the input {tokens}")
        limit = self.cos_sin.shape[0]
        if step.longest > limit:
            raise ValueError(f"a sequence has {step.longest} tokens, the rotation's table {limit} positions")
        step.positions_limit = limit if step.positions_limit is None else min(limit, step.positions_limit)
        x = hidden_states.reshape(tokens, -1)
        q, k, v = (proj(x).view(tokens, -1, self.head_dim) for proj in (self.q_proj, self.k_proj, self.v_proj))
        k_cache, v_cache = self.cache.layer(self.layer_idx)
        prompt = step.cu_seqlens is not None
        q, k = ops.rotary_append_paged(q, k, v, self.cos_sin, step.positions, step.slots, k_cache, v_cache,
                                       interleaved=self.interleaved, want_k=prompt)
        if prompt:
            out = ops.attention_prefill(q, k, v, step.cu_seqlens, scale=self.scale)
        else:
            out = ops.paged_attention_decode(q, k_cache, v_cache, step.page_table, step.seq_lens, scale=self.scale)
        return self.o_proj(out.view(tokens, -1)).view(*lead, -1), None
