"""The attention operators of a decoder layer, as cases that can be timed and compared.

A decoder layer's attention between its quantised linears: the new tokens' queries and keys are rotated by their
positions and keys and values go into a paged cache (``append``), prompts attend within themselves (``prefill``), and
every later token attends to its sequence's pages (``decode``).

``run`` makes the calls of ``mindpipe_b200.ops`` where ``own`` is set and otherwise computes the same in elementary
torch operations with 32-bit arithmetic, rounded once.  ``exact`` is the definition in 64 bits.

A case names its sizes: ``heads`` query heads and ``kv_heads`` heads of keys and values of ``dim`` values, ``page`` tokens
to a page, ``batch`` sequences of ``shortest`` to ``longest`` tokens whose lengths follow from ``pattern`` (spread over
their logarithm; the first is the longest), and for prompts ``behind`` rows of the batch that belong to no sequence.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_SPARE_PAGES = 3            # pages that no sequence owns


def listed():
    return [
        # one decode step's new tokens (8B-shaped heads): latency
        {"name": "append_8b_t16", "op": "append", "type": "fp16", "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128,
         "interleaved": False, "page": 16, "tokens": 16, "padding": 0, "far": 8000, "keys_out": False},
        # a padded decode batch: odd head counts, half of each head rotated, neighbours paired, far positions
        {"name": "append_d64_t333_padded", "op": "append", "type": "bf16", "heads": 21, "kv_heads": 3, "dim": 64, "rotated": 32,
         "interleaved": True, "page": 24, "tokens": 333, "padding": 13, "far": 130000, "keys_out": False},
        # a long prompt (70B-shaped heads), whose attention wants the rotated keys too
        {"name": "append_70b_t8192", "op": "append", "type": "fp16", "heads": 64, "kv_heads": 8, "dim": 128, "rotated": 128,
         "interleaved": False, "page": 64, "tokens": 8192, "padding": 0, "far": 8192, "keys_out": True},
        # one sequence early in its answer: latency
        {"name": "decode_8b_b1_len300", "op": "decode", "type": "fp16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "batch": 1, "shortest": 300, "longest": 300, "pattern": 0},
        # a serving batch of mixed lengths, grouped heads
        {"name": "decode_8b_b64_mixed", "op": "decode", "type": "fp16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "batch": 64, "shortest": 20, "longest": 8192, "pattern": 1},
        # every head with keys of its own (7B-shaped)
        {"name": "decode_7b_b16_len4096", "op": "decode", "type": "fp16", "heads": 32, "kv_heads": 32, "dim": 128, "page": 32,
         "batch": 16, "shortest": 4096, "longest": 4096, "pattern": 0},
        # few sequences with long contexts (70B-shaped)
        {"name": "decode_70b_b3_long", "op": "decode", "type": "bf16", "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "batch": 3, "shortest": 50001, "longest": 131000, "pattern": 2},
        # many short sequences, small heads, an odd group
        {"name": "decode_d64_b301_short", "op": "decode", "type": "bf16", "heads": 35, "kv_heads": 5, "dim": 64, "page": 8,
         "batch": 301, "shortest": 1, "longest": 700, "pattern": 3},
        # a handful of chat turns packed into one batch
        {"name": "prefill_8b_short_turns", "op": "prefill", "type": "fp16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 9,
         "shortest": 1, "longest": 300, "pattern": 4, "behind": 0},
        # one prompt of the length the prefill linears are measured at (7B-shaped)
        {"name": "prefill_7b_t2048", "op": "prefill", "type": "fp16", "heads": 32, "kv_heads": 32, "dim": 128, "batch": 1,
         "shortest": 2048, "longest": 2048, "pattern": 0, "behind": 0},
        # ragged prompts with small heads in a padded batch
        {"name": "prefill_d64_ragged", "op": "prefill", "type": "bf16", "heads": 30, "kv_heads": 6, "dim": 64, "batch": 12,
         "shortest": 33, "longest": 5001, "pattern": 5, "behind": 77},
        # a long document (70B-shaped)
        {"name": "prefill_70b_t8192", "op": "prefill", "type": "bf16", "heads": 64, "kv_heads": 8, "dim": 128, "batch": 1,
         "shortest": 8192, "longest": 8192, "pattern": 0, "behind": 0},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    case = {"op": op, "type": rng.choice(["fp16", "bf16"]), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim}
    if op == "append":
        tokens = _log_uniform(rng, 1, 8192)
        case.update(rotated=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, page=rng.choice([8, 16, 24, 64, 256]),
                    tokens=tokens, padding=rng.choice([0, 0, min(5, tokens - 1)]), far=_log_uniform(rng, 8192, 140000),
                    keys_out=rng.random() < 0.5)
    elif op == "decode":
        batch = _log_uniform(rng, 1, 300)
        longest = _log_uniform(rng, 1, max(2, min(120000, 380000 // batch)))
        case.update(page=rng.choice([8, 16, 24, 64, 256]), batch=batch, shortest=_log_uniform(rng, 1, longest), longest=longest,
                    pattern=rng.randrange(10, 10000))
    else:
        batch = _log_uniform(rng, 1, 40)
        longest = _log_uniform(rng, 1, int(8192 / math.sqrt(batch)))
        case.update(batch=batch, shortest=_log_uniform(rng, 1, longest), longest=longest, pattern=rng.randrange(10, 10000),
                    behind=rng.choice([0, 0, 9]))
    return case


def _lengths(case):
    rng = random.Random(case["pattern"])
    return [case["longest"]] + [_log_uniform(rng, case["shortest"], case["longest"]) for _ in range(case["batch"] - 1)]


def work(case):
    h, hk, d, size = case["heads"], case["kv_heads"], case["dim"], 2
    if case["op"] == "append":
        t, live = case["tokens"], case["tokens"] - case["padding"]
        rows = t * (2 * h + hk) + live * (hk + 2 * hk) + (t * hk if case["keys_out"] else 0)
        return {"bytes": rows * d * size + t * (4 * case["rotated"] + 8), "flops": 3 * t * (h + hk) * case["rotated"]}
    total = sum(_lengths(case))
    if case["op"] == "decode":
        pages = sum(-(-n // case["page"]) for n in _lengths(case))
        return {"bytes": (2 * total * hk + 2 * case["batch"] * h) * d * size + 4 * pages + 4 * case["batch"], "flops": 4 * h * d * total}
    pairs = sum(n * (n + 1) // 2 for n in _lengths(case))
    return {"bytes": (2 * h + 2 * hk) * d * size * total + 4 * case["batch"] + 4, "flops": 4 * h * d * pairs}


def _pool(case, pages, gen):
    """A cache's keys or values, as left by earlier sequences where no present one has written."""
    return torch.randn(pages, case["kv_heads"], case["page"], case["dim"], generator=gen, device="cuda",
                       dtype=_DTYPES[case["type"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    rng = random.Random(seed)
    dtype, h, hk, d = _DTYPES[case["type"]], case["heads"], case["kv_heads"], case["dim"]
    state = {"case": case}

    def qkv(rows):
        # what the concatenated projection of a layer gives; keys have channels of larger mean, as trained ones do
        x = torch.randn(rows, (h + 2 * hk) * d, generator=gen, device="cuda")
        bias = torch.randn(hk * d, generator=gen, device="cuda")
        x[:, h * d:(h + hk) * d] += bias * (bias.abs() > 1.5)
        x = x.to(dtype)
        q, k, v = x.split([h * d, hk * d, hk * d], dim=1)
        state.update(q=q.view(rows, h, d), k=k.view(rows, hk, d), v=v.view(rows, hk, d))

    if case["op"] == "append":
        t, page, half = case["tokens"], case["page"], case["rotated"] // 2
        qkv(t)
        frequency = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angle = torch.arange(case["far"], dtype=torch.float64, device="cuda")[:, None] * frequency
        pages = -(-t // page) + _SPARE_PAGES
        # tokens in order within pages of the pool in any order; the last page of the pool is nobody's
        order = list(range(pages - 1))
        rng.shuffle(order)
        order = torch.tensor(order, dtype=torch.int64, device="cuda")
        at = torch.arange(t, device="cuda")
        slots = order[at // page] * page + at % page
        if case["padding"]:
            slots[t - case["padding"]:] = -1
        # a prompt's tokens follow one another, a decode step's are anywhere in their sequences
        positions = at + rng.randrange(case["far"] - t + 1) if case["keys_out"] else \
            torch.randint(0, case["far"], (t,), generator=gen, device="cuda")
        state.update(cos_sin=torch.cat([angle.cos(), angle.sin()], dim=1).float(), positions=positions.int(), slots=slots.int(),
                     k_cache=_pool(case, pages, gen), v_cache=_pool(case, pages, gen))
        return state

    lengths = _lengths(case)
    state["lengths"] = lengths
    if case["op"] == "decode":
        page = case["page"]
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + _SPARE_PAGES
        order = torch.randperm(pages, generator=gen, device="cuda").int()
        table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)      # -1: pages not handed out yet
        order_host, used = order.cpu(), 0
        for row, n in zip(table, need):
            row[:n] = order_host[used:used + n]
            used += n
        qkv(len(lengths))
        state.update(page_table=table.cuda(), seq_lens=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                     k_cache=_pool(case, pages, gen), v_cache=_pool(case, pages, gen))
        return state

    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    qkv(ends[-1] + case["behind"])
    state.update(ends=ends, cu_seqlens=torch.tensor(ends, dtype=torch.int32, device="cuda"))
    if case["behind"]:
        state["out"] = torch.randn(ends[-1] + case["behind"], h, d, generator=gen, device="cuda", dtype=dtype)
    return state


# ------------------------------------------------------------------------------------------------------ plain form
def _rotate(x, cos, sin, rotated, interleaved):
    x = x.float()
    turn, rest = x[..., :rotated], x[..., rotated:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if interleaved else turn.chunk(2, dim=-1)
    cos, sin = cos[:, None], sin[:, None]
    a, b = a * cos - b * sin, b * cos + a * sin
    turn = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([turn, rest], dim=-1)


def _plain_append(s):
    case, dtype = s["case"], s["q"].dtype
    page, (cos, sin) = case["page"], s["cos_sin"][s["positions"].long()].chunk(2, dim=1)
    q = _rotate(s["q"], cos, sin, case["rotated"], case["interleaved"]).to(dtype)
    k = _rotate(s["k"], cos, sin, case["rotated"], case["interleaved"]).to(dtype)
    live = (s["slots"] >= 0)[:, None, None]
    slot = torch.where(s["slots"] >= 0, s["slots"].long(), s["k_cache"].shape[0] * page - 1)    # the last page is nobody's
    for cache, new in ((s["k_cache"], k), (s["v_cache"], s["v"])):
        cache[slot // page, :, slot % page] = torch.where(live, new, cache[slot // page, :, slot % page])
    return [q, s["k_cache"], s["v_cache"]] + ([k] if case["keys_out"] else [])


def _attend(q, k, v, scale, masked=None):
    """q [kv heads, rows, dim] over k, v [kv heads, keys, dim], 32 bits."""
    p = torch.matmul(q, k.transpose(1, 2)).mul_(scale)
    if masked is not None:
        p.masked_fill_(masked, float("-inf"))
    p.sub_(p.amax(dim=-1, keepdim=True)).exp_()
    return torch.matmul(p, v).div_(p.sum(dim=-1, keepdim=True))


def _plain_decode(s):
    q, (h, d) = s["q"], s["q"].shape[1:]
    hk, page = s["k_cache"].shape[1], s["k_cache"].shape[2]
    out = torch.empty_like(q)
    for i, n in enumerate(s["lengths"]):
        ids = s["page_table"][i, :-(-n // page)].long()
        k, v = (c[ids].transpose(0, 1).reshape(hk, -1, d)[:, :n].float() for c in (s["k_cache"], s["v_cache"]))
        out[i] = _attend(q[i].float().view(hk, h // hk, d), k, v, d ** -0.5).view(h, d).to(q.dtype)
    return out


def _plain_prefill(s):
    q, k, v = s["q"], s["k"], s["v"]
    (h, d), hk = q.shape[1:], k.shape[1]
    group = h // hk
    out = s["out"] if "out" in s else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    for begin, end in zip(s["ends"], s["ends"][1:]):
        step = max(1, (1 << 28) // (h * (end - begin)))
        for lo in range(begin, end, step):
            hi = min(lo + step, end)
            rows = q[lo:hi].float().view(hi - lo, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * (hi - lo), d)
            keys, values = (t[begin:hi].float().transpose(0, 1) for t in (k, v))
            later = torch.arange(begin, hi, device=q.device)[None] > torch.arange(lo, hi, device=q.device)[:, None]
            o = _attend(rows, keys, values, d ** -0.5, later.repeat(group, 1))
            out[lo:hi] = o.view(hk, group, hi - lo, d).permute(2, 0, 1, 3).reshape(hi - lo, h, d).to(q.dtype)
    return out


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[case["op"]](state)
    from mindpipe_b200 import ops
    if case["op"] == "append":
        q, k = ops.rotary_append_paged(state["q"], state["k"], state["v"], state["cos_sin"], state["positions"], state["slots"],
                                       state["k_cache"], state["v_cache"], interleaved=case["interleaved"],
                                       want_k=case["keys_out"])
        return [q, state["k_cache"], state["v_cache"]] + ([k] if case["keys_out"] else [])
    if case["op"] == "decode":
        return ops.paged_attention_decode(state["q"], state["k_cache"], state["v_cache"], state["page_table"], state["seq_lens"])
    return ops.attention_prefill(state["q"], state["k"], state["v"], state["cu_seqlens"], out=state.get("out"))


# -------------------------------------------------------------------------------------------------- the definition
def _softmax_average(scores, values):
    """Rows of scores (minus infinity: not attended to) and the values they weigh, 64 bits."""
    weights = torch.exp(scores - scores.max(dim=-1, keepdim=True).values)
    return torch.einsum("hqk,hkd->hqd", weights, values) / weights.sum(dim=-1)[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        n, page, half = case["tokens"], case["page"], case["rotated"] // 2
        row = s["cos_sin"].double()[s["positions"].long()]
        turn = torch.complex(row[:, :half], row[:, half:])

        def rotate(x):
            y = x.double().clone()
            first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else \
                (slice(0, half), slice(half, 2 * half))
            z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
            y[..., first], y[..., second] = z.real, z.imag
            return y

        q, k = rotate(s["q"]), rotate(s["k"])
        caches = []
        at = s["slots"].tolist()
        kept = [i for i in range(n) if at[i] >= 0]
        where = torch.tensor([at[i] for i in kept], device="cuda")
        for cache, new in ((s["k_cache"], k), (s["v_cache"], s["v"].double())):
            by_slot = cache.double().transpose(1, 2).reshape(-1, hk, d)
            by_slot[where] = new[kept]
            caches.append(by_slot.view(-1, page, hk, d).transpose(1, 2).contiguous())
        return [q, *caches] + ([k] if case["keys_out"] else [])
    if case["op"] == "decode":
        out = torch.empty(case["batch"], h, d, dtype=torch.float64, device="cuda")
        for i, n in enumerate(s["lengths"]):
            slot = torch.arange(n, device="cuda")
            ids = s["page_table"][i].long()[slot // case["page"]]
            for j in range(hk):
                keys, values = (s[c][ids, j, slot % case["page"]].double() for c in ("k_cache", "v_cache"))
                mine = s["q"][i, j * (h // hk):(j + 1) * (h // hk)].double()
                out[i, j * (h // hk):(j + 1) * (h // hk)] = _softmax_average((mine @ keys.T / math.sqrt(d))[None], values[None])[0]
        return out
    out = s["out"].double() if "out" in s else torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for begin, end in zip(s["ends"], s["ends"][1:]):
        for j in range(h):
            q, k, v = s["q"][begin:end, j].double(), s["k"][begin:end, j // (h // hk)].double(), s["v"][begin:end, j // (h // hk)].double()
            for lo in range(0, end - begin, 2048):
                rows = q[lo:lo + 2048]
                scores = rows @ k.T / math.sqrt(d)
                ahead = torch.ones(scores.shape, dtype=torch.bool, device="cuda").triu(diagonal=lo + 1)
                out[begin + lo:begin + lo + rows.shape[0], j] = _softmax_average(scores.masked_fill(ahead, -math.inf)[None], v[None])[0]
    return out
