"""Calls at the edges of what the attention operators' documentation allows, against the 64-bit statements."""
import pytest
import torch

from mindpipe_b200 import _lib, ops
from tests import _attention_ref as ref
from tests.test_attention_gpu import TYPES, heads, paged, randn, table

pytestmark = pytest.mark.gpu


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,hk,d", [(4, 2, 128), (3, 3, 64), (8, 1, 40)])
def test_prefill_more_sequences_than_are_sorted(h, hk, d, dtype):
    lens = [(37 * i) % 150 for i in range(297)] + [400, 0, 1]
    ends = [0]
    for n in lens:
        ends.append(ends[-1] + n)
    q, k, v = heads(ends[-1], h, hk, d, dtype, seed=d)
    got = ops.attention_prefill(q, k, v, i32(*ends))
    want, tol = ref.prefill(q, k, v, ends)
    ref.assert_close(got, want, tol)
    ops.check_device_errors()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,hk,d,page", [(6, 6, 128, 16), (32, 2, 128, 8), (40, 1, 128, 16), (48, 3, 64, 32), (5, 5, 128, 5)])
def test_decode_many_short_and_some_longer(h, hk, d, page, dtype):
    """Warps that take a short sequence alone beside teams, with a number of heads that is no multiple of four."""
    lens = [(11 * i) % 128 + 1 for i in range(330)] + [0, 127, 128, 129, 130, 1500, 2]
    args = paged(lens, h, hk, d, page, dtype, seed=d + h)
    want, tol = ref.decode(*args[:4], lens)
    ref.assert_close(ops.paged_attention_decode(*args), want, tol)
    ops.check_device_errors()


def many_small_weights(keys, d, steps):
    """A first key `steps` powers of two above all the others, whose values alone are not zero."""
    q, k, v = (torch.zeros(keys, 1, d, dtype=torch.float16, device="cuda") for _ in range(3))
    q[:, :, 0], k[0, :, 0], v[1:] = 1.0, steps, 1.0
    return q, k, v, 0.6931471805599453


def test_many_weights_below_the_types_bits_count():
    """30000 weights of 2^-24.6 are 0.12 % of the row: in fp16 without a shift each would round to 2^-24."""
    keys, d, page = 30001, 64, 16
    q, k, v, scale = many_small_weights(keys, d, 24.59375)
    pages = -(-keys // page)
    kc, vc = (torch.zeros(pages, 1, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
    kc.view(-1, d)[:keys], vc.view(-1, d)[:keys] = k[:, 0], v[:, 0]      # (one head: the pages are the keys' rows)
    rows = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    want, tol = ref.decode(q[:1], kc, vc, rows, [keys], scale)
    ref.assert_close(ops.paged_attention_decode(q[:1], kc, vc, rows, i32(keys), scale=scale), want, tol)
    keys = 6000
    want, tol = ref.prefill(q[:keys], k[:keys], v[:keys], [0, keys], scale)
    ref.assert_close(ops.attention_prefill(q[:keys], k[:keys], v[:keys], i32(0, keys), scale=scale), want, tol)


def test_results_may_replace_the_queries():
    lens = [700, 20, 0, 131]
    q, kc, vc, rows, n = paged(lens, 8, 2, 128, 16, torch.float16, seed=3)
    q = q.contiguous()
    want = ops.paged_attention_decode(q, kc, vc, rows, n)
    assert ops.paged_attention_decode(q, kc, vc, rows, n, out=q).data_ptr() == q.data_ptr() and torch.equal(q, want)
    q, k, v = (x.contiguous() for x in heads(900, 8, 2, 128, torch.bfloat16, 4))
    cu = i32(0, 300, 301, 900)
    want = ops.attention_prefill(q, k, v, cu)
    assert ops.attention_prefill(q, k, v, cu, out=q).data_ptr() == q.data_ptr() and torch.equal(q, want)


def test_overlapping_operands_are_refused():
    room = randn(3, 64, 2, 64)
    q, k, v = room
    flat = room.view(-1)
    part = flat[64:64 + q.numel()].view_as(q)                     # a row further on than q
    cu = i32(0, 64)
    for out in (k, v, part):
        with pytest.raises(ValueError, match="overlaps"):
            ops.attention_prefill(q, k, v, cu, out=out)
    kc, vc = randn(2, 4, 2, 16, 64, seed=1)
    pos = i32(0, 1)
    with pytest.raises(ValueError, match="overlaps"):
        ops.paged_attention_decode(q[:2], kc, vc, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), i32(1, 1), out=kc.view(-1, 2, 64)[:2])
    with pytest.raises(ValueError, match="same memory"):
        ops.rotary_append_paged(q[:2], k[:2], v[:2], table(8, 64), pos, pos, kc, kc)
    with pytest.raises(ValueError, match="share memory"):
        ops.rotary_append_paged(q[:2], k[:2], v[:2], table(8, 64), pos, pos, kc[:1].expand(4, -1, -1, -1), vc)
    ops.check_device_errors()


def test_decode_refuses_lists_beyond_32_bits():
    """256 heads on a sequence of 2^31 tokens (one page, named two million times) would be a list of 2^33 steps."""
    page, hk = 1024, 256
    kc, vc = (torch.zeros(1, hk, page, 8, dtype=torch.float16, device="cuda") for _ in range(2))
    rows = torch.zeros(1, (1 << 31) // page, dtype=torch.int32, device="cuda")
    ops.paged_attention_decode(torch.zeros(1, hk, 8, dtype=torch.float16, device="cuda"), kc, vc, rows, i32(0x7fffff00))
    with pytest.raises(_lib.MindPipeKernelError, match="out of range"):
        ops.check_device_errors()


def test_streams_at_once(new_stream):
    """The same calls on two streams side by side, many times: each stream has a workspace of its own."""
    cases = []
    for seed, lens in ((1, [3000, 5, 900]), (2, [40] * 30 + [2500])):
        args = paged(lens, 16, 4, 128, 16, torch.bfloat16, seed=seed)
        q, k, v = heads(1200, 8, 4, 64, torch.float16, seed)
        cases.append((args, (q, k, v, i32(0, 500, 1200)), new_stream()))
    torch.cuda.synchronize()
    alone = []
    for args, prompt, stream in cases:
        with torch.cuda.stream(stream):
            alone.append((ops.paged_attention_decode(*args), ops.attention_prefill(*prompt)))
        stream.synchronize()
    made = []
    for _ in range(20):
        for args, prompt, stream in cases:
            with torch.cuda.stream(stream):
                made.append((ops.paged_attention_decode(*args), ops.attention_prefill(*prompt)))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(made):
        assert torch.equal(a, alone[i % 2][0]) and torch.equal(b, alone[i % 2][1])
    ops.check_device_errors()


def test_captured_prompt_and_token_follow_their_tensors(new_stream):
    """Rotation with append, prompts and one token in a graph, replayed with other positions, slots, ends and values."""
    d, h, hk, page = 64, 4, 2, 16
    stream = new_stream()
    kc, vc = (torch.zeros(12, hk, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
    q, k, v = (x.contiguous() for x in heads(100, h, hk, d, torch.float16, 7))
    cs, pos, slots, cu = table(200, d), torch.zeros(100, dtype=torch.int32, device="cuda"), torch.zeros(100, dtype=torch.int32, device="cuda"), i32(0, 100, 100)
    slots[:] = -1
    rows, n = torch.zeros(2, 6, dtype=torch.int32, device="cuda"), i32(0, 0)

    def run():
        qr, kr = ops.rotary_append_paged(q, k, v, cs, pos, slots, kc, vc, want_k=True)
        return qr, ops.attention_prefill(qr, kr, v, cu), ops.paged_attention_decode(qr[:2], kc, vc, rows, n)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        run()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        qr, prompts, token = run()
    for seed, first in ((1, 61), (2, 7)):
        for x, y in zip((q, k, v), heads(100, h, hk, d, torch.float16, seed)):
            x.copy_(y)
        place = torch.randperm(12, generator=torch.Generator().manual_seed(seed))
        lens = [first, 100 - first]
        used = 0
        for s, count in enumerate(lens):
            own = place[used:used + -(-count // page)]
            used += len(own)
            at = torch.arange(count)
            begin = 0 if s == 0 else first
            pos[begin:begin + count] = at.int().cuda() + 3
            slots[begin:begin + count] = (own[at // page] * page + at % page).int().cuda()
            rows[s, :len(own)] = own.int().cuda()
        cu.copy_(i32(0, first, 100))
        n.copy_(i32(*lens))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, tol = ref.rotate(q, cs, pos, False)
        ref.assert_close(qr, want, tol)
        rotated = ops.rotary_append_paged(q, k, v, cs, pos, torch.full_like(slots, -1), kc, vc, want_k=True)[1]
        want, tol = ref.prefill(qr, rotated, v, [0, first, 100])
        ref.assert_close(prompts, want, tol)
        want, tol = ref.decode(qr[:2], kc, vc, rows, lens)
        ref.assert_close(token, want, tol)
    ops.check_device_errors()


def test_custom_ops_run_under_torch_compile():
    from mindpipe_b200.custom_ops import load_and_register
    ns = load_and_register()
    d, h, hk = 64, 4, 2
    q, k, v = (x.contiguous() for x in heads(40, h, hk, d, torch.float16, 7))
    cs, at = table(64, d), torch.arange(40, dtype=torch.int32, device="cuda")
    cu, rows, n = i32(0, 40), i32(0, 1, 2)[None], i32(40)

    def run(q, k, v, kc, vc):
        qr, kr = ns.rotary_append_paged(q, k, v, cs, at, at, kc, vc)
        return ns.attention_prefill(qr, kr, v, cu), ns.paged_attention_decode(qr[39:], kc, vc, rows, n)

    made = []
    for f in (run, torch.compile(run, fullgraph=True)):
        kc, vc = (torch.zeros(3, hk, 16, d, dtype=torch.float16, device="cuda") for _ in range(2))
        made.append((*f(q, k, v, kc, vc), kc, vc))
    qr, kr = ops.rotary_append_paged(q, k, v, cs, at, at, kc, vc, want_k=True)
    made.append((ops.attention_prefill(qr, kr, v, cu), ops.paged_attention_decode(qr[39:], kc, vc, rows, n), kc, vc))
    for x, y, z in zip(*made):
        assert torch.equal(x, y) and torch.equal(x, z)
    ops.check_device_errors()
