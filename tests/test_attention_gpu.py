"""Rotation with append, decode over a paged cache and prompts, against 64-bit statements (``tests/_attention_ref.py``)."""
import pytest
import torch

from mindpipe_b200 import _lib, ops
from tests import _attention_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def randn(*shape, seed=0, dtype=torch.float16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def heads(rows, h, hk, d, dtype, seed):
    """q, k and v as views of one projection's result."""
    return [x.view(rows, -1, d) for x in randn(rows, (h + 2 * hk) * d, seed=seed, dtype=dtype).split([h * d, hk * d, hk * d], 1)]


def table(positions, rotated, base=10000.0):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (-torch.arange(rotated // 2, dtype=torch.float64) / (rotated // 2))
    return torch.cat([angle.cos(), angle.sin()], 1).float().cuda()


def pool(pages, hk, page, d, dtype, layout, seed):
    """A cache side whose unused room is NaN-free garbage, in several layouts."""
    if layout == "heads_first":                                   # [pages, heads, page, D], dense
        return randn(pages, hk, page, d, seed=seed, dtype=dtype)
    if layout == "tokens_first":                                  # [pages, page, heads, D], seen from the other side
        return randn(pages, page, hk, d, seed=seed, dtype=dtype).transpose(1, 2)
    return randn(pages, 3, hk, page, d + 8, seed=seed, dtype=dtype)[:, 1, :, :, :d]      # a layer's slice, padded rows


LAYOUTS = ["heads_first", "tokens_first", "slice"]


# ------------------------------------------------------------------------------------------------ rotation and append
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("t,h,hk,d,rotated,interleaved,page", [
    (1, 1, 1, 8, 2, False, 1), (1, 32, 8, 128, 128, False, 16), (7, 5, 5, 64, 64, True, 3), (33, 6, 2, 80, 80, False, 16),
    (20, 8, 4, 80, 40, False, 24), (20, 8, 4, 80, 40, True, 24), (300, 7, 1, 96, 48, False, 8), (65, 4, 2, 128, 6, False, 64),
    (257, 64, 8, 128, 128, False, 256), (40, 3, 3, 72, 72, True, 5)])
def test_append_rotates_and_stores(t, h, hk, d, rotated, interleaved, page, layout, dtype):
    q, k, v = heads(t, h, hk, d, dtype, seed=t + d)
    cs = table(9000, rotated)
    g = torch.Generator(device="cuda").manual_seed(t)
    positions = torch.randint(0, 9000, (t,), generator=g, device="cuda", dtype=torch.int32)
    pages = t // page + 4
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].int()
    slots[::5] = -1                                               # padding
    kc, vc = pool(pages, hk, page, d, dtype, layout, 1), pool(pages, hk, page, d, dtype, layout, 2)
    want_k, want_v = kc.double(), vc.double()
    tol_k = torch.zeros_like(want_k)
    (qr, q_tol), (kr, k_tol) = (ref.rotate(x, cs, positions, interleaved) for x in (q, k))
    for i, slot in enumerate(slots.tolist()):
        if slot >= 0:
            want_k[slot // page, :, slot % page], tol_k[slot // page, :, slot % page] = kr[i], k_tol[i]
            want_v[slot // page, :, slot % page] = v[i].double()
    q_out, k_out = ops.rotary_append_paged(q, k, v, cs, positions, slots, kc, vc, interleaved=interleaved, want_k=True)
    ref.assert_close(q_out, qr, q_tol)
    ref.assert_close(k_out, kr, k_tol)
    ref.assert_close(kc, want_k, tol_k)
    ref.assert_close(vc, want_v, torch.zeros_like(want_v))
    ops.check_device_errors()


def test_append_far_slots_and_no_keys_back():
    """Byte offsets beyond 2^31 in the cache."""
    pages, hk, page, d = 1100, 8, 128, 128                        # 2.1 GB a side
    kc, vc = (torch.zeros(pages, hk, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
    q, k, v = heads(3, 8, hk, d, torch.float16, 5)
    slots = torch.tensor([pages * page - 1, 0, 130000], dtype=torch.int32, device="cuda")
    cs, pos = table(16, d), torch.tensor([0, 15, 3], dtype=torch.int32, device="cuda")
    _, none = ops.rotary_append_paged(q, k, v, cs, pos, slots, kc, vc)
    assert none is None
    rotated, tol = ref.rotate(k, cs, pos, False)
    for i, s in enumerate(slots.tolist()):
        ref.assert_close(kc[s // page, :, s % page], rotated[i], tol[i])
        assert torch.equal(vc[s // page, :, s % page], v[i])
    assert int((kc != 0).any(-1).sum()) == 3 * hk and int((vc != 0).any(-1).sum()) == 3 * hk


def test_append_indices_out_of_range_touch_nothing():
    page, pages, d = 4, 3, 64
    q, k, v = heads(5, 2, 1, d, torch.float16, 1)
    room = torch.zeros(pages + 2, 1, page, d, dtype=torch.float16, device="cuda")
    kc, vc = room[1:-1], room.clone()[1:-1]
    cs = table(10, d)
    for pos, slot in (([0, 1, 2, 3, 10], [0, 1, 2, 3, 4]), ([-1, 1, 2, 3, 4], [4, 1, 2, 3, 0]), ([0, 1, 2, 3, 4], [0, 1, 2, 3, 12]),
                      ([0, 1, 2, 3, 4], [2**31 - 1, 1, 2, 3, 0])):
        room.zero_()
        pos, slot = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (pos, slot))
        ops.rotary_append_paged(q, k, v, cs, pos, slot, kc, vc)
        with pytest.raises(_lib.MindPipeKernelError, match="out of range"):
            ops.check_device_errors()
        assert not room[0].any() and not room[-1].any()
        assert int((kc != 0).any(-1).sum()) == 4                  # the four good tokens
    pos, slot = torch.tensor([0, 99, 2, -5, 4], dtype=torch.int32, device="cuda"), torch.tensor([0, -1, 2, -7, 4], dtype=torch.int32, device="cuda")
    ops.rotary_append_paged(q, k, v, cs, pos, slot, kc, vc)       # padding tokens may have any position
    ops.check_device_errors()


# --------------------------------------------------------------------------------------------------------------- decode
def paged(lens, h, hk, d, page, dtype, layout="heads_first", seed=0, q_scale=1.0):
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    rows, used = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        rows[i, :n] = order[used:used + n]
        used += n
    kc, vc = pool(pages, hk, page, d, dtype, layout, seed + 1), pool(pages, hk, page, d, dtype, layout, seed + 2)
    for c in (kc, vc):                                            # what no token has written
        for i, n in enumerate(lens):
            if n % page:
                c[rows[i, need[i] - 1].long(), :, n % page:] = float("nan")
    q = heads(len(lens), h, hk, d, dtype, seed + 3)[0] * q_scale
    return q, kc, vc, rows.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [0, 1, 2, 0], [15, 16, 17], [63, 64, 65, 129, 31], [1000], [5, 3001, 0, 700], [300] * 40])
@pytest.mark.parametrize("h,hk,d,page,layout", [
    (1, 1, 8, 1, "heads_first"), (32, 8, 128, 16, "heads_first"), (8, 8, 64, 24, "tokens_first"), (35, 5, 80, 7, "slice"),
    (20, 1, 96, 16, "tokens_first"), (64, 4, 128, 64, "slice"), (40, 1, 64, 100, "heads_first")])
def test_decode(h, hk, d, page, layout, lens, dtype):
    args = paged(lens, h, hk, d, page, dtype, layout, seed=len(lens) + d)
    want, tol = ref.decode(*args[:4], lens)
    ref.assert_close(ops.paged_attention_decode(*args), want, tol)
    ops.check_device_errors()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_decode_scales_and_peaks(scale):
    """One weight near 1, all equal, and a maximum that comes last."""
    lens = [400, 90]
    q, kc, vc, rows, n = paged(lens, 8, 2, 128, 16, torch.float16, seed=9, q_scale=3.0)
    want, tol = ref.decode(q, kc, vc, rows, lens, scale)
    ref.assert_close(ops.paged_attention_decode(q, kc, vc, rows, n, scale=scale), want, tol)


def test_decode_infinities():
    """Keys that push a weight to zero and values that are infinite only where attended to."""
    lens = [70, 33]
    q, kc, vc, rows, n = paged(lens, 4, 2, 64, 16, torch.bfloat16, seed=3)
    kc[rows[0, 1].long(), 0, 3] = 3e38                            # an overflowing score: plus or minus infinity by the row
    vc[rows[1, 0].long(), 1, 5, 7] = float("inf")
    out = ops.paged_attention_decode(q, kc, vc, rows, n)
    want, tol = ref.decode(q, kc, vc, rows, lens)
    clean = torch.ones_like(want, dtype=torch.bool)
    clean[0, :2] = False
    clean[1, 2:, 7] = False
    ref.assert_close(out[clean], want[clean], tol[clean])
    assert (out[1, 2:, 7] == float("inf")).all()


def test_decode_long_and_few(dtype=torch.bfloat16):
    """A sequence over all blocks, twice the same bits, and a batch beyond one block's lanes."""
    lens = [70001, 17]
    args = paged(lens, 16, 2, 128, 64, dtype, seed=4)
    got = ops.paged_attention_decode(*args)
    want, tol = ref.decode(*args[:4], lens)
    ref.assert_close(got, want, tol)
    assert torch.equal(got, ops.paged_attention_decode(*args))
    lens = [(7 * i) % 90 for i in range(1500)]
    args = paged(lens, 4, 2, 64, 16, dtype, seed=5)
    want, tol = ref.decode(*args[:4], lens)
    ref.assert_close(ops.paged_attention_decode(*args), want, tol)


def test_decode_lengths_and_pages_out_of_range():
    lens = [40, 20]
    q, kc, vc, rows, n = paged(lens, 4, 2, 64, 16, torch.float16, seed=6)
    good = ops.paged_attention_decode(q, kc, vc, rows, n)
    ops.check_device_errors()
    bad_page, far_page = rows.clone(), rows.clone()
    bad_page[0, 1], far_page[0, 0] = -1, kc.shape[0]
    for table_, lens_ in ((bad_page, n), (far_page, n), (rows, torch.tensor([-3, 20], dtype=torch.int32, device="cuda")),
                          (rows, torch.tensor([16 * rows.shape[1] + 1, 20], dtype=torch.int32, device="cuda"))):
        out = ops.paged_attention_decode(q, kc, vc, table_, lens_)
        with pytest.raises(_lib.MindPipeKernelError, match="out of range"):
            ops.check_device_errors()
        assert torch.equal(out[1], good[1])


def test_decode_captured_serves_later_lengths(new_stream):
    q, kc, vc, rows, n = paged([500, 300, 7], 8, 2, 128, 16, torch.float16, seed=8)
    torch.nan_to_num_(kc), torch.nan_to_num_(vc)
    stream = new_stream()
    with torch.cuda.stream(stream):
        ops.paged_attention_decode(q, kc, vc, rows, n)
    stream.synchronize()
    graphs = []
    for _ in range(2):                                            # two graphs of one stream, replayed side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = ops.paged_attention_decode(q, kc, vc, rows, n)
        graphs.append((g, out))
    for lens in ([1, 300, 512], [0, 0, 3], [499, 2, 100]):
        rows[2] = rows[0]
        n.copy_(torch.tensor(lens))
        want, tol = ref.decode(q, kc, vc, rows, lens)
        side = new_stream()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            ref.assert_close(out, want, tol)


# --------------------------------------------------------------------------------------------------------------- prompts
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [2, 1, 0, 3], [127, 128, 129], [255, 256, 257], [64] * 5 + [0, 65], [700, 1, 385], [1025]])
@pytest.mark.parametrize("h,hk,d", [(1, 1, 8), (4, 1, 128), (6, 2, 64), (5, 5, 80), (3, 1, 128), (8, 8, 96)])
def test_prefill(h, hk, d, lens, dtype):
    ends = [0]
    for n in lens:
        ends.append(ends[-1] + n)
    q, k, v = heads(ends[-1], h, hk, d, dtype, seed=len(lens) + d)
    got = ops.attention_prefill(q, k, v, torch.tensor(ends, dtype=torch.int32, device="cuda"))
    want, tol = ref.prefill(q, k, v, ends)
    ref.assert_close(got, want, tol)
    ops.check_device_errors()


def test_prefill_rows_of_no_sequence_are_left_alone():
    """Rows in front of, and behind, the sequences; what they hold does not enter either."""
    t, ends = 300, [10, 140, 140, 271]
    q, k, v = (x.contiguous() for x in heads(t, 4, 2, 128, torch.float16, 1))
    for x in (q, k, v):
        x[:10], x[271:] = float("nan"), float("nan")
    out = randn(t, 4, 128, seed=2)
    before = out.clone()
    got = ops.attention_prefill(q, k, v, torch.tensor(ends, dtype=torch.int32, device="cuda"), out=out)
    assert got is out or got.data_ptr() == out.data_ptr()
    want, tol = ref.prefill(q, k, v, ends)
    ref.assert_close(out, want, tol)
    assert torch.equal(out[:10], before[:10]) and torch.equal(out[271:], before[271:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,hk,d", [(4, 2, 128), (3, 1, 64), (2, 2, 80)])
@pytest.mark.parametrize("at", [5, 127, 128, 200, 300, 399])
def test_prefill_infinite_and_nan_values_reach_only_later_rows(at, h, hk, d, dtype):
    """Values (and keys) of a token that are not finite: the rows in front of it are those of a clean token."""
    ends = [0, 37, 437, 500]
    q, k, v = (x.contiguous() for x in heads(500, h, hk, d, dtype, 6))
    token = ends[1] + at
    v[token, 0, 3], v[token, 0, d - 1] = float("inf"), float("nan")
    clean = v.clone()
    clean[token, 0, 3], clean[token, 0, d - 1] = 0, 0
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    got = ops.attention_prefill(q, k, v, cu)
    want, tol = ref.prefill(q, k, clean, ends)
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[token:ends[2], :h // hk, 3] = hit[token:ends[2], :h // hk, d - 1] = True
    ref.assert_close(got[~hit], want[~hit], tol[~hit])
    assert (got[token:ends[2], :h // hk, 3] == float("inf")).all() and got[token:ends[2], :h // hk, d - 1].isnan().all()
    k[token, 0] = float("nan")
    got = ops.attention_prefill(q, k, clean, cu)
    hit[token:ends[2], :h // hk] = True
    ref.assert_close(got[~hit], want[~hit], tol[~hit])
    assert got[token:ends[2], :h // hk].isnan().all()
    ops.check_device_errors()


def test_prefill_operands_of_other_strides():
    """Heads first in memory, padded rows, one head of keys for all by expansion, a slice of heads."""
    t, h, d, ends = 410, 4, 64, [0, 300, 410]
    q, k = randn(h, t, d, seed=1).transpose(0, 1), randn(2, t, d + 8, seed=2)[..., :d].transpose(0, 1)
    v = randn(t, 7, d, seed=3)[:, 2:6:2]
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    want, tol = ref.prefill(q, k, v, ends)
    ref.assert_close(ops.attention_prefill(q, k, v, cu), want, tol)
    one = k[:, :1].expand(t, 4, d)
    want, tol = ref.prefill(q, one, one, ends)
    ref.assert_close(ops.attention_prefill(q, one, one, cu), want, tol)
    with pytest.raises(_lib.MindPipeKernelError, match="not supported"):
        ops.attention_prefill(q, k[:1].expand(t, 2, d), v, cu)    # tokens that are all the same row


@pytest.mark.parametrize("scale", [0.0, -0.2, 5.0])
def test_prefill_scales(scale):
    ends = [0, 333, 600]
    q, k, v = heads(600, 4, 2, 64, torch.bfloat16, 3)
    want, tol = ref.prefill(q, k, v, ends, scale)
    ref.assert_close(ops.attention_prefill(q, k, v, torch.tensor(ends, dtype=torch.int32, device="cuda"), scale=scale), want, tol)


def test_prefill_long():
    ends = [0, 5000, 5003]
    q, k, v = heads(5003, 4, 2, 128, torch.bfloat16, 4)
    want, tol = ref.prefill(q, k, v, ends)
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    got = ops.attention_prefill(q, k, v, cu)
    ref.assert_close(got, want, tol)
    assert torch.equal(got, ops.attention_prefill(q, k, v, cu))


def test_prefill_sequence_ends_out_of_range():
    q, k, v = heads(200, 2, 1, 64, torch.float16, 5)
    for ends in ([0, 201], [-1, 100], [0, 150, 100]):
        ops.attention_prefill(q, k, v, torch.tensor(ends, dtype=torch.int32, device="cuda"))
        with pytest.raises(_lib.MindPipeKernelError, match="out of range"):
            ops.check_device_errors()


# -------------------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    q, k, v = heads(4, 4, 2, 64, torch.float16, 0)
    kc, vc = (randn(5, 2, 16, 64, seed=i) for i in (1, 2))
    cs = table(8, 64)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    pos, slots = i32(0, 1, 2, 3), i32(0, 1, 2, 3)
    rows, n, cu = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), i32(1, 2, 3, 4), i32(0, 4)

    def append(**kw):
        a = dict(q=q, k=k, v=v, cos_sin=cs, positions=pos, slots=slots, k_cache=kc, v_cache=vc) | kw
        return ops.rotary_append_paged(**a)

    def decode(**kw):
        return ops.paged_attention_decode(**(dict(q=q, k_cache=kc, v_cache=vc, page_table=rows, seq_lens=n) | kw))

    def prefill(**kw):
        return ops.attention_prefill(**(dict(q=q, k=k, v=v, cu_seqlens=cu) | kw))

    append(), decode(), prefill()
    ops.check_device_errors()
    odd = randn(4, 4 * 64 + 4)[:, 4:].view(4, 4, 64)               # rows that begin 8 bytes off
    for call, kw, error in [
            (append, dict(q=q.float()), TypeError), (append, dict(k=k.bfloat16()), TypeError), (append, dict(q=odd), ValueError),
            (append, dict(q=q.cpu()), ValueError), (append, dict(k=k.cpu()), ValueError), (append, dict(slots=[0, 1, 2, 3]), TypeError),
            (append, dict(positions=pos.long()), TypeError), (append, dict(slots=slots[:3]), ValueError),
            (append, dict(cos_sin=cs.double()), TypeError), (append, dict(cos_sin=table(8, 66)), ValueError),
            (append, dict(cos_sin=cs[:, :63].contiguous()), ValueError), (append, dict(k=k[:, :1]), ValueError),
            (append, dict(v_cache=vc[:4]), ValueError), (append, dict(k_cache=kc[..., :56]), ValueError),
            (decode, dict(q=q[:3]), ValueError), (decode, dict(q=q[:, :3]), ValueError), (decode, dict(q=q[:, 0]), ValueError),
            (decode, dict(page_table=rows.long()), TypeError), (decode, dict(page_table=rows[:, :0]), ValueError),
            (decode, dict(seq_lens=n[:3]), ValueError), (decode, dict(k_cache=kc.bfloat16()), TypeError),
            (decode, dict(out=torch.empty(4, 4, 64, device="cuda")), TypeError), (decode, dict(out=q), ValueError),
            (decode, dict(q=randn(4, 4, 136), k_cache=randn(5, 2, 16, 136), v_cache=randn(5, 2, 16, 136)), ValueError),
            (decode, dict(q=randn(4, 4, 60), k_cache=randn(5, 2, 16, 60), v_cache=randn(5, 2, 16, 60)), ValueError),
            (prefill, dict(q=q[:, :3]), ValueError), (prefill, dict(k=k[:3]), ValueError), (prefill, dict(v=v[..., :56]), ValueError),
            (prefill, dict(cu_seqlens=cu.long()), TypeError), (prefill, dict(cu_seqlens=cu[:0]), ValueError),
            (prefill, dict(scale="x"), TypeError), (prefill, dict(out=torch.empty(3, 4, 64, device="cuda", dtype=torch.float16)), ValueError)]:
        with pytest.raises(error):
            call(**kw)
    ops.check_device_errors()
    empty = ops.attention_prefill(q[:0], k[:0], v[:0], i32(0))
    assert empty.shape == (0, 4, 64)
    assert ops.paged_attention_decode(q[:0], kc, vc, rows[:0], n[:0]).shape == (0, 4, 64)
    assert append(q=q[:0], k=k[:0], v=v[:0], positions=pos[:0], slots=slots[:0])[0].shape == (0, 4, 64)
