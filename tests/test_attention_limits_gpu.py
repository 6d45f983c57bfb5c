"""Values that are not finite, scales, ends out of order and operands that share memory, for the attention operators."""
import pytest
import torch

from mindpipe_b200 import _lib, ops
from tests import _attention_ref as ref
from tests.test_attention_gpu import TYPES, heads, paged

pytestmark = pytest.mark.gpu


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,hk,d", [(4, 2, 128), (3, 1, 64), (2, 2, 80)])
@pytest.mark.parametrize("length", [50, 128, 250, 300])
def test_prefill_values_that_are_not_finite_in_many_rows(length, h, hk, d, dtype):
    """Every third token of a sequence has an infinite value in a column of its own: each row sees those of its own tokens."""
    ends = [0, 13, 13 + length]
    q, k, v = (x.contiguous() for x in heads(ends[-1], h, hk, d, dtype, length))
    clean, hit = v.clone(), torch.zeros(ends[-1], h, d, dtype=torch.bool, device="cuda")
    for n, token in enumerate(range(ends[1], ends[2], 3)):
        column = 7 * n % d
        v[token, :, column], clean[token, :, column] = float("inf"), 0
        hit[token:ends[2], :, column] = True
    got = ops.attention_prefill(q, k, v, i32(*ends))
    want, tol = ref.prefill(q, k, clean, ends)
    ref.assert_close(got[~hit], want[~hit], tol[~hit])
    assert (got[hit] == float("inf")).all()
    ops.check_device_errors()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,hk,d", [(9, 3, 72), (5, 1, 24), (14, 2, 128), (33, 3, 56), (26, 2, 120)])
def test_decode_short_sequences_with_odd_groups_and_heads(h, hk, d, dtype):
    """A warp alone, with fewer rows than the eight or sixteen of a tile: only some of its lanes have results to store."""
    lens = [(13 * i) % 125 + 1 for i in range(320)]
    args = paged(lens, h, hk, d, 16, dtype, seed=d)
    want, tol = ref.decode(*args[:4], lens)
    ref.assert_close(ops.paged_attention_decode(*args), want, tol)
    ops.check_device_errors()


@pytest.mark.parametrize("sequences", [257, 300, 5000])
@pytest.mark.parametrize("h,hk", [(2, 1), (3, 3)])
def test_prefill_one_end_out_of_order_among_many(sequences, h, hk):
    """Beyond the number of sequences that are sorted, too: wherever the end is, and whichever way it is off."""
    t = 20 * sequences
    q, k, v = heads(t, h, hk, 64, torch.float16, 1)
    good = list(range(0, t + 1, 20))
    ops.attention_prefill(q, k, v, i32(*good))
    ops.check_device_errors()
    for at in (0, 1, sequences // 2, sequences - 1, sequences):
        for end in (-1, 0, t, t + 1):
            ends = good[:at] + [end] + good[at + 1:]
            if ends == good or (end == 0 and at <= 1) or (end == t and at >= sequences - 1):
                continue                                          # still ascending
            ops.attention_prefill(q, k, v, i32(*ends))
            with pytest.raises(_lib.MindPipeKernelError, match="out of range"):
                ops.check_device_errors()
    ops.check_device_errors()


@pytest.mark.parametrize("d", [64, 128])
def test_rows_of_minus_infinity_are_not_numbers(d):
    """A softmax over scores that are all minus infinity is 0 / 0; one finite score among them takes all the weight."""
    h, hk, n, page = 4, 2, 300, 16
    q, k, v = (x.contiguous() for x in heads(n, h, hk, d, torch.bfloat16, d))
    q[..., 0] = 1.0
    k[:, 0], k[:, 0, 0] = 0, -float("inf")                        # every score of the first two heads
    k[140, 0, 0] = 0.0                                            # ... but this token's, 0
    out = ops.attention_prefill(q, k, v, i32(0, n))
    assert out[:140, :2].isnan().all()
    assert torch.equal(out[140:, :2], v[140, 0].expand(n - 140, 2, d))
    want, tol = ref.prefill(q[:, 2:], k[:, 1:], v[:, 1:], [0, n])
    ref.assert_close(out[:, 2:], want, tol)
    pages = -(-n // page)
    kc, vc = (torch.zeros(pages, hk, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for cache, x in ((kc, k), (vc, v)):
        for t in range(n):
            cache[t // page, :, t % page] = x[t]
    rows = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    for lens, some in ((300, True), (130, False), (12, False), (0, None)):
        for batch in (1, 200):                                    # cut over the SMs; and a warp alone for the short ones
            out = ops.paged_attention_decode(q[:1].expand(batch, h, d).contiguous(), kc, vc, rows.expand(batch, -1).contiguous(),
                                             torch.full((batch,), lens, dtype=torch.int32, device="cuda"))
            if some is None:
                assert not out.any()
                continue
            assert torch.equal(out[:, :2], v[140, 0].expand(batch, 2, d)) if some else out[:, :2].isnan().all()
            assert out[:, 2:].isfinite().all()
    ops.check_device_errors()


def test_a_scale_of_zero_is_zero_and_one_that_is_not_a_number_stays_so():
    """With scores near the largest of fp32 too: all weights are equal, and a tiny scale counts as what it is."""
    n, h, hk, d = 200, 2, 1, 64
    q, k, v = (x.contiguous() for x in heads(n, h, hk, d, torch.bfloat16, 5))
    q[..., 0], q[..., 1:], k[..., 1:] = 1e19, 0, 0
    k[:, 0, 0] = torch.where(torch.arange(n, device="cuda") % 2 == 0, 1e19, -1e19).bfloat16()     # scores of 1e38 and -1e38
    cu, page = i32(0, n), 8
    kc, vc = (x.view(n // page, page, hk, d).transpose(1, 2) for x in (k, v))
    rows, one = torch.arange(n // page, dtype=torch.int32, device="cuda")[None], i32(n)
    for scale in (0.0, -0.0, 1e-38, -1e-38, 1e-33):
        want, tol = ref.prefill(q, k, v, [0, n], scale)
        ref.assert_close(ops.attention_prefill(q, k, v, cu, scale=scale), want, tol)
        ref.assert_close(ops.paged_attention_decode(q[n - 1:], kc, vc, rows, one, scale=scale), want[n - 1:], tol[n - 1:])
    assert ops.attention_prefill(q, k, v, cu, scale=float("nan")).isnan().all()
    assert ops.paged_attention_decode(q[n - 1:], kc, vc, rows, one, scale=float("nan")).isnan().all()
    ops.check_device_errors()


@pytest.mark.parametrize("h", [16, 32])
def test_decode_lists_beyond_32_bits_write_nothing(h):
    """2^25 tokens and 16 heads of keys (or 16 and twice as many queries) are within the limit, 2^27 are beyond it; one page
    stands for all of them."""
    page, hk, d = 8192, 16, 8
    kc = torch.zeros(1, hk, page, d, dtype=torch.float16, device="cuda")
    vc = torch.ones_like(kc)
    q = torch.zeros(2, h, d, dtype=torch.float16, device="cuda")
    rows = torch.zeros(2, (1 << 27) // page, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    ops.paged_attention_decode(q, kc, vc, rows, i32(5, 1 << 27), out=out)
    with pytest.raises(_lib.MindPipeKernelError, match="out of range"):
        ops.check_device_errors()
    assert (out == 7).all()
    ops.paged_attention_decode(q, kc, vc, rows, i32(5, 1 << 25), out=out)
    assert (out == 1).all()                                       # (all values are 1, all weights equal)
    ops.check_device_errors()


def pieces(x, room):
    """The 16-byte pieces of `room` that each entry of a tensor [..., D] covers."""
    at = torch.arange(room.numel()).as_strided(x.shape, x.stride(), (x.data_ptr() - room.data_ptr()) // 2)
    return (at[..., ::8] // 8).flatten().tolist()


def append_of(q, k, v, kc, vc):
    at = torch.arange(q.shape[0], dtype=torch.int32, device="cuda")
    cs = torch.cat([torch.ones(8, 4), torch.zeros(8, 4)], 1).cuda()
    return ops.rotary_append_paged(q, k, v, cs, at, at, kc, vc)


def test_caches_of_one_memory_are_taken_where_their_entries_are_apart():
    room = torch.zeros(6 * 2 * 4 * 8 * 16, dtype=torch.float16, device="cuda")
    q, k, v = torch.zeros(3, 2, 4, 8, dtype=torch.float16, device="cuda").unbind()
    dense, parts = room[:6 * 4 * 8 * 8].view(6, 4, 8, 8), room.view(6, 2, 4, 8, 16)
    apart = [(parts[:, 0, ..., :8], parts[:, 1, ..., :8]),                    # a page of keys, a page of values
             (parts[:, 0, ..., :8], parts[:, 0, ..., 8:]),                    # a key's values beside it
             (parts[:, 0, ..., :8], parts[:, 1, ..., :8].reshape(6, 8, 4, 8).transpose(1, 2)),
             (dense[:3], dense[3:]), (parts[::2, 0, ..., :8], parts[1::2, 0, ..., :8])]
    for kc, vc in apart:
        append_of(q, k, v, kc, vc)
    shifted = room[8 * 8:8 * 8 + dense.numel()].view(6, 4, 8, 8)
    for kc, vc in ((dense[:4], dense[2:]), (dense, shifted), (dense, dense.view(6, 8, 4, 8).transpose(1, 2)), (dense[::2], dense[:3])):
        with pytest.raises(ValueError, match="overlap"):
            append_of(q, k, v, kc, vc)
    with pytest.raises(ValueError, match="share memory"):
        append_of(q, k, v, room.as_strided((6, 4, 8, 8), (8 * 8, 8, 8, 1)), parts[:, 1, ..., :8])
    kc, vc = parts[:, 0, ..., :8], parts[:, 1, ..., :8]
    for i in range(3):
        mine = [q, k, v]
        mine[i] = kc[2, :, :4].transpose(0, 1)                    # the tokens' place is in the cache
        with pytest.raises(ValueError, match="overlaps the cache"):
            append_of(*(x[:2] for x in mine), kc, vc)
    beside = parts[2, 0, :, :4, 8:].transpose(0, 1)[:2]           # between a cache's rows, not in it
    append_of(beside, beside, beside, kc, vc)
    ops.check_device_errors()


def test_whether_random_views_share_memory_is_told_exactly():
    import random
    rng = random.Random(7)
    room = torch.zeros(1 << 15, dtype=torch.float16, device="cuda")
    q, k, v = torch.zeros(3, 1, 2, 8, dtype=torch.float16, device="cuda").unbind()
    counts = {True: 0, False: 0}
    for _ in range(3000):
        shape = (rng.randint(1, 4), 2, rng.randint(1, 4), 8)
        sides = []
        for _ in range(2):
            stride = [8 * rng.choice((1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64)) for _ in range(3)] + [1]
            sides.append(room.as_strided(shape, stride, 8 * rng.randint(0, 40)))
        if rng.random() < 0.6:
            sides[1] = room.as_strided(shape, sides[0].stride(), 8 * rng.randint(0, 40))
        one, two = (pieces(x, room) for x in sides)
        shared = len(set(one)) < len(one) or len(set(two)) < len(two) or bool(set(one) & set(two))
        counts[shared] += 1
        if shared:
            with pytest.raises(ValueError, match="memory"):
                append_of(q, k, v, *sides)
        else:
            append_of(q, k, v, *sides)
    assert min(counts.values()) > 200
    ops.check_device_errors()


def test_append_without_query_heads_is_refused():
    """(It would have to store keys and values all the same.)"""
    k, v = torch.zeros(2, 3, 4, 8, dtype=torch.float16, device="cuda").unbind()
    kc, vc = torch.zeros(2, 6, 4, 8, 8, dtype=torch.float16, device="cuda").unbind()
    with pytest.raises(ValueError, match="no heads"):
        append_of(k[:, :0], k, v, kc, vc)


def test_results_over_index_tensors_are_refused():
    room = torch.zeros(4, 4, 64, dtype=torch.float16, device="cuda")
    index = room.view(-1).view(torch.int32)
    q, k, v = torch.zeros(3, 4, 4, 64, dtype=torch.float16, device="cuda").unbind()
    kc, vc = torch.zeros(2, 4, 4, 16, 64, dtype=torch.float16, device="cuda").unbind()
    rows, n = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.paged_attention_decode(q, kc, vc, index[:4].view(4, 1), n, out=room),
                 lambda: ops.paged_attention_decode(q, kc, vc, rows, index[-4:], out=room),
                 lambda: ops.attention_prefill(q, k, v, index[:2], out=room)):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    ops.check_device_errors()
