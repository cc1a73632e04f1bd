"""Attention over pages and the paged append on the GPU where they went wrong or could: cuts of many pairs, windows
behind which pages were given back, memory that overlaps, values that are not finite, widths between the tested ones."""
from __future__ import annotations

import pytest
import torch

from avqa_b200 import BackendError, RotaryEmbedding, ops
from paged_reference import DTYPES, assert_within, attention64, half, rotate64
from test_gpu_paged import Batch, fault

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128)])
def test_many_cut_pairs_give_the_same_bits_again(dt, D) -> None:
    """More (key head, 256-row) pairs than SMs, each with more key tiles than a piece: where a pair is cut hangs on
    the sums of all items before it, so a sum read before it is written moves the cuts and with them the bits."""
    b = Batch(dt, 8, 8, D, 64, [256] * 22, [4096 - 96 * i for i in range(22)])
    first = b.check()
    for _ in range(30):
        assert torch.equal(ops.paged_attention(b.q, *b.lists), first)
    assert fault() == 0


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("bf16", 128), ("f16", 72), ("f32", 64)])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("less", [0, 1, 127, 65536])
def test_the_longest_sequence_that_a_table_may_hold(dt, D, new, less) -> None:
    """A window at the end of 2^31 - 65537 tokens, which all lie on one page whose slots are the same row."""
    room = 2 ** 31 - 65537
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(new, 4, D, generator=g, device="cuda").to(DTYPES[dt])
    k, v = (torch.randn(1, 2, 1, D, generator=g, device="cuda").to(DTYPES[dt]) for _ in range(2))
    lists = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0]], [room - less], [0, new])]
    pools = [x.expand(-1, -1, room, -1) for x in (k, v)]
    got = ops.paged_attention(q, *pools, *lists, window=300)
    # every key scores the same: the values' own row, which each sum's roundings reach
    want = v[0, :, 0].double().repeat_interleave(2, 0).expand(new, -1, -1)
    assert_within(got, want, want.abs() * 4 * half(DTYPES[dt]) + want.abs() * 400 * 2.0 ** -24, "one row everywhere")
    assert fault() == 0
    lists[1] -= room  # no keys at all, and fewer than none
    assert (ops.paged_attention(q, *pools, *lists, window=300) == 0).all()
    assert fault() == (2 if less else 0)


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("bf16", 72), ("f32", 64)])
@pytest.mark.parametrize("page", [8, 16, 24, 100, 128, 384])
@pytest.mark.parametrize("new,window", [([1, 2], 50), ([40, 300], 50), ([40, 300], 700), ([300], 1)])
def test_pages_behind_the_window_are_not_looked_up(dt, D, page, new, window) -> None:
    """Pages whose keys no token of the sequence sees may have been given back: no fault, and the same bits."""
    lens = [1200 + n for n in new]
    b = Batch(dt, 4, 2, D, page, new, lens)
    want = b.check(window=window)
    gone = [(n - k + 1 - window) // page for n, k in zip(lens, new)]  # pages before the first token's first key
    assert all(n > 0 for n in gone)
    used = set(b.block_table.flatten().tolist())
    spare = next(p for p in range(b.key_pool.shape[0]) if p not in used)
    assert torch.isnan(b.key_pool[spare].float()).all()
    for other in (-1, b.key_pool.shape[0], spare):  # none, none, one that holds NaN
        for row, n in enumerate(gone):
            b.block_table[row, :n] = other
        assert torch.equal(ops.paged_attention(b.q, *b.lists, window=window), want)
        assert fault() == 0
    row = len(new) - 1
    b.block_table[row, gone[row]] = -1  # a page that is seen
    ops.paged_attention(b.q, *b.lists, window=window)
    assert fault() == 2


@pytest.mark.parametrize("dt,D,page", [("bf16", 128, 16), ("f16", 64, 24), ("f16", 72, 16), ("bf16", 256, 16)])
@pytest.mark.parametrize("new,length", [(3, 40), (60, 2000), (200, 200), (200, 6000)])
def test_values_that_are_not_finite_leave_the_rest_its_bits(dt, D, page, new, length) -> None:
    """A value that is not finite, and that every row sees, changes its own column; the rest keeps the bits that it has
    without: no row is formed again another way.  A key or a query changes the rows that see it; the others stay within
    the bounds of fp64 (the tensor-core kernel's rows of a warp take over a new maximum together, so that the bits of
    a row hang on its neighbours' scores)."""
    b = Batch(dt, 4, 2, D, page, [new, 1], [length, 30])
    clean = b.check()
    want, bound, _ = attention64(b.q, *b.lists)

    def run():
        got = ops.paged_attention(b.q, *b.lists)
        return got, (got.view(torch.int16) == clean.view(torch.int16))

    at = (length - new) // 2  # a token that every row of the first sequence sees
    slot = int(b.block_table[0, at // page]), 1, at % page
    for value in (float("nan"), float("inf")):  # a value, in one column of the second key head
        kept = b.value_pool[slot].clone()
        b.value_pool[slot][7] = value
        got, same = run()
        b.value_pool[slot] = kept
        assert not torch.isfinite(got[:new, 2:, 7].float()).any()
        same[:new, 2:, 7] = True
        assert same.all()
    at = length - new + new // 2  # a token that the later rows see
    slot = int(b.block_table[0, at // page]), 1, at % page
    kept = b.key_pool[slot].clone()
    b.key_pool[slot][7] = float("nan")
    got = run()[0]
    b.key_pool[slot] = kept
    assert torch.isnan(got[new // 2:new, 2:].float()).all()
    seen = torch.zeros(b.N, 4, dtype=torch.bool, device="cuda")
    seen[new // 2:new, 2:] = True
    assert_within(got[~seen], want[~seen], bound[~seen], "a key")
    kept = b.q[new // 2, 3].clone()
    b.q[new // 2, 3, 5] = float("nan")
    got = run()[0]
    b.q[new // 2, 3] = kept
    assert torch.isnan(got[new // 2, 3].float()).all()
    seen.fill_(False)
    seen[new // 2, 3] = True
    assert_within(got[~seen], want[~seen], bound[~seen], "a query")
    assert run()[1].all()


def test_outputs_in_the_memory_of_inputs_are_refused() -> None:
    b = Batch("bf16", 4, 2, 64, 16, [3, 2], [20, 30])
    want = ops.paged_attention(b.q, *b.lists)
    room = torch.zeros(b.N * 2 + 1, 8, 64, device="cuda", dtype=b.dt)
    q = room[:b.N, :4]
    q.copy_(b.q)
    for out in (q, room[1:b.N + 1, :4], room[:b.N, 3:7], room.view(-1, 64)[2:2 + 4 * b.N].view(b.N, 4, 64)):
        with pytest.raises(BackendError):
            ops.paged_attention(q, *b.lists, out=out)
    out = room[:b.N, 4:]  # beside the query's heads, in the same rows
    assert torch.equal(ops.paged_attention(q, *b.lists, out=out), want) and torch.equal(q, b.q)
    rot = RotaryEmbedding(64)
    k, v = room[b.N:2 * b.N, :2], room[b.N:2 * b.N, 2:4]
    k.copy_(b.k)
    v.copy_(b.v)
    for out in (room[1:b.N + 1, :4], room[:b.N, 2:6], room[b.N:2 * b.N, 1:5], room[b.N + 1:2 * b.N + 1, 3:7]):
        with pytest.raises(BackendError):
            ops.paged_append(k, v, *b.lists, q=q, rotary=rot, q_out=out)
    want = ops.paged_append(b.k, b.v, *b.lists, q=b.q, rotary=rot)
    assert torch.equal(ops.paged_append(k, v, *b.lists, q=q, rotary=rot, q_out=room[:b.N, 4:]), want)
    assert ops.paged_append(k, v, *b.lists, q=q, rotary=rot, q_out=q) is q
    assert torch.equal(q, want) and torch.equal(k, b.k) and torch.equal(v, b.v)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [80, 96, 112, 192])
@pytest.mark.parametrize("new,lens,kw", [([1, 1], [300, 5], {}), ([30, 1], [200, 70], {}), ([90], [500], dict(window=40)),
                                         ([20], [77], dict(causal=False))])
def test_widths_between_the_padded_ones(dt, D, new, lens, kw) -> None:
    b = Batch(dt, 6, 2, D, 16, new, lens, seed=D)
    first = b.check(**kw)
    assert torch.equal(ops.paged_attention(b.q, *b.lists, **kw), first)
    rot = RotaryEmbedding(D, rotary_dim=D // 4 * 2)
    pos = torch.cat([torch.arange(n - t, n) for t, n in zip(new, lens)]).cuda()
    q = ops.paged_append(b.k, b.v, *b.lists, q=b.q, rotary=rot)
    assert_within(q.transpose(0, 1), *rotate64(b.q.transpose(0, 1), pos[None], rot), "queries")
    b.check("behind the append", q=q, **kw)
    assert fault() == 0
