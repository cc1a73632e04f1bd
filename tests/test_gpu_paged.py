"""The paged append and attention over pages on the GPU against fp64
(``paged_reference``, whose bounds count the roundings): types, head groups,
page sizes, ragged batches with empty sequences, windows, strided pools and
operands, dirty pages, shared pages, bad pages, graphs and streams.
"""
from __future__ import annotations

import ctypes
import random

import pytest
import torch

from avqa_b200 import (AVQAttention, AVQConfig, BackendError, BlockKVCache, DeviceError, DtypeError,
                       NotInitializedError, RotaryEmbedding, ShapeError, _lib, ops)
from avqa_b200.config import AttentionShapeConfig, ExecutionConfig
from paged_reference import DTYPES, assert_within, attention64, rotate64

pytestmark = pytest.mark.gpu


def fault() -> int:
    code = ctypes.c_int(-1)
    _lib.check(_lib.load().avq_device_fault(ctypes.byref(code), None), "avq_device_fault")
    return code.value


class Batch:
    """A packed batch over a pool whose unwritten slots hold NaN."""

    def __init__(self, dt, H, Hkv, D, page, new, lens, seed=0, slot_major=False, width=0, scale=2.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dt, self.page = DTYPES[dt], page
        randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        W = max([1, width, *need])
        rows, at = [], 0
        for n in need:
            rows.append(order[at:at + n] + [-7] * (W - n))  # entries behind the last page are never looked at
            at += n
        shape = (pages, page, Hkv, D) if slot_major else (pages, Hkv, page, D)
        self.key_pool, self.value_pool = (torch.full(shape, float("nan"), device="cuda", dtype=self.dt)
                                          for _ in range(2))
        if slot_major:
            self.key_pool, self.value_pool = self.key_pool.transpose(1, 2), self.value_pool.transpose(1, 2)
        for row, n, length in zip(rows, need, lens):
            for i in range(n):
                take = min(page, length - i * page)
                self.key_pool[row[i], :, :take] = randn(Hkv, take, D).to(self.dt)
                self.value_pool[row[i], :, :take] = randn(Hkv, take, D).to(self.dt)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.block_table = torch.tensor(rows, **i32)
        self.kv_len = torch.tensor(lens, **i32)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.q_start = torch.tensor(starts, **i32)
        self.N = starts[-1]
        self.q = (randn(self.N, H, D) * scale).to(self.dt)
        self.k, self.v = randn(self.N, Hkv, D).to(self.dt), randn(self.N, Hkv, D).to(self.dt)

    @property
    def lists(self):
        return self.key_pool, self.value_pool, self.block_table, self.kv_len, self.q_start

    def check(self, what="", q=None, **kw):
        q = self.q if q is None else q
        got = ops.paged_attention(q, *self.lists, **kw)
        kw.pop("max_q_len", None)
        want, bound, _ = attention64(q, *self.lists, **kw)
        assert_within(got, want, bound, what)
        return got


# dtype, H, Hkv, D, page, new, lens, kwargs
CASES = {
    "one_token": ("bf16", 4, 4, 64, 16, [1], [1], {}),
    "one_token_long": ("bf16", 8, 2, 128, 16, [1], [4099], {}),
    "many_spans": ("f16", 2, 1, 64, 256, [1, 1], [9000, 17], {}),
    "ragged_decode": ("bf16", 32, 8, 128, 24, [1] * 7, [1, 16, 17, 24, 25, 700, 333], {}),
    "seventy": ("f16", 4, 2, 64, 8, [1] * 70, [1 + 13 * i % 97 for i in range(70)], {}),
    "empty_ones": ("bf16", 4, 2, 64, 16, [0, 3, 0, 2, 1, 0], [40, 3, 0, 1, 0, 9], {}),  # rows that see nothing
    "chunk": ("bf16", 8, 2, 128, 16, [37, 5], [100, 64], {}),
    "chunk_mha_page1": ("f16", 3, 3, 64, 1, [20], [33], {}),
    "chunk_odd_page": ("bf16", 4, 1, 128, 5, [130], [301], {}),
    "prefill_only": ("bf16", 2, 2, 64, 64, [129, 64, 1], [129, 64, 1], {}),
    "not_causal": ("f16", 4, 2, 128, 16, [9, 2], [50, 130], dict(causal=False)),
    "window": ("bf16", 4, 2, 64, 16, [50, 1, 3], [400, 90, 3], dict(window=33)),
    "window_one": ("bf16", 2, 1, 128, 16, [70], [200], dict(window=1)),
    "scale": ("f16", 2, 2, 64, 16, [3], [77], dict(scale=0.7)),
    "scale_zero": ("f16", 2, 2, 64, 16, [3, 40], [77, 60], dict(scale=0.0)),
    "negative_scale": ("bf16", 2, 2, 64, 16, [3], [77], dict(scale=-0.2)),
    "wide_group": ("bf16", 40, 1, 128, 32, [1, 2, 9], [500, 40, 9], {}),
    "group_of_three": ("bf16", 9, 3, 64, 16, [1, 20], [129, 61], {}),
    "d40": ("bf16", 4, 2, 40, 16, [6, 1], [70, 200], {}),
    "d72": ("f16", 2, 1, 72, 100, [30], [250], {}),
    "d256": ("bf16", 4, 2, 256, 16, [17, 1], [120, 300], {}),
    "d33": ("bf16", 2, 1, 33, 16, [6], [70], {}),  # rows at odd addresses
    "d1": ("f32", 1, 1, 1, 3, [2], [7], {}),
    "f32": ("f32", 8, 8, 64, 16, [64, 64], [1064, 500], {}),
    "f32_d128": ("f32", 4, 2, 128, 16, [5, 1], [70, 2000], {}),
    "f32_d256": ("f32", 2, 1, 256, 16, [5], [70], {}),
    "f32_d30": ("f32", 2, 1, 30, 16, [20], [70], dict(window=9)),
    "mixed_step": ("bf16", 8, 4, 128, 16, [300, 1, 1, 1, 70], [900, 50, 2000, 1, 70], {}),
    "big_chunk": ("bf16", 8, 1, 128, 256, [300], [1500], {}),
    "big_chunk_f16_d64": ("f16", 4, 4, 64, 16, [260, 515], [260, 1030], {}),
    "big_window": ("bf16", 4, 2, 128, 32, [400, 3], [1700, 800], dict(window=300)),
    "chunk_longer_than_its_cache": ("bf16", 4, 2, 64, 16, [60, 0, 33], [40, 5, 0], {}),  # rows that see nothing
    "rows_16_and_17": ("f16", 1, 1, 64, 16, [16, 17], [200, 150], {}),
    "rows_128_and_129": ("bf16", 2, 1, 128, 16, [64, 65], [64, 300], {}),
    "rows_256_and_257": ("bf16", 1, 1, 128, 128, [256, 257], [400, 257], {}),
    "page_384": ("f16", 4, 2, 64, 384, [90, 1], [1000, 385], {}),
    "page_8": ("bf16", 4, 2, 128, 8, [40, 1], [333, 41], {}),
    "many_sequences": ("bf16", 2, 1, 64, 16, [1] * 1100, [1 + 7 * i % 45 for i in range(1100)], {}),
    "many_chunks": ("bf16", 1, 1, 64, 16, [20] * 1100, [20 + 7 * i % 45 for i in range(1100)], {}),
    "big_not_causal": ("bf16", 4, 2, 64, 16, [200], [700], dict(causal=False)),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("slot_major", [False, True])
def test_attention_matches_formula(name, slot_major) -> None:
    dt, H, Hkv, D, page, new, lens, kw = CASES[name]
    b = Batch(dt, H, Hkv, D, page, new, lens, seed=len(name), slot_major=slot_major)
    first = b.check(name, **kw)
    # the bound on new tokens steers the kernels, right or wrong, and the result stays in its bounds
    for most in (1, max(new), 100000):
        b.check(f"{name}, max_q_len {most}", max_q_len=most, **kw)
    assert torch.equal(ops.paged_attention(b.q, *b.lists, **kw), first)  # the same bits again
    assert fault() == 0


@pytest.mark.parametrize("dt,D", [("bf16", 128), ("f16", 64), ("bf16", 72), ("f32", 64), ("f32", 256)])
@pytest.mark.parametrize("new,lens", [([1], [1]), ([1, 0, 1], [2, 900, 1023]), ([2, 1], [1000, 0]), ([3, 1], [2, 70])])
@pytest.mark.parametrize("window", [0, 40])
def test_few_short_sequences_by_either_split(dt, D, new, lens, window) -> None:
    """Tables of different widths hold the same keys: clusters of CTAs for the narrow, spans and a join for the wide."""
    for pages in (0, 600):
        b = Batch(dt, 4, 2, D, 16, new, lens, width=pages)
        b.check(f"{pages} pages to a row", window=window)
        b.check(f"{pages} pages to a row, every key", causal=False)


def test_many_keys_take_the_larger_count_of_pieces() -> None:
    """More keys than a single round of CTAs takes: 16 heads of 17 sequences, with rows that see little among them."""
    b = Batch("bf16", 16, 16, 64, 32, [1] * 17, [2300] * 15 + [1, 0])
    b.check()
    b.check(window=100)


def test_one_pair_over_more_keys_than_its_pieces_number() -> None:
    """One key head and one row tile over 350000 keys: the most pieces that a pair may have."""
    b = Batch("bf16", 2, 1, 64, 256, [20], [350000])
    b.check()
    b.check(window=330000)
    assert fault() == 0


@pytest.mark.parametrize("dt,D", [("bf16", 128), ("f16", 64), ("f32", 40)])
@pytest.mark.parametrize("B", [64, 65, 300, 1025])
@pytest.mark.parametrize("chunk", [1, 40])
def test_long_lists_of_sequences(dt, D, B, chunk) -> None:
    """Sequences of all kinds by the hundreds: empty ones, ones longer than a span, none seen, beside chunks or not."""
    r = random.Random(B)
    new = [r.choice([0, 1, 1, 1, 2]) for _ in range(B)]
    new[B // 2] = chunk
    lens = [r.choice([0, 1, 5, 17, 40]) + n for n in new]
    lens[B // 3], lens[B - 1] = 2000, 700
    b = Batch(dt, 4, 2, D, 16, new, lens, seed=B)
    b.check()
    b.check("window", window=30)
    assert fault() == 0
    lens = b.kv_len.clone()
    b.kv_len[5] = 1 << 30  # beyond the table's row
    ops.paged_attention(b.q, *b.lists)
    assert fault() == 2
    b.kv_len.copy_(lens)
    want = b.check()
    b.q_start[:B // 4] = b.q_start[B // 4].clone()  # the first quarter has no tokens any more
    out = torch.full_like(want, 7.0)
    ops.paged_attention(b.q, *b.lists, out=out)
    first = int(b.q_start[B // 4])
    assert (out[:first] == 7.0).all()
    rest, bound, _ = attention64(b.q, *b.lists)
    assert_within(out[first:], rest[first:], bound[first:], "a quarter without tokens")


@pytest.mark.parametrize("dt,D", [("bf16", 128), ("f16", 64), ("f32", 64)])
@pytest.mark.parametrize("new,lens", [([3, 1], [1, 50]), ([60, 40], [40, 90])])
def test_window_of_any_size(dt, D, new, lens) -> None:
    """A window larger than every cache hides nothing, with rows before the first position too."""
    b = Batch(dt, 4, 2, D, 16, new, lens)
    want = b.check()
    for window in (91, 2 ** 31 - 2, 2 ** 31 - 1):
        b.check(f"window {window}", window=window)
        assert torch.equal(ops.paged_attention(b.q, *b.lists, window=window) == 0, want == 0)


def test_attention_refuses_what_it_cannot_take() -> None:
    b = Batch("bf16", 4, 2, 64, 16, [2], [20])
    for kw in (dict(window=2 ** 31), dict(window=-1), dict(max_q_len=2 ** 31), dict(max_q_len=-1), dict(out=b.q),
               dict(scale=float("nan")), dict(scale=3e38), dict(window=4, causal=False)):
        with pytest.raises(BackendError):
            ops.paged_attention(b.q, *b.lists, **kw)
    b.check()  # nothing is left behind


def test_cache_refuses_to_reserve_inside_a_graph() -> None:
    cache = BlockKVCache(4, num_heads=1, head_dim=64, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(BackendError):
            cache.reserve([3])
    assert cache.lengths == [] and len(cache.free_pages) == 4


def test_attention_rows_behind_the_last_sequence_stay() -> None:
    for new, lens in (([2, 1], [40, 9]), ([200, 3], [300, 9])):
        b = Batch("bf16", 4, 2, 64, 16, new, lens)
        q = torch.cat([b.q, torch.randn(5, 4, 64, device="cuda").bfloat16()])
        out = torch.full_like(q, 7.0)
        assert ops.paged_attention(q, *b.lists, out=out) is out
        assert torch.equal(out[:b.N], ops.paged_attention(b.q, *b.lists))
        assert (out[b.N:] == 7.0).all()


def test_attention_strided_operands() -> None:
    for new, lens, dt, D in (([3, 1], [40, 90], "bf16", 64), ([150], [400], "f16", 128), ([4], [30], "f32", 36)):
        b = Batch(dt, 6, 2, D, 16, new, lens)
        fused = torch.randn(b.N, 9, D + 3, device="cuda").to(b.dt)
        q = fused[:, 1:7, :D]
        q.copy_(b.q)
        out = torch.zeros(b.N, 6, D + 1, device="cuda", dtype=b.dt)[..., :D]
        ops.paged_attention(q, *b.lists, out=out)
        want, bound, _ = attention64(b.q, *b.lists)
        assert_within(out, want, bound, "strided q and out")
        wide = torch.full((b.key_pool.shape[0], 2, 16, D + 1), float("nan"), device="cuda", dtype=b.dt)
        odd = wide[..., :D]  # pool rows at odd addresses
        odd.copy_(b.key_pool)
        got = ops.paged_attention(b.q, odd, *b.lists[1:])
        assert_within(got, want, bound, "odd pool rows")
        table = torch.full((len(new), 2 * b.block_table.shape[1]), -1, dtype=torch.int32, device="cuda")
        half = table[:, :b.block_table.shape[1]]
        half.copy_(b.block_table)
        got = ops.paged_attention(b.q, *b.lists[:2], half, *b.lists[3:])
        assert_within(got, want, bound, "a table that is part of a wider one")


def test_attention_nan_and_infinity() -> None:
    """A query, key or value that is not finite reaches the rows that see it, as a softmax carries it."""
    b = Batch("bf16", 2, 1, 64, 16, [1, 1, 1, 1], [30, 30, 30, 30])
    table = b.block_table.tolist()
    b.key_pool[table[1][0], 0, 3, 5] = float("nan")
    b.value_pool[table[2][1], 0, 2, 9] = float("inf")
    b.q[3, 1, 0] = float("inf")
    out = ops.paged_attention(b.q, *b.lists).float()
    assert torch.isfinite(out[0]).all()
    assert torch.isnan(out[1]).all()
    assert torch.isinf(out[2, :, 9]).all() and torch.isfinite(out[2, :, :9]).all()
    assert torch.isfinite(out[3, 0]).all() and not torch.isfinite(out[3, 1]).any()
    b = Batch("f32", 2, 1, 64, 16, [1, 1, 1], [30, 30, 30])  # fp32: its parts of an infinity are formed again
    b.value_pool[int(b.block_table[0, 1]), 0, 2, 9] = float("-inf")
    b.q[2, 0, 0] = float("nan")
    minus = b.key_pool[int(b.block_table[1, 0]), 0, 3]
    minus.zero_()
    minus[5] = float("-inf")
    b.q[1, :, 5] = b.q[1, :, 5].abs() + 1  # that key scores -inf: no weight, and no NaN
    out = ops.paged_attention(b.q, *b.lists)
    assert (out[0, :, 9] == float("-inf")).all() and torch.isfinite(out[0, :, :9]).all()
    assert torch.isfinite(out[1]).all()
    assert torch.isnan(out[2, 0]).all() and torch.isfinite(out[2, 1]).all()
    # scores of -inf on every visible key: 0 / 0, as softmax over -inf
    b = Batch("f32", 1, 1, 64, 16, [1], [20])
    b.key_pool[b.block_table[0].long()] = 0
    b.key_pool[b.block_table[0].long(), :, :, 0] = float("-inf")
    b.q.zero_()
    b.q[..., 0] = 1
    assert torch.isnan(ops.paged_attention(b.q, *b.lists)).all()


@pytest.mark.parametrize("dt,D,page", [("bf16", 128, 16), ("f16", 64, 24), ("bf16", 72, 16), ("f32", 64, 16)])
@pytest.mark.parametrize("new,length,window", [(3, 40, 0), (60, 200, 0), (200, 200, 0), (200, 4000, 0), (70, 300, 50)])
def test_attention_unseen_keys_reach_no_row(dt, D, page, new, length, window) -> None:
    """A key or value that is not finite changes the rows that see it, and no other, whatever tile they share."""
    b = Batch(dt, 4, 2, D, page, [new, 1], [length, 30])
    clean = ops.paged_attention(b.q, *b.lists, window=window)
    at = length - new + new // 2  # a token in the middle of the new ones
    slot = int(b.block_table[0, at // page]), slice(None), at % page
    for pool, value in ((b.value_pool, float("nan")), (b.value_pool, float("inf")), (b.key_pool, float("nan"))):
        kept = pool[slot].clone()
        pool[slot] = value
        got = ops.paged_attention(b.q, *b.lists, window=window)
        pool[slot] = kept
        pos = length - new + torch.arange(new, device="cuda")
        sees = torch.zeros(b.N, dtype=torch.bool, device="cuda")
        sees[:new] = (pos >= at) & ((pos < at + window) if window else True)
        want, bound, _ = attention64(b.q, *b.lists, window=window)
        assert_within(got[~sees], want[~sees], bound[~sees], "rows that do not see it")
        assert not torch.isfinite(got[sees].float()).any()
    assert torch.equal(ops.paged_attention(b.q, *b.lists, window=window), clean)


@pytest.mark.parametrize("new,length", [(1, 700), (40, 700)])
def test_offsets_beyond_32_bits(new, length) -> None:
    """Pools of more than 2^32 elements each, with the pages in use at their end."""
    D, page = 128, 256
    pages = 2 ** 32 // (page * D) + 8
    b = Batch("bf16", 4, 1, D, page, [new], [length])
    used = b.block_table[0].long()
    key_pool, value_pool = (torch.empty(pages, 1, page, D, device="cuda", dtype=b.dt) for _ in range(2))
    far = torch.tensor([[pages - 1 - i for i in range(len(used))]], dtype=torch.int32, device="cuda")
    key_pool[far[0].long()], value_pool[far[0].long()] = b.key_pool[used], b.value_pool[used]
    want = ops.paged_attention(b.q, *b.lists)
    assert torch.equal(ops.paged_attention(b.q, key_pool, value_pool, far, b.kv_len, b.q_start), want)
    rot = RotaryEmbedding(D)
    ops.paged_append(b.k, b.v, *b.lists, rotary=rot)
    ops.paged_append(b.k, b.v, key_pool, value_pool, far, b.kv_len, b.q_start, rotary=rot)
    for big, small in ((key_pool, b.key_pool), (value_pool, b.value_pool)):
        assert torch.equal(big[far[0].long()].view(torch.int16), small[used].view(torch.int16))
    assert fault() == 0


def test_attention_large_scores_do_not_overflow() -> None:
    for new, lens in (([2], [300]), ([200], [500])):
        b = Batch("bf16", 4, 2, 128, 16, new, lens, scale=300.0)
        b.check("large scores")


def test_attention_bad_pages_are_read_as_zeros_and_reported() -> None:
    assert fault() == 0
    for new, lens in (([1], [64]), ([100], [160])):
        b = Batch("bf16", 4, 2, 64, 16, new, lens)
        want_table = b.block_table.clone()
        zero = int(b.key_pool.shape[0]) - 1
        used = set(b.block_table.flatten().tolist())
        zero = next(p for p in range(b.key_pool.shape[0]) if p not in used)
        b.key_pool[zero] = 0
        b.value_pool[zero] = 0
        want_table[0, 1], want_table[0, 2] = zero, zero
        want = ops.paged_attention(b.q, b.key_pool, b.value_pool, want_table, b.kv_len, b.q_start)
        assert fault() == 0
        for page in (-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1):
            b.block_table[0, 1] = page
            b.block_table[0, 2] = b.key_pool.shape[0]
            got = ops.paged_attention(b.q, *b.lists)
            assert fault() == 2
            assert torch.equal(got, want)


def test_attention_unsound_lists_are_reported_and_stay_inside() -> None:
    for new in ([2, 3], [90, 130]):
        lens = [150, 170]
        b = Batch("bf16", 2, 1, 64, 16, new, lens)
        N = b.N
        good = ops.paged_attention(b.q, *b.lists)
        # a length beyond the table's row is cut to it; the other sequence is unharmed
        kv = b.kv_len.clone()
        kv[1] = 10 ** 6
        got = ops.paged_attention(b.q, *b.lists[:3], kv, b.q_start)
        assert fault() == 2
        assert torch.equal(got[:new[0]], good[:new[0]])
        for bad in ([0, N + 1, N], [0, -5, N], [N, 0, 0], [2 ** 31 - 1, -2 ** 31, 5], [0, N, 0]):
            out = torch.full((N + 4, 2, 64), 3.0, device="cuda", dtype=b.dt)
            ops.paged_attention(b.q, *b.lists[:4], torch.tensor(bad, dtype=torch.int32, device="cuda"), out=out[:N])
            assert fault() == 2
            assert (out[N:] == 3.0).all()


def test_attention_overlapping_ranges_stay_inside_the_workspace() -> None:
    b = Batch("bf16", 2, 1, 64, 16, [40, 0, 0], [3000, 3000, 3000])
    starts = torch.tensor([0, 40, 0, 40], dtype=torch.int32, device="cuda")  # two sequences claim the same tokens
    ops.paged_attention(b.q, *b.lists[:4], starts)
    assert fault() == 2


def test_attention_graph_follows_the_lists() -> None:
    for new, lens, dt, D in (([1, 1, 1], [5, 300, 77], "bf16", 128), ([70, 1, 200], [90, 700, 300], "f16", 64)):
        b = Batch(dt, 8, 2, D, 16, new, lens, width=60)
        out = torch.empty_like(b.q)
        ops.paged_attention(b.q, *b.lists, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention(b.q, *b.lists, out=out)
        second = torch.cuda.CUDAGraph()
        out2 = torch.empty_like(b.q)
        with torch.cuda.graph(second):
            ops.paged_attention(b.q, *b.lists, out=out2)
        for cut in (0, 3, 5):
            b.kv_len.copy_(torch.tensor([n - cut for n in lens], dtype=torch.int32))
            b.q.copy_(torch.randn_like(b.q))
            out.fill_(9)
            graph.replay()
            second.replay()
            want, bound, _ = attention64(b.q, *b.lists)
            assert_within(out, want, bound, f"replay with lengths less {cut}")
            assert torch.equal(out, out2)


def test_attention_on_side_streams() -> None:
    batches = [Batch("bf16", 8, 2, 128, 16, [1, 90], [4000, 500], seed=s) for s in range(2)]
    want = [ops.paged_attention(b.q, *b.lists) for b in batches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in batches], []
    for _ in range(5):
        for s, b in zip(streams, batches):
            with torch.cuda.stream(s):
                got.append(ops.paged_attention(b.q, *b.lists))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2])


def test_attention_shared_prefix_pages() -> None:
    b = Batch("bf16", 4, 2, 64, 16, [1, 2], [70, 70])
    b.block_table[1, :4] = b.block_table[0, :4]
    b.check("two sequences on the same pages")


# -- the append ------------------------------------------------------------------------


APPENDS = [
    # dtype, H, Hkv, D, page, new, lens, embedding
    ("bf16", 32, 8, 128, 16, [1, 1, 1], [5, 17, 16], {}),
    ("f16", 4, 4, 64, 24, [40, 0, 3], [100, 10, 3], dict(interleaved=True)),
    ("f32", 2, 1, 40, 1, [7, 2], [9, 2], dict(rotary_dim=20)),
    ("bf16", 0, 2, 33, 5, [11], [30], dict(rotary_dim=32)),
    ("bf16", 3, 1, 72, 100, [150], [150], dict(sections=(9, 13, 14))),
    ("f16", 2, 2, 64, 16, [5], [20], None),  # no rotation: keys as they are
]


@pytest.mark.parametrize("slot_major", [False, True])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{c[0]}_D{c[3]}_p{c[4]}")
def test_append_matches_formula(case, slot_major) -> None:
    dt, H, Hkv, D, page, new, lens, kw = case
    b = Batch(dt, max(H, 1), Hkv, D, page, new, lens, slot_major=slot_major)
    rot = None if kw is None else RotaryEmbedding(D, **kw)
    before = b.key_pool.clone(), b.value_pool.clone()
    pos = torch.cat([torch.arange(n - t, n) for t, n in zip(new, lens)]).cuda()
    q = b.q if H else None
    out = ops.paged_append(b.k, b.v, *b.lists, q=q, rotary=rot)
    written = torch.zeros(b.key_pool.shape[:3:2], dtype=torch.bool, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    pages, slots = b.block_table[seq, pos // page].long(), pos % page
    written[pages, slots] = True
    if rot is None:
        assert torch.equal(b.key_pool[pages, :, slots], b.k)
        assert out is None or torch.equal(out, b.q)
    else:
        axes = pos.expand(rot.num_axes, -1)
        assert_within(b.key_pool[pages, :, slots].transpose(0, 1), *rotate64(b.k.transpose(0, 1), axes, rot), "keys")
        if H:
            assert_within(out.transpose(0, 1), *rotate64(b.q.transpose(0, 1), axes, rot), "queries")
            same = b.q.clone()
            assert ops.paged_append(b.k, b.v, *b.lists, q=same, rotary=rot, q_out=same) is same
            assert torch.equal(same, out)
        # the same values as the embedding on its own
        alone = rot(b.k.transpose(0, 1)[None], positions=pos)[0].transpose(0, 1)
        assert torch.equal(b.key_pool[pages, :, slots], alone)
    assert torch.equal(b.value_pool[pages, :, slots], b.v)
    for pool, old in zip((b.key_pool, b.value_pool), before):  # every other slot is as it was
        keep = ~written[:, None, :, None].expand_as(pool)
        assert torch.equal(pool[keep].view(torch.int32 if dt == "f32" else torch.int16),
                           old[keep].view(torch.int32 if dt == "f32" else torch.int16))
    assert fault() == 0


def test_append_positions_of_several_axes() -> None:
    b = Batch("bf16", 4, 2, 64, 16, [30, 6], [50, 6])
    rot = RotaryEmbedding(64, sections=(8, 12, 12))
    pos = torch.randint(0, 900, (3, b.N), device="cuda", dtype=torch.int32)
    q = ops.paged_append(b.k, b.v, *b.lists, q=b.q, rotary=rot, positions=pos)
    assert_within(q.transpose(0, 1), *rotate64(b.q.transpose(0, 1), pos[:, None], rot), "queries")


def test_append_skips_tokens_without_a_place() -> None:
    """Negative positions are quietly skipped, bad pages and full tables reported, rows behind the last one stay."""
    rot = RotaryEmbedding(64)
    b = Batch("bf16", 2, 1, 64, 16, [6, 2], [4, 20])  # the first sequence brings more tokens than it holds
    b.block_table[1, 1] = b.key_pool.shape[0]
    pool = b.key_pool.clone()
    q = torch.cat([b.q, b.q[:3]])
    out = torch.full_like(q, 5.0)
    k, v = torch.cat([b.k, b.k[:3]]), torch.cat([b.v, b.v[:3]])
    ops.paged_append(k, v, *b.lists, q=q, rotary=rot, q_out=out)
    assert fault() == 2
    changed = (b.key_pool.view(torch.int16) != pool.view(torch.int16)).any(-1).any(1)  # [pages, slots]
    want = torch.zeros_like(changed)
    want[int(b.block_table[0, 0]), :4] = True
    assert torch.equal(changed, want)
    assert (out[b.N:] == 5.0).all() and torch.isfinite(out[:b.N].float()).all()
    b = Batch("bf16", 2, 1, 64, 16, [2], [16])
    b.kv_len.fill_(17)  # one page in the table: the last token has no slot
    pool = b.value_pool.clone()
    ops.paged_append(b.k, b.v, *b.lists, rotary=rot)
    assert fault() == 2
    assert torch.equal(b.value_pool[b.block_table[0, 0], :, 15], b.v[0])
    b.value_pool[b.block_table[0, 0], :, 15] = pool[b.block_table[0, 0], :, 15]
    assert torch.equal(b.value_pool.view(torch.int16), pool.view(torch.int16))
    for bad in ([0, 3], [-1, 2], [2, 0], [2 ** 31 - 1, 0]):
        before = b.key_pool.clone()
        ops.paged_append(b.k, b.v, *b.lists[:4], torch.tensor(bad, dtype=torch.int32, device="cuda"), rotary=rot)
        if bad != [2 ** 31 - 1, 0]:
            assert fault() in (0, 2)
        assert torch.equal(b.key_pool.view(torch.int16), before.view(torch.int16))
    fault()


# -- the cache and the module -------------------------------------------------------------


def test_cache_serves_ragged_sequences() -> None:
    """Prompts, steps, an ended sequence whose pages another takes: every step's output against fp64 over the
    keys and values kept on the side."""
    rot = RotaryEmbedding(64)
    H, Hkv, D = 4, 2, 64
    cache = BlockKVCache(40, page_size=16, num_heads=Hkv, head_dim=D, rotary=rot, dtype=torch.bfloat16)
    kept_k: list[list[torch.Tensor]] = []
    kept_v: list[list[torch.Tensor]] = []
    r = random.Random(3)
    g = torch.Generator(device="cuda").manual_seed(3)

    def step(new):
        N = sum(new)
        q, k, v = (torch.randn(N, h, D, generator=g, device="cuda").bfloat16() for h in (H, Hkv, Hkv))
        past = cache.lengths + [0] * (len(new) - len(cache.lengths))
        out = cache.attend(q, k, v, new)
        at = 0
        for b, n in enumerate(new):
            if b == len(kept_k):
                kept_k.append([])
                kept_v.append([])
            if n:
                pos = torch.arange(past[b], past[b] + n, device="cuda")
                kept_k[b].append(rot(k[at:at + n].transpose(0, 1)[None], positions=pos)[0])
                kept_v[b].append(v[at:at + n].transpose(0, 1))
                kk, vv = torch.cat(kept_k[b], 1), torch.cat(kept_v[b], 1)
                qq = rot(q[at:at + n].transpose(0, 1)[None], positions=pos)[0].transpose(0, 1)
                L = kk.shape[1]
                lists = (kk[None], vv[None], torch.zeros(1, 1, dtype=torch.int32), torch.tensor([L]),
                         torch.tensor([0, n]))
                want, bound, _ = attention64(qq.contiguous(), *lists)
                assert_within(out[at:at + n], want, bound, f"sequence {b}")
            at += n

    step([30, 100])
    step([1, 1])
    step([0, 1, 50])
    with pytest.raises(NotInitializedError):
        cache.reserve([0, 0, 10000])
    assert cache.lengths == [31, 102, 50]
    free = len(cache.free_pages)
    cache.release(1)
    kept_k[1], kept_v[1] = [], []
    assert len(cache.free_pages) == free + 7 and cache.lengths == [31, 0, 50]
    step([1, 200, 3])
    for _ in range(4):
        step([r.randrange(3) for _ in range(3)])
    # a refused step leaves the cache as it was
    lengths, pages = list(cache.lengths), [list(p) for p in cache.pages]
    with pytest.raises(DtypeError):
        cache.attend(torch.zeros(3, H, D, device="cuda"), torch.zeros(3, Hkv, D, device="cuda"),
                     torch.zeros(3, Hkv, D, device="cuda"), [1, 1, 1])
    assert cache.lengths == lengths and cache.pages == pages
    state = cache.state_dict()
    other = BlockKVCache(60, page_size=16, num_heads=Hkv, head_dim=D, rotary=rot, dtype=torch.bfloat16)
    other.load_state_dict(state)
    cache, new = other, [1, 2, 40]
    step(new)
    assert fault() == 0


def _module(H, D, causal, rotary=None, mode="reference"):
    torch.manual_seed(11)
    cfg = AVQConfig(causal=causal, attention=AttentionShapeConfig(embed_dim=H * D, num_heads=H),
                    execution=ExecutionConfig(mode=mode))
    return AVQAttention(cfg, rotary=rotary).to("cuda", torch.bfloat16).requires_grad_(False)


@pytest.mark.parametrize("causal", [False, True])
def test_module_attends_over_the_block_cache(causal) -> None:
    """The dense path over pages against the same module over a concatenated cache: both are within the dense
    path's 5e-3 of the exact outputs (two bf16 roundings of scores up to about 4), so within 1e-2 of each other."""
    from avqa_b200 import InMemoryKVCache
    B, H, D = 3, 4, 64
    rot = RotaryEmbedding(D)
    m = _module(H, D, causal, rot)
    block = BlockKVCache(64, page_size=16, num_heads=H, head_dim=D, dtype=torch.bfloat16)
    plain = InMemoryKVCache(num_heads=H, head_dim_k=D, head_dim_v=D, device="cuda", dtype=torch.bfloat16)
    for T in (50, 1, 7, 1):
        x = torch.randn(B, T, H * D, device="cuda").bfloat16()
        a, b = m(x, x, x, kv_cache=block), m(x, x, x, kv_cache=plain)
        assert a.dtype == b.dtype and a.shape == b.shape
        assert (a.float() - b.float()).norm() <= 1e-2 * b.float().norm()
    k, v = block.lookup()
    ck, cv = plain.lookup()
    assert torch.equal(k, ck) and torch.equal(v, cv)


def test_module_rotates_by_positions_of_several_axes() -> None:
    B, H, D, T = 2, 2, 64, 24
    rot = RotaryEmbedding(D, sections=(8, 12, 12))
    m, bare = _module(H, D, False, rot), _module(H, D, False)
    x = torch.randn(B, T, H * D, device="cuda").bfloat16()
    pos = torch.randint(0, 50, (3, B, T), device="cuda")
    got = m(x, x, x, positions=pos)
    split = lambda t: t.view(B, T, H, D).transpose(1, 2)
    q, k = rot(split(bare.q_proj(x)), split(bare.k_proj(x)), positions=pos)
    out = ops.dense_attention(q, k, split(bare.v_proj(x)))
    assert torch.equal(got, bare.out_proj(out.transpose(1, 2).reshape(B, T, H * D)))
    block = BlockKVCache(16, page_size=8, num_heads=H, head_dim=D, dtype=torch.bfloat16)
    paged = m(x, x, x, kv_cache=block, positions=pos)
    assert (paged.float() - got.float()).norm() <= 1e-2 * got.float().norm()
    assert torch.equal(block.lookup()[0], k)
    with pytest.raises(BackendError):
        bare(x, x, x, positions=pos)
    with pytest.raises(BackendError):
        m(x, x, x, mask=torch.ones(T, T, dtype=torch.bool, device="cuda"), kv_cache=block)
    with pytest.raises(ShapeError):
        m(x[:, :4], x, x, positions=pos)


def test_module_quantized_path_rotates_and_refuses_the_block_cache() -> None:
    """The AVQ path over rotated keys: the module with an embedding equals the bare one on rotated projections."""
    B, H, D, T = 2, 2, 64, 96
    rot = RotaryEmbedding(D)
    torch.manual_seed(5)
    cfg = AVQConfig(attention=AttentionShapeConfig(embed_dim=H * D, num_heads=H))
    m = AVQAttention(cfg, in_proj=False, out_proj=False, rotary=rot)
    bare = AVQAttention(cfg, in_proj=False, out_proj=False)
    bare.codebook.parents, bare.codebook.children = m.codebook.parents.clone(), m.codebook.children.clone()
    q, k, v = (torch.randn(B, T, H * D, device="cuda").bfloat16() for _ in range(3))
    split = lambda t: t.view(B, T, H, D).transpose(1, 2)
    qr, kr = (x.transpose(1, 2).reshape(B, T, H * D) for x in rot(split(q), split(k)))
    assert torch.equal(m(q, k, v), bare(qr, kr, v))
    with pytest.raises(BackendError):
        m(q, k, v, kv_cache=BlockKVCache(4, num_heads=H, head_dim=D, dtype=torch.bfloat16))


def test_serving_run_of_the_three_operators() -> None:
    """Projection rows rotated, appended and attended to over several steps, through the ops as a program calls
    them, equal the same tokens in one prefill (each within its bounds of fp64)."""
    rot = RotaryEmbedding(128)
    H, Hkv, D, page, total = 8, 2, 128, 16, 75
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (torch.randn(total, h, D, generator=g, device="cuda").half() for h in (H, Hkv, Hkv))
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.randperm(8, device="cuda").to(torch.int32)[None, :5]
    pools = [torch.full((8, Hkv, page, D), float("nan"), device="cuda").half() for _ in range(2)]
    outs, at = [], 0
    for n in (40, 1, 1, 30, 3):
        rows = slice(at, at + n)
        at += n
        lists = (*pools, table, torch.tensor([at], **i32), torch.tensor([0, n], **i32))
        qr = ops.paged_append(k[rows], v[rows], *lists, q=q[rows], rotary=rot)
        outs.append(ops.paged_attention(qr, *lists))
    qr = rot(q.transpose(0, 1)[None])[0].transpose(0, 1).contiguous()
    lists = (*pools, table, torch.tensor([total], **i32), torch.tensor([0, total], **i32))
    want, bound, _ = attention64(qr, *lists)
    assert_within(torch.cat(outs), want, bound, "steps")
    assert_within(ops.paged_attention(qr, *lists), want, bound, "one prefill")
