"""The block cache's bookkeeping over many sequences and after refusals, without a GPU."""
from __future__ import annotations

import pytest
import torch

from avqa_b200 import BackendError, BlockKVCache, NotInitializedError, RotaryEmbedding, ShapeError, ops
from avqa_b200.parallel import CudaShardCompute, ShardedAVQAttention


def _cache(**kw):
    return BlockKVCache(**{**dict(num_pages=6, page_size=4, num_heads=2, head_dim=8, device="cpu"), **kw})


def _whole(c) -> bool:
    """Every page of the pool is held once, and the table's rows are the sequences' pages."""
    held = [p for pages in c.pages for p in pages]
    return sorted(held + c.free_pages) == list(range(c.num_pages)) and \
        all(c._table[b, :len(p)].tolist() == p for b, p in enumerate(c.pages))


@pytest.mark.parametrize("tokens", [1, 9])
def test_host_table_stays_small_as_sequences_come_one_by_one(tokens) -> None:
    c = _cache(num_pages=1000)
    for n in range(1, 301):
        batch = c.reserve([0] * (n - 1) + [tokens])
        need = -(-tokens // 4)
        assert batch.block_table.shape == (n, need) and batch.block_table.tolist() == c.pages
        assert c._table.numel() <= 2 * n * 2 * need  # each side at most doubled
    assert _whole(c)


def test_host_table_grows_with_one_sequence_up_to_the_pool() -> None:
    c = _cache(num_pages=50)
    for n in range(50):
        c.reserve([4])
        assert c._table.shape[0] == 1 and n < c._table.shape[1] <= min(50, 2 * (n + 1))
    assert c.pages == [list(range(50))] and c.free_pages == [] and _whole(c)


@pytest.mark.parametrize("call", ["empty", "zeros"])
def test_a_step_whose_memory_cannot_be_had_changes_nothing(call, monkeypatch) -> None:
    c = _cache()
    c.reserve([5, 1])
    before = list(c.lengths), [list(p) for p in c.pages], list(c.free_pages)

    def refuse(*args, **kw):
        raise RuntimeError("out of memory")

    monkeypatch.setattr(torch, call, refuse)
    with pytest.raises(RuntimeError):
        c.reserve([4, 1, 2])
    monkeypatch.undo()
    assert (c.lengths, c.pages, c.free_pages) == before and _whole(c)
    assert c.reserve([4, 1, 2]).kv_len.tolist() == [9, 2, 2] and _whole(c)


def test_a_state_that_does_not_fit_changes_nothing(monkeypatch) -> None:
    big = _cache(num_pages=12)
    big.reserve([30, 9])
    big.key_pool.copy_(torch.randn_like(big.key_pool))
    state = big.state_dict()
    c = _cache()
    c.reserve([5, 9])
    c.key_pool.copy_(torch.randn_like(c.key_pool))
    before = list(c.lengths), [list(p) for p in c.pages], list(c.free_pages), c.key_pool.clone()

    def same() -> bool:
        return (c.lengths, c.pages, c.free_pages) == before[:3] and torch.equal(c.key_pool, before[3]) and _whole(c)

    with pytest.raises(NotInitializedError):
        c.load_state_dict(state)
    assert same()
    small = _cache()
    small.reserve([4, 1])
    for bad in (dict(lengths=torch.tensor([5, 1])), dict(lengths=torch.tensor([8, -3])),
                dict(key_pages=small.key_pool[:1]), dict(value_pages=small.value_pool[:2, :1])):
        with pytest.raises(ShapeError):
            c.load_state_dict({**small.state_dict(), **bad})
        assert same()
    real = c.reserve
    monkeypatch.setattr(c, "reserve", lambda new: (real(new), 1 / 0))  # fails when the lists have changed already
    with pytest.raises(ZeroDivisionError):
        c.load_state_dict(small.state_dict())
    monkeypatch.undo()
    assert same()
    c.load_state_dict(small.state_dict())
    assert c.lengths == [4, 1] and _whole(c)
    c.load_state_dict(_cache().state_dict())  # an empty one
    assert c.lengths == [] and len(c.free_pages) == 6


@pytest.mark.parametrize("rotary", [None, RotaryEmbedding(8)])
def test_the_sharded_quantized_path_refuses_the_cache(rotary) -> None:
    """A quantized state of raw keys would ignore the cache's rotation, and outlive the sequences it covers."""
    sharded = ShardedAVQAttention.__new__(ShardedAVQAttention)
    sharded.h0, sharded.h1, sharded.D, sharded.world = 0, 2, 8, 1
    sharded.compute = CudaShardCompute.__new__(CudaShardCompute)
    sharded.compute.ops, sharded.compute.cb = ops, object()
    c = _cache(rotary=rotary)
    c.reserve([3])
    x = torch.zeros(1, 1, 16)
    with pytest.raises(BackendError, match="BlockKVCache"):
        sharded.forward(x, x, x, kv_cache=c)
    assert c.lengths == [3]


@pytest.mark.parametrize("change", [lambda c: c.reserve([1, 0]), lambda c: c.release(1), lambda c: c.reset(),
                                    lambda c: c.load_state_dict(c.state_dict())])
def test_what_changes_the_pages_drops_the_states_over_them(change) -> None:
    c = _cache()
    c.reserve([5, 2])
    c.quant_states["a module's"] = object()
    change(c)
    assert c.quant_states == {}


@pytest.mark.parametrize("shape", [(1, 4, 8), (3, 4, 8), (0, 4, 8), (2, 4, 16), (2, 8), (1, 2, 4, 8)])
def test_queries_that_are_not_the_new_tokens_are_refused(shape) -> None:
    """Without a rotation nothing else compared them with the step's tokens: missing rows were never written."""
    c = _cache()
    c.reserve([5])
    x = torch.zeros(2, 2, 8)
    with pytest.raises(ShapeError):
        c.attend(torch.zeros(shape), x, x, [1, 1])
    assert c.lengths == [5] and _whole(c)


def test_append_refuses_other_shapes_and_takes_no_tokens(monkeypatch) -> None:
    c = _cache()
    x = torch.zeros(2, 2, 3, 8)
    for key, value in ((x, x[:, :, :2]), (x, x[:1]), (x[:, :1], x[:, :1]), (x[..., :4], x[..., :4]), (x[0], x[0]),
                       (x.reshape(2, 1, 3, 16), x.reshape(2, 1, 3, 16))):
        with pytest.raises(ShapeError):
            c.append(key, value)
        assert c.lengths == []
    calls = []
    monkeypatch.setattr(ops, "paged_append", lambda k, v, *a, **kw: calls.append((k.shape, v.shape)))
    c.append(x[:, :, :0], x[:, :, :0])  # no token yet, of two sequences
    assert c.lengths == [0, 0] and calls == [((0, 2, 8), (0, 2, 8))]
    c.append(x, x)
    assert c.lengths == [3, 3] and calls[1] == ((6, 2, 8), (6, 2, 8))
