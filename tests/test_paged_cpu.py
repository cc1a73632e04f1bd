"""What the rotary embedding, the page pool's operators and the block cache
refuse, and the cache's bookkeeping, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from avqa_b200 import (AVQAttention, AVQConfig, BlockKVCache, ConfigurationError, DeviceError, NotInitializedError,
                       RotaryEmbedding, ShapeError, _lib, ops)

S2 = (ctypes.c_longlong * 2)(8, 8)
S3 = (ctypes.c_longlong * 3)(8, 8, 8)
FREQ = (ctypes.c_double * 4)(1, 1, 1, 1)
ANY = 16  # any non-null address: every case fails before a dereference


@pytest.mark.parametrize("kw", [dict(head_dim=0), dict(head_dim=258), dict(head_dim=64, rotary_dim=7),
                                dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=0),
                                dict(head_dim=64, base=0.0), dict(head_dim=64, base=float("nan")),
                                dict(head_dim=64, sections=(8, 8)),
                                dict(head_dim=64, sections=(40, -8)), dict(head_dim=64, frequencies=[1.0])])
def test_embedding_refuses_bad_configurations(kw) -> None:
    with pytest.raises(ConfigurationError):
        RotaryEmbedding(**kw)


def test_embedding_deals_out_its_frequencies() -> None:
    r = RotaryEmbedding(64, base=100.0, rotary_dim=32, sections=(4, 6, 6))
    assert r.num_axes == 3 and list(r.c_axes) == [0] * 4 + [1] * 6 + [2] * 6
    assert r.frequencies[0] == 1.0 and r.frequencies[8] == pytest.approx(100.0 ** -0.5, rel=1e-15)
    assert RotaryEmbedding(64).c_axes is None
    assert RotaryEmbedding(4, frequencies=[2.0, 3.0]).frequencies == (2.0, 3.0)


def test_operators_refuse_cpu_tensors() -> None:
    x = torch.zeros(1, 2, 3, 8)
    with pytest.raises(DeviceError):
        RotaryEmbedding(8)(x)
    lists = (torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(DeviceError):
        ops.paged_append(x[0], x[0], x, x, *lists)
    with pytest.raises(DeviceError):
        ops.paged_attention(x[0], x, x, *lists)


def _rotary(dtype=1, q=ANY, Hq=2, B=1, T=1, D=8, R=8, freq=FREQ, axes=None, num_axes=1, pos=None, pos_bytes=0,
            strides=S3):
    return _lib.load().avq_rotary(dtype, q, strides, Hq, None, None, 0, B, T, D, R, 0, freq, axes, num_axes, pos,
                                  pos_bytes, S3, 0, 0, ANY, S3, None, None, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), 1), (dict(q=None), 1), (dict(strides=None), 1), (dict(B=-1), 1), (dict(T=-1), 1),
    (dict(B=1 << 16, T=1 << 16), 1), (dict(D=0), 3), (dict(D=258), 3), (dict(R=7), 1), (dict(R=10), 1),
    (dict(freq=None), 1), (dict(num_axes=0), 1), (dict(axes=(ctypes.c_int * 4)(0, 1, 0, 0)), 1),
    (dict(pos=ANY, pos_bytes=2), 1), (dict(Hq=5000), 3)])
def test_rotary_entry_refuses(kw, code) -> None:
    assert _rotary(**kw) == code, _lib.last_error()
    assert _lib.last_error().startswith("avq_rotary")


def test_rotary_entry_of_nothing() -> None:
    assert _rotary(T=0, q=None) == 0 and _rotary(Hq=0, q=None) == 0


def _append(dtype=1, k=ANY, Hq=0, q=None, Hkv=2, D=8, pages=4, page_size=16, table=ANY, W=2, kv_len=ANY, B=1, N=1, R=8,
            freq=FREQ):
    return _lib.load().avq_paged_append(dtype, q, S2, Hq, q, S2, k, S2, ANY, S2, Hkv, D, ANY, S3, ANY, S3, pages,
                                        page_size, table, 2, W, kv_len, ANY, B, N, R, 0, freq, None, 1, None, 0, None,
                                        None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=-1), 1), (dict(k=None), 1), (dict(kv_len=None), 1), (dict(table=None), 1), (dict(Hq=2, q=None), 1),
    (dict(Hkv=0), 1), (dict(page_size=0), 1), (dict(W=-1), 1), (dict(pages=-1), 1), (dict(B=-1), 1), (dict(N=-1), 1),
    (dict(page_size=1 << 20, W=1 << 20), 1), (dict(D=300), 3), (dict(R=9), 1), (dict(freq=None), 1),
    (dict(Hkv=4000), 3)])
def test_append_entry_refuses(kw, code) -> None:
    assert _append(**kw) == code, _lib.last_error()
    assert _lib.last_error().startswith("avq_paged_append")


def _attention(dtype=1, q=ANY, H=4, Hkv=2, D=8, pages=4, page_size=16, table=ANY, W=2, B=1, N=1, causal=1, window=0,
               scale=1.0, most=0, ws=ANY, ws_bytes=1 << 40):
    return _lib.load().avq_paged_attention(dtype, q, S2, H, ANY, S3, ANY, S3, Hkv, D, pages, page_size, table, 2, W,
                                           ANY, ANY, B, N, causal, window, scale, most, ANY, S2, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=9), 1), (dict(q=None), 1), (dict(table=None), 1), (dict(H=3), 1), (dict(H=0), 1), (dict(Hkv=0), 1),
    (dict(D=0), 3), (dict(D=257), 3), (dict(page_size=0), 1), (dict(page_size=1 << 20, W=1 << 20), 1),
    (dict(window=-1), 1), (dict(causal=0, window=4), 1), (dict(scale=float("inf")), 1), (dict(scale=float("nan")), 1),
    (dict(most=-1), 1), (dict(N=1 << 30, H=1 << 10), 1), (dict(ws=None), 4), (dict(ws_bytes=8), 4)])
def test_attention_entry_refuses(kw, code) -> None:
    assert _attention(**kw) == code, _lib.last_error()
    assert _lib.last_error().startswith("avq_paged_attention")


def test_entries_of_nothing_and_workspace_query() -> None:
    lib = _lib.load()
    assert _append(N=0, k=None) == 0 and _append(B=0) == 0
    assert _attention(N=0, q=None, ws=None) == 0 and _attention(B=0) == 0
    size = lib.avq_paged_attention_workspace_size
    assert size(1, 2, 5, 8, 2, 128, 0) > 5 * 8 * 128 * 4
    for bad in ((7, 1, 1, 1, 1, 8, 0), (1, -1, 1, 1, 1, 8, 0), (1, 1, 1, 3, 2, 8, 0), (1, 1, 1, 1, 1, 300, 0)):
        assert size(*bad) == 0


def _cache(**kw):
    return BlockKVCache(**{**dict(num_pages=6, page_size=4, num_heads=2, head_dim=8, device="cpu"), **kw})


def test_block_cache_hands_out_and_takes_back_pages() -> None:
    c = _cache()
    assert c.size == 0 and c.lookup()[0].shape == (1, 2, 0, 8)
    b = c.reserve([5, 0])
    assert c.lengths == [5, 0] and [len(p) for p in c.pages] == [2, 0]
    assert b.kv_len.tolist() == [5, 0] and b.q_start.tolist() == [0, 5, 5] and b.max_q_len == 5 and b.tokens == 5
    assert b.block_table.shape == (2, 2) and b.block_table[0].tolist() == c.pages[0]
    b = c.reserve([3, 4, 1])
    assert c.lengths == [8, 4, 1] and [len(p) for p in c.pages] == [2, 1, 1] and b.q_start.tolist() == [0, 3, 7, 8]
    held = [p for pages in c.pages for p in pages] + c.free_pages
    assert sorted(held) == list(range(6))
    with pytest.raises(NotInitializedError):
        c.reserve([1, 1, 8])
    assert c.lengths == [8, 4, 1] and sorted([p for pages in c.pages for p in pages] + c.free_pages) == list(range(6))
    for bad in ([1], [1, 1, -1]):
        with pytest.raises(ShapeError):
            c.reserve(bad)
    c.release(0)
    assert c.lengths == [0, 4, 1] and len(c.free_pages) == 4 and c.size == 4
    with pytest.raises(ShapeError):
        c.release(3)
    with pytest.raises(ShapeError):
        c.lookup()
    c.reserve([16, 0, 0])
    assert len(c.free_pages) == 0
    c.reset()
    assert c.size == 0 and sorted(c.free_pages) == list(range(6))
    assert c.reserve([]).block_table.shape == (0, 1)


def test_block_cache_steps_that_are_refused_change_nothing() -> None:
    c = _cache()
    c.reserve([5])
    x = torch.zeros(2, 2, 8)
    with pytest.raises(DeviceError):  # the kernels need the GPU
        c.attend(x, x, x, [1, 1])
    assert c.lengths == [5] and len(c.pages) == 1 and len(c.free_pages) == 4
    for bad in ((x, x, [1]), (x[:, :1], x[:, :1], [1, 1]), (x, x[:1], [1, 1])):
        with pytest.raises(ShapeError):
            c.attend(x, *bad)
    rot = RotaryEmbedding(8)
    with pytest.raises(ConfigurationError):
        _cache(rotary=rot).attend(x, x, x, [1, 1], rotary=rot)


def test_block_cache_state_round_trip() -> None:
    c = _cache()
    c.reserve([5, 3])
    c.key_pool.copy_(torch.randn_like(c.key_pool))
    c.value_pool.copy_(torch.randn_like(c.value_pool))
    d = _cache(num_pages=9)
    d.load_state_dict(c.state_dict())
    assert d.lengths == c.lengths
    for mine, theirs in zip(c.pages, d.pages):
        assert torch.equal(c.key_pool[mine], d.key_pool[theirs]) and torch.equal(c.value_pool[mine], d.value_pool[theirs])
    with pytest.raises(ShapeError):
        _cache(page_size=8).load_state_dict(c.state_dict())


@pytest.mark.parametrize("kw", [dict(num_pages=0), dict(page_size=0), dict(num_heads=0), dict(head_dim=0),
                                dict(rotary=RotaryEmbedding(16))])
def test_block_cache_refuses_bad_configurations(kw) -> None:
    with pytest.raises(ConfigurationError):
        _cache(**kw)


def test_module_refuses_an_embedding_of_another_width() -> None:
    with pytest.raises(ConfigurationError):
        AVQAttention(AVQConfig(), rotary=RotaryEmbedding(32))
