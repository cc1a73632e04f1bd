"""The dense path over a block cache up to the kernels, which stand-ins replace here."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from avqa_b200 import BackendError, BlockKVCache, RotaryEmbedding, ShapeError
from avqa_b200.attention_module import block_dense_path

B, H, T, D = 2, 3, 5, 8


def _run(monkeypatch, positions, sections):
    """What the append is given as positions."""
    seen = {}
    cache = BlockKVCache(8, page_size=4, num_heads=H, head_dim=D, device="cpu")
    m = SimpleNamespace(rotary=RotaryEmbedding(D, sections=sections), config=SimpleNamespace(causal=True),
                        dropout=lambda x: x, out_proj=lambda x: x)

    def append(k, v, *lists, q, rotary, positions):
        seen["positions"] = positions
        return q

    monkeypatch.setattr("avqa_b200.ops.paged_append", append)
    monkeypatch.setattr("avqa_b200.ops.paged_attention", lambda q, *lists, **kw: q)
    q, k, v = (torch.randn(B, H, T, D) for _ in range(3))
    out = block_dense_path(m, q, k, v, None, cache, positions=positions)
    assert torch.equal(out, q.transpose(1, 2).reshape(B, T, H * D)) and cache.lengths == [T, T]
    return seen["positions"]


@pytest.mark.parametrize("sections,shape", [(None, (T,)), (None, (1, T)), (None, (B, T)), (None, (1, 1, T)),
                                            (None, (1, B, T)), ((1, 3), (T,)), ((1, 3), (2, T)), ((1, 3), (2, 1, T)),
                                            ((1, 3), (2, B, T)), ((1, 1, 2), (3, B, T))])
def test_positions_become_the_packed_tokens_own(monkeypatch, sections, shape) -> None:
    pos = torch.arange(torch.Size(shape).numel()).view(shape)
    got = _run(monkeypatch, pos, sections)
    axes = 1 if sections is None else len(sections)
    whole = pos if len(shape) == 3 else pos[None] if axes == 1 or len(shape) == 1 else pos[:, None]
    whole = (whole if whole.dim() == 3 else whole[:, None]).expand(axes, B, T)
    assert torch.equal(got.expand(axes, -1) if got.dim() == 1 else got, whole.reshape(axes, B * T))


@pytest.mark.parametrize("sections,shape", [(None, ()), (None, (T + 1,)), (None, (B * T,)), (None, (3, T)),
                                            (None, (B, T - 1)), (None, (2, B, T)), (None, (1, 3, T)),
                                            ((1, 3), (3, T)), ((1, 3), (1, T)), ((1, 3), (1, B, T)),
                                            ((1, 3), (2, 3, T)), ((1, 3), (2, B, T, 1)), (None, (1, 1, B, T))])
def test_positions_that_do_not_fit_are_refused(monkeypatch, sections, shape) -> None:
    with pytest.raises(ShapeError):
        _run(monkeypatch, torch.zeros(shape, dtype=torch.int64), sections)


def test_positions_without_an_embedding_are_refused() -> None:
    m = SimpleNamespace(rotary=None)
    cache = BlockKVCache(8, page_size=4, num_heads=H, head_dim=D, device="cpu")
    x = torch.zeros(B, H, T, D)
    with pytest.raises(BackendError):
        block_dense_path(m, x, x, x, None, cache, positions=torch.arange(T))
