"""A module with an embedding where its positions follow from caches and lengths, on the GPU."""
from __future__ import annotations

import pytest
import torch

from avqa_b200 import AVQAttention, AVQConfig, InMemoryKVCache, PagedKVCache, RotaryEmbedding
from avqa_b200.config import AttentionShapeConfig, ExecutionConfig

pytestmark = pytest.mark.gpu

B, H, D = 2, 2, 64


def _pair(mode, rot):
    """The same module with and without the embedding, both on their inputs as they are."""
    torch.manual_seed(5)
    cfg = AVQConfig(attention=AttentionShapeConfig(embed_dim=H * D, num_heads=H), execution=ExecutionConfig(mode=mode))
    m = AVQAttention(cfg, in_proj=False, out_proj=False, rotary=rot)
    bare = AVQAttention(cfg, in_proj=False, out_proj=False)
    bare.codebook.parents, bare.codebook.children = m.codebook.parents.clone(), m.codebook.children.clone()
    return m, bare


def _rotate(rot, x, offset):
    return rot(x.view(B, -1, H, D).transpose(1, 2), offset=offset).transpose(1, 2).reshape(x.shape)


@pytest.mark.parametrize("mode", ["optimized", "reference"])
@pytest.mark.parametrize("cache", ["paged", "memory"])
def test_steps_over_a_cache_rotate_behind_it(mode, cache) -> None:
    """A prompt and single tokens: the keys' positions go on where the cache ends, on both paths."""
    rot = RotaryEmbedding(D)
    m, bare = _pair(mode, rot)
    kw = dict(num_heads=H, head_dim_k=D, head_dim_v=D, device="cuda", dtype=torch.bfloat16)
    make = (lambda: PagedKVCache(page_size=16, **kw)) if cache == "paged" else (lambda: InMemoryKVCache(**kw))
    mine, theirs = make(), make()
    past = 0
    for T in (50, 1, 1, 7):
        q, k, v = (torch.randn(B, T, H * D, device="cuda").bfloat16() for _ in range(3))
        got = m(q, k, v, kv_cache=mine)
        want = bare(_rotate(rot, q, past), _rotate(rot, k, past), v, kv_cache=theirs)
        assert torch.equal(got, want)
        past += T
    assert torch.equal(mine.lookup()[0], theirs.lookup()[0])


@pytest.mark.parametrize("mode", ["optimized", "reference"])
@pytest.mark.parametrize("T,S", [(1, 40), (8, 40), (40, 8)])
def test_queries_and_keys_of_other_counts_end_together(mode, T, S) -> None:
    rot = RotaryEmbedding(D)
    m, bare = _pair(mode, rot)
    q = torch.randn(B, T, H * D, device="cuda").bfloat16()
    k, v = (torch.randn(B, S, H * D, device="cuda").bfloat16() for _ in range(2))
    assert torch.equal(m(q, k, v), bare(_rotate(rot, q, S - T), _rotate(rot, k, 0), v))
