"""The rotary embedding as an object, without a GPU."""
from __future__ import annotations

import copy
import io
import pickle

import pytest
import torch

from avqa_b200 import AVQAttention, AVQConfig, RotaryEmbedding
from avqa_b200.config import AttentionShapeConfig


@pytest.mark.parametrize("kw", [{}, dict(base=500.0, rotary_dim=32, sections=(4, 12), interleaved=True),
                                dict(rotary_dim=4, frequencies=[0.3, 1 / 3])])
@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda r: pickle.loads(pickle.dumps(r))])
def test_copies_and_pickles_rotate_alike(kw, again) -> None:
    r = RotaryEmbedding(64, **kw)
    s = again(r)
    for name in ("head_dim", "rotary_dim", "base", "sections", "interleaved", "frequencies", "num_axes"):
        assert getattr(r, name) == getattr(s, name)
    assert list(r.c_frequencies) == list(s.c_frequencies)
    assert (r.c_axes is None) == (s.c_axes is None) and list(r.c_axes or []) == list(s.c_axes or [])


def test_a_module_with_an_embedding_is_saved_whole() -> None:
    m = AVQAttention(AVQConfig(attention=AttentionShapeConfig(embed_dim=128, num_heads=2)),
                     rotary=RotaryEmbedding(64, base=777.0))
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    again = torch.load(file, weights_only=False)
    assert again.rotary.base == 777.0 and list(again.rotary.c_frequencies) == list(m.rotary.c_frequencies)
    assert all(torch.equal(a, b) for a, b in zip(m.state_dict().values(), again.state_dict().values()))
