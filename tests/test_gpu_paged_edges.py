"""Attention over pages and the paged append on the GPU where they went wrong or could: cuts of many pairs, windows
behind which pages were given back, memory that overlaps, values that are not finite, widths between the tested ones."""
from __future__ import annotations

import pytest
import torch

from avqa_b200 import ops
from paged_reference import assert_within, attention64
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
