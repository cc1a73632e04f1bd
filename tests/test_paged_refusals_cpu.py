"""More of what the page pool's operators refuse, without a GPU."""
from __future__ import annotations

import pytest

from avqa_b200 import _lib
from test_paged_cpu import _append, _attention

MOST = 2 ** 31 - 1 - 65536  # tokens that a table's row may hold: the kernels step past the last key in 32 bits


@pytest.mark.parametrize("page_size,W", [(1, MOST + 1), (MOST + 1, 1), (2 ** 31 - 1, 1), (16, 2 ** 27 - 1),
                                         (65536, 32767)])
def test_tables_near_the_end_of_32_bits_are_refused(page_size, W) -> None:
    for call in (_append, _attention):
        assert call(page_size=page_size, W=W) == 1, _lib.last_error()
        assert str(MOST) in _lib.last_error()
        assert call(page_size=page_size, W=W, N=0) == 1
    assert _append(page_size=MOST, W=1, N=0) == 0 and _attention(page_size=1, W=MOST, B=0) == 0
