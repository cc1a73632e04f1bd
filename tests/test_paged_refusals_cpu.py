"""More of what the page pool's operators refuse, without a GPU."""
from __future__ import annotations

import ctypes
import random

import pytest
import torch

from avqa_b200 import BackendError, _lib, ops
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


def _sets(t):
    """The bytes that a packed operand's rows cover."""
    n = t.element_size()
    return {t.storage_offset() * n + i * t.stride(0) * n + h * t.stride(1) * n + d
            for i in range(t.shape[0]) for h in range(t.shape[1]) for d in range(t.shape[2] * n)}


def _view(store, N, H, D, t, h, at):
    return store.as_strided((N, H, D), (t, h, 1), at)


def test_overlap_of_packed_operands_is_found() -> None:
    """Views of one memory by every kind of stride against the bytes that they cover."""
    r = random.Random(4)
    store = torch.zeros(4000, dtype=torch.bfloat16)
    seen = {True: 0, False: 0}
    for _ in range(1500):
        D = r.choice([1, 4, 8])
        N, H = r.randint(1, 6), r.randint(1, 5)
        h = r.choice([D, D + 3, 40, 2 * D])
        t = r.choice([H * h, 3 * H * h, H * h + 5, D, 0])
        if r.random() < 0.3:  # heads outermost
            t, h = h, t
        a = _view(store, N, H, D, t, h, r.randint(0, 150))
        H2 = r.choice([H, 1, 3])
        same = r.random() < 0.6
        b = _view(store, N, H2, D, t if same else r.choice([H2 * D, 17]), h if same else r.choice([D, 60]),
                  r.randint(0, 400))
        want = bool(_sets(a) & _sets(b))
        assert ops._overlap(a, b) == want and ops._overlap(b, a) == want, (a.shape, a.stride(), b.shape, b.stride())
        seen[want] += 1
    assert min(seen.values()) > 200
    fused = torch.zeros(7, 12, 16)
    q, k, v = fused[:, :8], fused[:, 8:10], fused[:, 10:]
    assert not ops._overlap(q, k) and not ops._overlap(k, v) and ops._overlap(q, fused[:, 7:9])
    assert not ops._overlap(q[:0], q) and ops._overlap(q, q[3:])


def test_attention_entry_refuses_a_shifted_workspace_and_negative_strides() -> None:
    """Vector loads of the workspace, and offsets whose sign says that a page is missing."""
    for shift in (1, 4, 8):
        assert _attention(ws=16 + shift) == 4, _lib.last_error()
    call = _lib.load().avq_paged_attention
    two, three = ctypes.c_longlong * 2, ctypes.c_longlong * 3
    for which in range(6):
        strides = [8] * 6
        strides[which] = -8
        assert call(1, 16, two(8, 8), 4, 16, three(*strides[:3]), 16, three(*strides[3:]), 2, 8, 4, 16, 16, 2, 2, 16, 16,
                    1, 1, 1, 0, 1.0, 0, 16, two(8, 8), 16, 1 << 40, None) == 1, _lib.last_error()
        assert "strides" in _lib.last_error()


def test_a_call_on_another_device_makes_it_current(monkeypatch) -> None:
    """A launch goes to the current device: a call for tensors of another one switches to it, and back."""
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *error):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    calls = []

    def entry(*args):
        calls.append((current[0], args))
        return 0

    ops._call("entry", entry, 0, 5)
    ops._call("entry", entry, 1, 6)
    assert calls == [(0, (5, 100)), (1, (6, 101))] and current == [0]
    with pytest.raises(BackendError):
        ops._call("entry", lambda *a: 1, 1)
    assert current == [0]
