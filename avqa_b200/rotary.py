"""Rotary positions of queries and keys, with one axis or several.

:class:`RotaryEmbedding` rotates the pairs of a head's first ``rotary_dim``
dimensions by ``position * frequency``.  Text has one position per token;
the patches of an image or a video have one per axis (time, height, width),
and ``sections`` deals the frequencies out to the axes in order.

The reference has no counterpart: its keys arrive rotated, as the long-context
workload's do (:func:`avqa_b200.workloads.rope_rotate`, whose half-split
pairing is the default here).
"""
from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch
from torch.autograd import forward_ad

from avqa_b200 import ops
from avqa_b200.exceptions import ConfigurationError, ShapeError


class RotaryEmbedding:
    """Rotation by positions: ``y_a = x_a cos t - x_b sin t``, ``y_b = x_a sin t + x_b cos t``.

    ``head_dim``     dimensions of a head (at most 256).
    ``base``         frequency ``i`` is ``base ** (-2 i / rotary_dim)``.
    ``rotary_dim``   dimensions that rotate (even; default all); the rest pass through.
    ``sections``     frequencies of each axis, summing to ``rotary_dim / 2``; default one axis.
    ``interleaved``  pairs are ``(2i, 2i + 1)`` instead of ``(i, i + rotary_dim / 2)``.
    ``frequencies``  radians per position of each pair, instead of ``base``'s.

    It holds host values only: any device and stream may use it, and a call
    can be captured into a CUDA graph.  (A backward pass captured into one needs,
    as every one of torch's does, that no eager graph over the same leaves is
    alive: their gradients are accumulated on the eager graph's stream.)
    """

    def __init__(self, head_dim: int, base: float = 10000.0, rotary_dim: int | None = None,
                 sections: Sequence[int] | None = None, interleaved: bool = False,
                 frequencies: Sequence[float] | None = None) -> None:
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if not 0 < head_dim <= 256:
            raise ConfigurationError(f"head_dim must be in [1, 256], got {head_dim}", {"head_dim": head_dim})
        if not 0 < rotary_dim <= head_dim or rotary_dim % 2:
            raise ConfigurationError(f"rotary_dim must be even and in [2, {head_dim}], got {rotary_dim}",
                                     {"rotary_dim": rotary_dim})
        if not base > 0:
            raise ConfigurationError(f"base must be > 0, got {base}", {"base": base})
        pairs = rotary_dim // 2
        sections = (pairs,) if sections is None else tuple(int(n) for n in sections)
        if any(n < 0 for n in sections) or sum(sections) != pairs or not 1 <= len(sections) <= 255:
            raise ConfigurationError(f"sections must sum to rotary_dim / 2 = {pairs}, got {sections}",
                                     {"sections": sections})
        if frequencies is None:
            frequencies = [float(base) ** (-2.0 * i / rotary_dim) for i in range(pairs)]
        frequencies = tuple(float(f) for f in frequencies)
        if len(frequencies) != pairs:
            raise ConfigurationError(f"{pairs} frequencies are needed, got {len(frequencies)}",
                                     {"frequencies": len(frequencies)})
        self.head_dim, self.rotary_dim, self.base = head_dim, rotary_dim, float(base)
        self.sections, self.interleaved, self.frequencies = sections, bool(interleaved), frequencies
        self.num_axes = len(sections)
        self._c_arrays()

    def __call__(self, q: torch.Tensor, k: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 offset: int = 0):
        """Rotate ``q [B, H, T, D]`` and, in the same launch, ``k [B, Hk, T, D]``
        (views with any b/h/t strides; fp32, bf16 or fp16).

        ``positions``: int32 or int64 on the same device, ``[T]`` for every
        batch entry and axis, with one axis ``[B, T]``, with several
        ``[axes, T]`` or ``[axes, B, T]``; without it token t is at
        ``offset + t``.  Returns the rotated tensor, or the pair with ``k``.
        Differentiable in ``q`` and ``k``, in reverse and forward mode and any
        number of times: the gradient is the rotation by the negative angle.
        (``torch.func`` transforms are refused by torch: the kernel has no
        batching rule.)
        """
        if q.dim() != 4 or (k is not None and k.dim() != 4):
            raise ShapeError("query and key must be [B, H, T, head_dim]", expected=4,
                             actual=(tuple(q.shape), None if k is None else tuple(k.shape)))
        if _recorded(q) or (k is not None and _recorded(k)):
            out = _Rotate.apply(self, positions, offset, False, q, k)
            return out[0] if k is None else out
        q_out, k_out = ops.rotary(self, q, k, positions, offset)
        return q_out if k is None else (q_out, k_out)

    def _c_arrays(self) -> None:
        pairs = self.rotary_dim // 2
        self.c_frequencies = (ctypes.c_double * pairs)(*self.frequencies)
        axes = [a for a, n in enumerate(self.sections) for _ in range(n)]
        self.c_axes = (ctypes.c_int * pairs)(*axes) if self.num_axes > 1 else None

    def __getstate__(self) -> dict:
        # the C arrays cannot be pickled, and a module that holds an embedding has to be
        return {name: x for name, x in self.__dict__.items() if name not in ("c_frequencies", "c_axes")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._c_arrays()

    def __repr__(self) -> str:
        return (f"RotaryEmbedding(head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, base={self.base}, "
                f"sections={self.sections}, interleaved={self.interleaved})")


def _recorded(x: torch.Tensor) -> bool:
    """Whether a derivative through ``x`` is wanted, in reverse or forward mode."""
    if x.requires_grad and torch.is_grad_enabled():
        return True
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None


class _Rotate(torch.autograd.Function):
    """The rotation and its transpose; both are the same kernel, so gradients of gradients work too."""

    @staticmethod
    def forward(ctx, rotary, positions, offset, reverse, q, k):
        ctx.args = (rotary, offset, reverse)
        if positions is not None:
            ctx.save_for_backward(positions)
            ctx.save_for_forward(positions)
        ctx.set_materialize_grads(False)
        if forward_ad._current_level >= 0:
            ctx.shapes = [None if x is None else (x.shape, x.dtype, x.device) for x in (q, k)]
        return ops.rotary(rotary, q, k, positions, offset, reverse)

    @staticmethod
    def _rotate(ctx, reverse, q, k):
        """The rotation of ``q`` and ``k``, either of which may be ``None``."""
        rotary, offset, _ = ctx.args
        saved = ctx.saved_tensors
        positions = saved[0] if saved else None
        # a gradient expanded along D (a sum's, say) has no unit stride there
        have = [x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous() for x in (q, k) if x is not None]
        if not have:
            return None, None
        second = have[1] if len(have) > 1 else None
        if any(_recorded(x) for x in have):  # a derivative of this one is wanted
            out = _Rotate.apply(rotary, positions, offset, reverse, have[0], second)
        else:
            out = ops.rotary(rotary, have[0], second, positions, offset, reverse)
        return (None, out[0]) if q is None else out

    @staticmethod
    def jvp(ctx, *tangents):
        out = _Rotate._rotate(ctx, ctx.args[2], tangents[4], tangents[5])
        # (an output whose input has no tangent still needs one)
        return tuple(torch.zeros(like[0], dtype=like[1], device=like[2]) if t is None and like is not None else t
                     for t, like in zip(out, ctx.shapes))

    @staticmethod
    def backward(ctx, gq, gk):
        gq, gk = _Rotate._rotate(ctx, not ctx.args[2], gq if ctx.needs_input_grad[4] else None,
                                 gk if ctx.needs_input_grad[5] else None)
        return None, None, None, None, gq, gk


__all__ = ["RotaryEmbedding"]
