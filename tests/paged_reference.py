"""Plain fp64 forms of the rotary embedding and of attention over pages, and
the error bounds that the GPU tests hold the kernels to.

Bounds are per element and count roundings: ``half(dtype)`` is the most that
one rounding to the dtype is off, relative to the value.

* Rotary.  Sine and cosine are within 2^-22 (the reduced angle in half turns
  rounds to fp32, off by at most 2^-25, times pi; sincospif adds its ulps), the
  two fp32 products and their sum round three times, the output once.
* Attention, out = sum p v / l over scores s:
  - a score's fp32 sum of D products is off by at most
    (D + 8) 2^-24 sum |q k| scale, and exp2 of it by a few 2^-23 more and by
    2^-22 |s| (the scaling by log2 e rounds); a relative error of p each;
  - p is rounded to the dtype (fp32 operands: split into tf32 parts, whose
    products are off by 2^-21 at most, in the scores too); below fp16's normal
    range by 2^-25 of the largest probability instead;
  - the tcgen05 kernel takes some exponentials from a polynomial, within 2^-13
    (bf16) or 2^-18 (fp16) of exp2; in p and in l;
  - the fp32 sums over L keys: L 2^-24;
  - each of these acts on sum p |v| / l at most, twice where it is in the
    numerator and in l;
  - the output's own rounding.
"""
from __future__ import annotations

import math

import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half the smallest step of the type (gradual underflow)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rotate64(x: torch.Tensor, positions: torch.Tensor, rotary, reverse: bool = False):
    """fp64 rotation of ``x [..., T, D]`` by ``positions [axes, ..., T]`` (broadcastable to x's
    leading dims), and the bound of a kernel's error."""
    x64 = x.double()
    y, size = x64.clone(), torch.zeros_like(x64)
    pairs = rotary.rotary_dim // 2
    axis = [a for a, n in enumerate(rotary.sections) for _ in range(n)]
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if rotary.interleaved else (i, i + pairs)
        t = positions[axis[i]].double() * rotary.frequencies[i] * (-1 if reverse else 1)
        c, s = t.cos(), t.sin()
        y[..., a] = x64[..., a] * c - x64[..., b] * s
        y[..., b] = x64[..., a] * s + x64[..., b] * c
        size[..., a] = size[..., b] = x64[..., a].abs() + x64[..., b].abs()
    bound = size * (2.0 ** -22 + 3 * 2.0 ** -24) + y.abs() * half(x.dtype) * (1 + 2.0 ** -10) + tiny(x.dtype)
    bound[..., 2 * pairs:] = 0  # copied
    if x.dtype != torch.float32:
        bound = bound + size * half(x.dtype) * 2.0 ** -10  # the fp32 error can move the value before it is rounded
        bound[..., 2 * pairs:] = 0
    return y, bound


def attention64(q, key_pool, value_pool, block_table, kv_len, q_start, causal=True, window=0, scale=None):
    """fp64 attention of a packed batch, its error bound, and the rows that belong to a sequence."""
    N, H, D = q.shape
    Hkv, page = key_pool.shape[1], key_pool.shape[2]
    G = H // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(N, H, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    rows = torch.zeros(N, dtype=torch.bool, device=q.device)
    dt = q.dtype
    part = 2.0 ** -21 if dt == torch.float32 else half(dt)
    poly = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -13, torch.float16: 2.0 ** -18}[dt]
    table, lens, starts = block_table.tolist(), kv_len.tolist(), q_start.tolist()
    for b, L in enumerate(lens):
        at, end = starts[b], starts[b + 1]
        n = end - at
        rows[at:end] = True
        if n == 0 or L == 0:
            continue
        pages = torch.tensor(table[b][:-(-L // page)], device=q.device, dtype=torch.long)
        k = key_pool[pages].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :L].repeat_interleave(G, 0)
        v = value_pool[pages].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :L].repeat_interleave(G, 0)
        qb = q[at:end].double().transpose(0, 1)
        pos = L - n + torch.arange(n, device=q.device)[:, None]
        j = torch.arange(L, device=q.device)[None]
        seen = torch.ones(n, L, dtype=torch.bool, device=q.device)
        if causal:
            seen &= j <= pos
        if window:
            seen &= j > pos - window
        s = (qb @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        off = qb.abs() @ k.abs().transpose(1, 2) * abs(scale)
        ds = off * ((D + 8) * 2.0 ** -24 + (2.0 ** -21 if dt == torch.float32 else 0)) + 2.0 ** -20 + \
            s.abs().masked_fill(~seen, 0) * 2.0 ** -21
        ds = ds.masked_fill(~seen, 0).amax(-1, keepdim=True)
        m = s.amax(-1, keepdim=True)
        p = torch.where(seen, (s - m.clamp(min=-1e300)).exp(), torch.zeros_like(s))
        l = p.sum(-1, keepdim=True)
        some = seen.any(-1)[None, :, None]
        o = torch.where(some, p @ v / l, torch.zeros((), dtype=torch.float64, device=q.device))
        weight = torch.where(some, p @ v.abs() / l, torch.zeros_like(o))
        few = torch.where(some, seen.double() @ v.abs() / l, torch.zeros_like(o)) * \
            (2.0 ** -25 if dt == torch.float16 else 2.0 ** -126)
        e = weight * (part + 2 * ds + 2 * poly + (L + 64) * 2.0 ** -24) + few
        e = e + (o.abs() + e) * half(dt) + tiny(dt)
        out[at:end], bound[at:end] = o.transpose(0, 1), e.transpose(0, 1)
    return out, bound, rows


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: got "
                             f"{got[tuple(i)].item()}, want {want[tuple(i)].item()} +- {bound[tuple(i)].item()}")
