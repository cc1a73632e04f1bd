"""Tensor-level wrappers of the C ABI: device state objects and the calls
that fill them.  Every tensor passed here must live on one CUDA device.

``PreparedCodebook``  the codebook in the input dtype plus squared norms.
``QuantState``        the quantized key set of one (batch, heads) block:
                      assignments, dtype aggregates, fp32 bucket sums, exact
                      int32 counts, per-(b,h) valid-parent counts and their
                      minimum (the routing budget's floor).
"""
from __future__ import annotations

from dataclasses import dataclass

import ctypes
import functools

import torch

from avqa_b200 import _lib
from avqa_b200.exceptions import BackendError, DeviceError, DtypeError, ShapeError


def _cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise DeviceError(f"{name} must be a CUDA tensor", expected="cuda", actual=str(t.device))


@dataclass
class PreparedCodebook:
    parents: torch.Tensor  # [H, M0, D] dtype
    children: torch.Tensor  # [H, M0, C, D] dtype
    p_sq: torch.Tensor  # [H, M0] fp32
    c_sq: torch.Tensor  # [H, M0, C] fp32

    @property
    def dims(self) -> tuple[int, int, int, int]:
        H, M0, C, D = self.children.shape
        return H, M0, C, D


def prepare_codebook(parents: torch.Tensor, children: torch.Tensor, dtype: torch.dtype,
                     device: torch.device) -> PreparedCodebook:
    """Cast the codebook to ``dtype`` on ``device`` and compute its norms."""
    lib = _lib.load()
    p32 = parents.detach().to(device=device, dtype=torch.float32).contiguous()
    c32 = children.detach().to(device=device, dtype=torch.float32).contiguous()
    H, M0, C, D = c32.shape
    if tuple(p32.shape) != (H, M0, D):
        raise BackendError("codebook parents/children shapes disagree",
                           {"parents": tuple(p32.shape), "children": tuple(c32.shape)})
    out = PreparedCodebook(torch.empty(H, M0, D, dtype=dtype, device=device),
                           torch.empty(H, M0, C, D, dtype=dtype, device=device),
                           torch.empty(H, M0, dtype=torch.float32, device=device),
                           torch.empty(H, M0, C, dtype=torch.float32, device=device))
    rc = lib.avq_prepare_codebook(_lib.dtype_code(dtype), p32.data_ptr(), c32.data_ptr(), H, M0, C, D,
                                  out.parents.data_ptr(), out.children.data_ptr(), out.p_sq.data_ptr(),
                                  out.c_sq.data_ptr(), _lib.stream_of(device))
    _lib.check(rc, "avq_prepare_codebook")
    return out


@dataclass
class QuantState:
    B: int
    H: int
    S: int
    dtype: torch.dtype
    passign: torch.Tensor | None  # [G, S] int32 (None in append-only decode states)
    cassign: torch.Tensor | None
    pagg: torch.Tensor  # [G, M0, D] dtype
    cagg: torch.Tensor  # [G, M0, C, D] dtype
    pacc: torch.Tensor | None  # [G, M0, D] fp32 bucket sums (decode)
    cacc: torch.Tensor | None
    pcnt: torch.Tensor  # [G, M0] int32
    ccnt: torch.Tensor  # [G, M0, C] int32
    nvalid: torch.Tensor  # [G] int32
    gmin: torch.Tensor  # [1] int32: min over (b,h) of nvalid

    def counts_in_dtype(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Counts as the reference reports them: saturating at 2^(mantissa+1)."""
        sat = {torch.bfloat16: 256, torch.float16: 2048, torch.float32: 1 << 24}[self.dtype]
        return self.pcnt.clamp(max=sat).to(self.dtype), self.ccnt.clamp(max=sat).to(self.dtype)


def quantize(keys: torch.Tensor, values: torch.Tensor, cb: PreparedCodebook, keep_sums: bool = False) -> QuantState:
    """Quantize ``keys``/``values`` ``[B, H, S, D]`` views (any b/h/s strides)."""
    lib = _lib.load()
    _cuda(keys, "keys")
    dev = keys.device
    B, H, S, D = keys.shape
    Hc, M0, C, Dc = cb.dims
    if Hc != H or Dc != D:
        raise BackendError("codebook does not match the keys", {"heads": (Hc, H), "head_dim": (Dc, D)})
    if values.shape != keys.shape:
        raise BackendError("keys and values must have identical shapes",
                           {"keys": tuple(keys.shape), "values": tuple(values.shape)})
    dt = keys.dtype
    G = B * H
    i32 = dict(dtype=torch.int32, device=dev)
    st = QuantState(
        B, H, S, dt,
        torch.empty(G, S, **i32),
        torch.empty(G, S, **i32),
        torch.empty(G, M0, D, dtype=dt, device=dev),
        torch.empty(G, M0, C, D, dtype=dt, device=dev),
        torch.empty(G, M0, D, dtype=torch.float32, device=dev) if keep_sums else None,
        torch.empty(G, M0, C, D, dtype=torch.float32, device=dev) if keep_sums else None,
        torch.empty(G, M0, **i32), torch.empty(G, M0, C, **i32), torch.empty(G, **i32),
        torch.full((1,), 2 ** 31 - 1, **i32))
    ws_bytes = lib.avq_quantize_workspace_size(B, H, S, M0)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    rc = lib.avq_quantize(_lib.dtype_code(dt), keys.data_ptr(), _lib.strides3(keys), values.data_ptr(),
                          _lib.strides3(values), B, H, S, D, M0, C, cb.parents.data_ptr(), cb.p_sq.data_ptr(),
                          cb.children.data_ptr(), cb.c_sq.data_ptr(), _lib.ptr(st.passign), _lib.ptr(st.cassign),
                          st.pagg.data_ptr(), st.cagg.data_ptr(), _lib.ptr(st.pacc), _lib.ptr(st.cacc),
                          st.pcnt.data_ptr(), st.ccnt.data_ptr(), st.nvalid.data_ptr(), st.gmin.data_ptr(),
                          ws.data_ptr(), ws_bytes, _lib.stream_of(dev))
    _lib.check(rc, "avq_quantize")
    if G == 0:
        st.gmin.zero_()
    return st


def append(state: QuantState, k: torch.Tensor, v: torch.Tensor, cb: PreparedCodebook,
           kpage: torch.Tensor | None = None, vpage: torch.Tensor | None = None, slot0: int = 0) -> None:
    """Append ``k``/``v`` ``[B, H, Tn, D]`` to ``state`` in key order (and
    optionally write them into page slots ``slot0..`` of ``kpage``/``vpage``
    ``[B, H, page_size, D]``); refreshes ``state.gmin``."""
    lib = _lib.load()
    if state.pacc is None:
        raise BackendError("this quantization state keeps no fp32 bucket sums; quantize with keep_sums=True")
    B, H, Tn, D = k.shape
    _, M0, C, _ = cb.dims
    dev = k.device
    ws_bytes = lib.avq_append_workspace_size(B, H, Tn)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    rc = lib.avq_append(_lib.dtype_code(k.dtype), k.data_ptr(), _lib.strides3(k), v.data_ptr(), _lib.strides3(v),
                        B, H, Tn, D, M0, C, cb.parents.data_ptr(), cb.p_sq.data_ptr(), cb.children.data_ptr(),
                        cb.c_sq.data_ptr(), state.pacc.data_ptr(), state.cacc.data_ptr(), state.pagg.data_ptr(),
                        state.cagg.data_ptr(), state.pcnt.data_ptr(), state.ccnt.data_ptr(), state.nvalid.data_ptr(),
                        _lib.ptr(kpage), _lib.ptr(vpage), _lib.strides3(kpage) if kpage is not None else None,
                        slot0, ws.data_ptr(), ws_bytes, _lib.stream_of(dev))
    _lib.check(rc, "avq_append")
    state.S += Tn
    state.passign = None  # per-key assignments are not tracked across appends
    state.cassign = None
    rc = lib.avq_reduce_min(state.nvalid.data_ptr(), state.nvalid.numel(), state.gmin.data_ptr(),
                            _lib.stream_of(dev))
    _lib.check(rc, "avq_reduce_min")


def codeword_presence(state: QuantState, T: int, mask: torch.Tensor | None = None, causal_offset: int | None = None,
                      query_batch: int | None = None) -> torch.Tensor:
    """Codeword visibility bits ``[Bq*H, T, ceil(M0/32)]`` int32 for ``T``
    queries per (b,h) (pipeline.py:82-106): a parent is visible to a query
    when one of its keys is allowed by the mask.

    ``mask``: bool/uint8 ``[T, S]`` or ``[B, H, T, S]`` (True = attend; size-1
    leading dims broadcast); without it the causal mask, query t seeing keys
    ``0 .. t + causal_offset`` (the reference uses ``S - T``).  ``query_batch``
    is the query batch when the state (batch 1) serves several."""
    from avqa_b200.exceptions import NotInitializedError
    lib = _lib.load()
    if state.passign is None:
        raise NotInitializedError("the codeword mask needs the key assignments of this state (not kept after a "
                                  "decode append)")
    dev = state.pcnt.device
    Bq = state.B if query_batch is None else query_batch
    H, S, M0 = state.H, state.S, state.pcnt.shape[-1]
    W = lib.avq_presence_words(M0)
    out = torch.empty(Bq * H, T, W, dtype=torch.int32, device=dev)
    m, strides = _mask_operand(mask, Bq, H, T, S, dev)  # m stays referenced until the kernel is enqueued
    offset = (S - T) if causal_offset is None else causal_offset
    ws_bytes = lib.avq_presence_workspace_size(H, M0, state.B) if m is None else 0
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    rc = lib.avq_codeword_presence(_lib.ptr(state.passign), Bq, H, S, M0, T, state.B, _lib.ptr(m), strides, offset,
                                   out.data_ptr(), ws.data_ptr(), ws_bytes, _lib.stream_of(dev))
    _lib.check(rc, "avq_codeword_presence")
    return out


def _mask_operand(mask: torch.Tensor | None, B: int, H: int, T: int, S: int, dev):
    """(uint8 mask tensor or None, ctypes strides {b, h, t} or None) of a
    rank-2 [T, S] or rank-4 [B|1, H|1, T, S] mask (True = attend)."""
    from avqa_b200.exceptions import ConfigurationError, ShapeError
    if mask is None:
        return None, None
    if mask.ndim not in (2, 4):
        raise ConfigurationError("mask must be rank 2 [T_q, T_k] or rank 4 [B, H, T_q, T_k]", {"got_rank": mask.ndim})
    if tuple(mask.shape[-2:]) != (T, S):
        raise ShapeError("mask shape does not match the queries and keys", expected=(T, S),
                         actual=tuple(mask.shape[-2:]))
    m = mask.to(device=dev, dtype=torch.uint8)
    if m.stride(-1) != 1:
        m = m.contiguous()
    if m.ndim == 2:
        st = (0, 0, m.stride(0))
    else:
        if m.shape[0] not in (1, B) or m.shape[1] not in (1, H):
            raise ShapeError("rank-4 mask does not broadcast to [B, H, T, S]", expected=(B, H, T, S),
                             actual=tuple(m.shape))
        st = (m.stride(0) if m.shape[0] > 1 else 0, m.stride(1) if m.shape[1] > 1 else 0, m.stride(2))
    return m, (ctypes.c_longlong * 3)(*st)


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    mask: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(mask(q k^T / sqrt(D))) v for ``[B, H, T|N, D]`` views, in the
    input dtype (backend.py:190-203); returns a ``[B, H, T, D]`` view."""
    lib = _lib.load()
    _cuda(q, "query")
    B, H, T, D = q.shape
    N = k.shape[2]
    dev = q.device
    out = torch.empty(B, T, H, D, dtype=q.dtype, device=dev).permute(0, 2, 1, 3)
    m, mst = _mask_operand(mask, B, H, T, N, dev)
    rc = lib.avq_dense_attention(_lib.dtype_code(q.dtype), q.data_ptr(), _lib.strides3(q), k.data_ptr(),
                                 _lib.strides3(k), v.data_ptr(), _lib.strides3(v), B, H, T, N, D, _lib.ptr(m), mst,
                                 out.data_ptr(), _lib.strides3(out), _lib.stream_of(dev))
    _lib.check(rc, "avq_dense_attention")
    return out


def bcar_update(keys: torch.Tensor, state: QuantState, parents: torch.Tensor, children: torch.Tensor,
                decay: float) -> None:
    """BCAR (online_adaptation.py:37-127): adapt ``children`` [H, M0, C, D]
    toward the means of the keys ``[B, H, S, D]`` that ``state`` assigned to
    each child cell and re-derive ``parents`` [H, M0, D] as their children's
    means, in place, in the codebook dtype (= the keys' dtype)."""
    from avqa_b200.exceptions import NotInitializedError
    lib = _lib.load()
    if state.passign is None:
        raise NotInitializedError("BCAR needs the key assignments of this state (not kept after a decode append)")
    B, H, S, D = keys.shape
    _, M0, C, _ = children.shape
    dev = keys.device
    new_c = torch.empty_like(children)
    new_p = torch.empty_like(parents)
    ws_bytes = lib.avq_bcar_workspace_size(B, H, M0, C, D)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    rc = lib.avq_bcar_update(_lib.dtype_code(keys.dtype), keys.data_ptr(), _lib.strides3(keys),
                             _lib.ptr(state.passign), _lib.ptr(state.cassign), B, H, S, D, M0, C, float(decay),
                             children.data_ptr(), new_c.data_ptr(), new_p.data_ptr(), ws.data_ptr(), ws_bytes,
                             _lib.stream_of(dev))
    _lib.check(rc, "avq_bcar_update")
    children.copy_(new_c)
    parents.copy_(new_p)


@dataclass
class ForwardDiagnostics:
    importance: torch.Tensor  # [G, M0] fp32 (pre-HVAQ importance, dtype values)
    selected: torch.Tensor  # [G, stride] int32, -1 padded, pass after pass
    pass_counts: torch.Tensor  # [passes] int32
    stride: int
    caps: list[int]

    def selections(self) -> list[torch.Tensor]:
        """Per pass, the ``[G, n_k]`` selected parent indices."""
        out, off = [], 0
        counts = self.pass_counts.tolist()
        for cap, n in zip(self.caps, counts):
            if n > 0:
                out.append(self.selected[:, off:off + n])
            off += cap
        return out


def pass_caps(P: int, passes: int, decay: float) -> list[int]:
    return [max(1, round(P * (decay ** i))) if i else P for i in range(passes)]


def forward(q: torch.Tensor, cb: PreparedCodebook, st: QuantState, P: int, passes: int = 1, pass_decay: float = 1.0,
            hvaq: int = 0, beta0: float = 0.0, alpha: float = 1.0, out: torch.Tensor | None = None,
            min_valid: torch.Tensor | None = None, diagnostics: bool = False,
            min_valid_ready: torch.cuda.Event | None = None, present: torch.Tensor | None = None):
    """AVQ attention of ``q`` ``[B, H, T, D]`` over ``st``.

    ``st`` holds either B batches of keys, or one batch that every query
    batch attends to (query chunks of one sequence over keys quantized once;
    each batch entry is routed on its own, exactly as separate calls over the
    same keys).  ``min_valid_ready``: an event recorded after ``min_valid``
    was produced on another stream; the library waits on it only right
    before routing.  ``present``: codeword visibility bits of a mask
    (:func:`codeword_presence`) for these queries.

    Returns ``out`` as a ``[B, H, T, D]`` fp32 view (module layout when
    ``out`` is given as a ``[B, T, H, D]``-strided tensor) and optional
    diagnostics.
    """
    lib = _lib.load()
    _cuda(q, "query")
    B, H, T, D = q.shape
    _, M0, C, _ = cb.dims
    dev = q.device
    if st.B != B and st.B != 1:
        raise BackendError("quantized state batch must equal the query batch or be 1",
                           {"state_batch": st.B, "query_batch": B})
    if out is None:
        out = torch.empty(B, T, H, D, dtype=torch.float32, device=dev).permute(0, 2, 1, 3)
    ws_bytes = lib.avq_forward_workspace_size(_lib.dtype_code(q.dtype), B, H, T, D, M0, C, P, passes, pass_decay, hvaq)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    diag = None
    imp = sel = pc = None
    if diagnostics:
        stride = lib.avq_selection_stride(P, passes, pass_decay)
        imp = torch.empty(B * H, M0, dtype=torch.float32, device=dev)
        sel = torch.full((B * H, stride), -1, dtype=torch.int32, device=dev)
        pc = torch.zeros(passes, dtype=torch.int32, device=dev)
        diag = ForwardDiagnostics(imp, sel, pc, stride, pass_caps(P, passes, pass_decay))
    mv = st.gmin if min_valid is None else min_valid
    rc = lib.avq_forward(_lib.dtype_code(q.dtype), q.data_ptr(), _lib.strides3(q), B, H, T, D, M0, C,
                         cb.parents.data_ptr(), cb.children.data_ptr(), st.pagg.data_ptr(), st.cagg.data_ptr(),
                         st.pcnt.data_ptr(), st.ccnt.data_ptr(), st.B, mv.data_ptr(),
                         None if min_valid_ready is None else min_valid_ready.cuda_event, _lib.ptr(present), P,
                         passes, pass_decay,
                         hvaq, beta0, alpha, out.data_ptr(), _lib.strides3(out), _lib.ptr(imp), _lib.ptr(sel),
                         _lib.ptr(pc), ws.data_ptr(), ws_bytes, _lib.stream_of(dev))
    _lib.check(rc, "avq_forward")
    return out, diag


# -- rotary positions, the paged append and paged attention ---------------------------

_POSITION_BYTES = {torch.int32: 4, torch.int64: 8}


def _call(what: str, fn, index: int, *args) -> None:
    """``fn(*args, stream)`` on the current stream of device ``index`` (made current where it is
    not: a launch goes to the current device), its status checked."""
    if index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, what)


def _cuda_index(t: torch.Tensor, name: str) -> int:
    index = t.get_device()
    if index < 0:
        _cuda(t, name)
    return index


def _same(name: str, t: torch.Tensor, index: int, dtype: torch.dtype) -> None:
    if t.get_device() != index:
        raise DeviceError(f"{name} must be on the same device", expected=f"cuda:{index}", actual=str(t.device))
    if t.dtype != dtype:
        raise DtypeError(f"{name} has the wrong dtype", expected=str(dtype), actual=str(t.dtype))


def _positions_operand(positions: torch.Tensor | None, axes: int, B: int, T: int, index: int):
    """(pointer, bytes, strides (axis, b, t)) of positions ``[T]``, ``[B, T]`` with one axis, or
    ``[axes, T]`` / ``[axes, B, T]``."""
    if positions is None:
        return None, 0, (0, 0, 0)
    if positions.get_device() != index:
        raise DeviceError("positions must be on the same device", expected=f"cuda:{index}",
                          actual=str(positions.device))
    nbytes = _POSITION_BYTES.get(positions.dtype)
    if nbytes is None:
        raise DtypeError("positions must be int32 or int64", expected="int32 | int64", actual=str(positions.dtype))
    shape, st = tuple(positions.shape), positions.stride()
    ok = 1 <= len(shape) <= 3 and shape[-1] == T
    if len(shape) == 1:
        strides = (0, 0, st[0])
    elif len(shape) == 2 and axes == 1:
        ok = ok and shape[0] in (1, B)
        strides = (0, st[0] if shape[0] > 1 else 0, st[1])
    elif len(shape) == 2:
        ok = ok and shape[0] == axes
        strides = (st[0], 0, st[1])
    elif len(shape) == 3:
        ok = ok and shape[0] == axes and shape[1] in (1, B)
        strides = (st[0], st[1] if shape[1] > 1 else 0, st[2])
    if not ok:
        raise ShapeError("positions do not fit the tokens", expected=f"[{T}] or [{axes} axes, {B}, {T}]", actual=shape)
    return positions.data_ptr(), nbytes, strides


@functools.lru_cache(maxsize=4096)
def _rotary_layout(q: tuple, q_strides: tuple, q_out_strides: tuple, k: tuple | None, k_strides: tuple | None,
                   k_out_strides: tuple | None, head_dim: int) -> tuple:
    """Check the shapes and strides of a rotation; (B, heads of q and k, T, D, stride arrays of
    q, k and their outputs).  The same layouts come again on every step."""
    if len(q) != 4:
        raise ShapeError("query and key must be [B, H, T, head_dim]", expected=4, actual=tuple(q))
    B, H, T, D = q
    if D != head_dim:
        raise ShapeError("the rotary embedding's head_dim differs from the query's", expected=head_dim, actual=D)
    if k is not None and (len(k) != 4 or k[0] != B or k[2] != T or k[3] != D):
        raise ShapeError("key must have the query's batch, tokens and head_dim", expected=(B, "Hk", T, D),
                         actual=tuple(k))
    arrays = []
    for st in (q_strides, k_strides, q_out_strides, k_out_strides):
        if st is not None and st[3] != 1 and D > 1:
            raise BackendError("operand must be a 4-D view with a contiguous last dimension", {"stride": tuple(st)})
        arrays.append(None if st is None else _lib.longs(*st[:3]))
    return B, H, 0 if k is None else k[1], T, D, *arrays


def rotary(embedding, q: torch.Tensor, k: torch.Tensor | None = None, positions: torch.Tensor | None = None,
           offset: int = 0, reverse: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotate ``q [B, H, T, D]`` and ``k [B, Hk, T, D]`` (or ``None``) by a
    :class:`~avqa_b200.rotary.RotaryEmbedding` (by the negative angle with
    ``reverse``) into new tensors; no gradient is recorded here."""
    lib = _lib.load()
    at, dt = _cuda_index(q, "query"), q.dtype
    q_out = torch.empty_like(q)
    kp = kop = k_out = None
    if k is None:
        B, H, Hk, T, D, qs, ks, qos, kos = _rotary_layout(q.shape, q.stride(), q_out.stride(), None, None, None,
                                                          embedding.head_dim)
    else:
        _same("key", k, at, dt)
        k_out = torch.empty_like(k)
        kp, kop = k.data_ptr(), k_out.data_ptr()
        B, H, Hk, T, D, qs, ks, qos, kos = _rotary_layout(q.shape, q.stride(), q_out.stride(), k.shape, k.stride(),
                                                          k_out.stride(), embedding.head_dim)
    pos, pos_bytes, pos_strides = _positions_operand(positions, embedding.num_axes, B, T, at)
    _call("avq_rotary", lib.avq_rotary, at, _lib.dtype_code(dt), q.data_ptr(), qs, H, kp, ks, Hk, B, T, D,
          embedding.rotary_dim, embedding.interleaved, embedding.c_frequencies, embedding.c_axes, embedding.num_axes,
          pos, pos_bytes, _lib.longs(*pos_strides), offset, reverse, q_out.data_ptr(), qos, kop, kos)
    return q_out, k_out


def _packed(t: torch.Tensor, name: str, heads: int, tokens: int, dim: int) -> ctypes.Array:
    """Element strides (token, head) of a packed ``[tokens, heads, dim]`` operand."""
    if t.shape != (tokens, heads, dim):
        raise ShapeError(f"{name} must be packed [tokens, heads, head_dim]", expected=(tokens, heads, dim),
                         actual=tuple(t.shape))
    st = t.stride()
    if st[2] != 1 and dim > 1:
        raise BackendError(f"{name} must have a contiguous last dimension", {"stride": st})
    return _lib.longs(st[0], st[1])


@functools.lru_cache(maxsize=4096)
def _rows_meet(delta: int, width: int, a: tuple, b: tuple) -> bool:
    """Whether any row of ``b`` shares memory with a row of ``a``; each is (tokens, heads, bytes from
    token to token, from head to head), with rows of ``width`` bytes, and b begins ``delta`` bytes
    behind a."""
    (Na, Ha, ta, ha), (Nb, Hb, tb, hb) = a, b
    if (ta, ha) == (tb, hb):  # as rows of one grid
        for dh in range(1 - Ha, Hb):
            rest = -(delta + dh * ha)  # what dt tokens have to make up for
            for dt in (rest // ta, rest // ta + 1) if ta else (0,):
                if abs(rest - min(max(dt, 1 - Na), Nb - 1) * ta) < width:
                    return True
        return False
    if Na * Ha + Nb * Hb > 1 << 22:
        return True  # (grids of different strides, woven into each other: not looked into)
    mine, theirs = (((torch.arange(N) * t)[:, None] + torch.arange(H) * h).flatten().sort()[0]
                    for N, H, t, h in (a, b))
    theirs = theirs + delta
    at = torch.searchsorted(mine, theirs)
    gap = torch.minimum((mine[at.clamp(max=len(mine) - 1)] - theirs).abs(), (mine[(at - 1).clamp(min=0)] - theirs).abs())
    return bool((gap < width).any())


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two packed ``[tokens, heads, dim]`` operands of one dtype and dim share memory."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (Na, Ha, D), (Nb, Hb, _), n = a.shape, b.shape, a.element_size()
    (ta, ha, _), (tb, hb, _) = a.stride(), b.stride()
    delta = b.data_ptr() - a.data_ptr()
    if delta >= ((Na - 1) * ta + (Ha - 1) * ha + D) * n or -delta >= ((Nb - 1) * tb + (Hb - 1) * hb + D) * n:
        return False
    return _rows_meet(delta, D * n, (Na, Ha, ta * n, ha * n), (Nb, Hb, tb * n, hb * n))


def _packed_shape(t: torch.Tensor, name: str) -> torch.Size:
    if t.dim() != 3:
        raise ShapeError(f"{name} must be packed [tokens, heads, head_dim]", expected="[N, H, D]",
                         actual=tuple(t.shape))
    return t.shape


@functools.lru_cache(maxsize=4096)
def _pool_layout(keys: tuple, key_strides: tuple, values: tuple, value_strides: tuple, table: tuple,
                 table_strides: tuple, lens: tuple, len_strides: tuple, starts: tuple, start_strides: tuple,
                 D: int) -> tuple:
    """Check a pool's and a batch's shapes and strides; (heads, the pools' stride arrays, pages,
    page size, table row stride and width, batch).  The same layouts come again on every step."""
    if len(keys) != 4 or keys[3] != D or values != keys:
        raise ShapeError("pools must be [pages, heads, page_size, head_dim], the values' like the keys'",
                         expected=("pages", "heads", "page_size", D), actual=(tuple(keys), tuple(values)))
    if D > 1 and (key_strides[3] != 1 or value_strides[3] != 1):
        raise BackendError("pools must have a contiguous last dimension",
                           {"stride": (tuple(key_strides), tuple(value_strides))})
    if len(table) != 2 or len(lens) != 1 or table[0] != lens[0] or tuple(starts) != (lens[0] + 1,):
        raise ShapeError("the batch's lists disagree: block_table [B, W], kv_len [B], q_start [B + 1]",
                         expected=("[B, W]", "[B]", "[B + 1]"), actual=(tuple(table), tuple(lens), tuple(starts)))
    if (table_strides[1] != 1 and table[1] > 1) or (len_strides[0] != 1 and lens[0] > 1) or start_strides[0] != 1:
        raise BackendError("the batch's lists must be contiguous along their last dimension")
    return (keys[1], _lib.longs(*key_strides[:3]), _lib.longs(*value_strides[:3]), keys[0], keys[2], table_strides[0],
            table[1], lens[0])


def _pool(key_pool: torch.Tensor, value_pool: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor,
          q_start: torch.Tensor, at: int, dtype: torch.dtype, D: int) -> tuple:
    """Check a page pool and a batch's lists on device ``at``; see :func:`_pool_layout`."""
    i32 = torch.int32
    if not (key_pool.dtype is dtype and value_pool.dtype is dtype and block_table.dtype is i32
            and kv_len.dtype is i32 and q_start.dtype is i32 and key_pool.get_device() == at
            and value_pool.get_device() == at and block_table.get_device() == at and kv_len.get_device() == at
            and q_start.get_device() == at):  # which one it is
        for name, t, want in (("key_pool", key_pool, dtype), ("value_pool", value_pool, dtype),
                              ("block_table", block_table, i32), ("kv_len", kv_len, i32), ("q_start", q_start, i32)):
            _same(name, t, at, want)
    return _pool_layout(key_pool.shape, key_pool.stride(), value_pool.shape, value_pool.stride(), block_table.shape,
                        block_table.stride(), kv_len.shape, kv_len.stride(), q_start.shape, q_start.stride(), D)


def paged_append(k: torch.Tensor, v: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor,
                 block_table: torch.Tensor, kv_len: torch.Tensor, q_start: torch.Tensor,
                 q: torch.Tensor | None = None, rotary=None, positions: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write a packed batch's new ``k``/``v`` ``[N, Hkv, D]`` to their pages,
    the keys rotated on the way when ``rotary`` (a
    :class:`~avqa_b200.rotary.RotaryEmbedding`) is given; ``q [N, H, D]`` is
    rotated in the same launch and returned (in ``q_out`` if given, which may
    be ``q`` but must not overlap it, ``k`` or ``v`` otherwise).

    ``key_pool``/``value_pool`` ``[pages, Hkv, page_size, D]`` (any page, head
    and slot strides); ``block_table [B, W]``, ``kv_len [B]`` (with the new
    tokens) and ``q_start [B + 1]`` are int32 on the device.  New token i of n
    is at position ``kv_len - n + i``, which ``positions`` (``[N]``, or
    ``[axes, N]``) replaces for the rotation only.  Tokens behind
    ``q_start[B]`` are left alone.  Serving only: no gradient is recorded."""
    lib = _lib.load()
    at, dt = _cuda_index(k, "key"), k.dtype
    N, Hkv, D = _packed_shape(k, "key")
    ks = _packed(k, "key", Hkv, N, D)
    _same("value", v, at, dt)
    vs = _packed(v, "value", Hkv, N, D)
    heads, kst, vst, pages, page_size, row, width, B = _pool(key_pool, value_pool, block_table, kv_len, q_start, at, dt,
                                                             D)
    if heads != Hkv:
        raise ShapeError("the pool's heads differ from the keys'", expected=heads, actual=Hkv)
    H, qp, qs, qop, qos = 0, None, None, None, None
    if q is not None:
        _same("query", q, at, dt)
        H = _packed_shape(q, "query")[1]
        qs = _packed(q, "query", H, N, D)
        if q_out is None:
            q_out = torch.empty_like(q)
            qos = _packed(q_out, "q_out", H, N, D)
        else:
            _same("q_out", q_out, at, dt)
            qos = _packed(q_out, "q_out", H, N, D)
            itself = q_out.data_ptr() == q.data_ptr() and q_out.stride() == q.stride()
            if (not itself and _overlap(q, q_out)) or _overlap(k, q_out) or _overlap(v, q_out):
                raise BackendError("q_out must be q or share no memory with q, k and v")
        qp, qop = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise BackendError("q_out needs q")
    R, inter, freq, axes, num_axes = 0, False, None, None, 1
    if rotary is not None:
        if rotary.head_dim != D:
            raise ShapeError("the rotary embedding's head_dim differs from the keys'", expected=rotary.head_dim,
                             actual=D)
        R, inter, num_axes = rotary.rotary_dim, rotary.interleaved, rotary.num_axes
        freq, axes = rotary.c_frequencies, rotary.c_axes
    elif positions is not None:
        raise BackendError("positions need a rotary embedding")
    pos, pos_bytes, pos_strides = _positions_operand(positions, num_axes, 1, N, at)
    _call("avq_paged_append", lib.avq_paged_append, at, _lib.dtype_code(dt), qp, qs, H, qop, qos, k.data_ptr(), ks,
          v.data_ptr(), vs, Hkv, D, key_pool.data_ptr(), kst, value_pool.data_ptr(), vst, pages, page_size,
          block_table.data_ptr(), row, width, kv_len.data_ptr(), q_start.data_ptr(), B, N, R, inter, freq, axes,
          num_axes, pos, pos_bytes, _lib.longs(pos_strides[0], pos_strides[2]))
    return q_out


@functools.lru_cache(maxsize=4096)
def _attention_workspace(code: int, B: int, N: int, H: int, Hkv: int, D: int, max_q_len: int) -> int:
    """Bytes of scratch, a multiple of 256."""
    return max(256, _lib.load().avq_paged_attention_workspace_size(code, B, N, H, Hkv, D, max_q_len))


@functools.lru_cache(maxsize=4096)
def _query_layout(q: tuple, strides: tuple) -> tuple:
    """Check a packed query; (N, H, D, its stride array, that of a contiguous output)."""
    if len(q) != 3:
        raise ShapeError("query must be packed [tokens, heads, head_dim]", expected="[N, H, D]", actual=tuple(q))
    N, H, D = q
    if strides[2] != 1 and D > 1:
        raise BackendError("query must have a contiguous last dimension", {"stride": tuple(strides)})
    return N, H, D, _lib.longs(strides[0], strides[1]), _lib.longs(H * D, D)


def paged_attention(q: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, block_table: torch.Tensor,
                    kv_len: torch.Tensor, q_start: torch.Tensor, causal: bool = True, window: int = 0,
                    scale: float | None = None, max_q_len: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a packed batch's new tokens ``q [N, H, D]`` over their
    sequences' pages (operands as in :func:`paged_append`, the new tokens' keys
    and values appended already): ``softmax(scale q k^T) v`` with ``scale``
    ``D ** -0.5`` by default.

    Each token sees its sequence's keys, with ``causal`` those at its position
    and before, with ``window > 0`` the last ``window`` of these.  ``H`` may be
    a multiple of the pool's heads (query head h reads key head
    ``h // (H // Hkv)``).  A token that sees no key gets zeros; rows behind
    ``q_start[B]`` are left as they are in ``out`` (without ``out`` they hold
    anything).  Pages whose keys no token sees, behind the window, are not looked up.  ``max_q_len``: the most new
    tokens of a sequence, if known; it only steers the choice of kernels.
    ``out`` must not overlap ``q``, also as another view of its memory.
    Probabilities are rounded to the dtype for the product with the values
    (bf16, fp16), all sums are fp32.  Serving only: no gradient is recorded."""
    lib = _lib.load()
    at, dt = _cuda_index(q, "query"), q.dtype
    N, H, D, qs, os = _query_layout(q.shape, q.stride())
    Hkv, kst, vst, pages, page_size, row, width, B = _pool(key_pool, value_pool, block_table, kv_len, q_start, at, dt,
                                                           D)
    if not (0 <= window < 1 << 31 and 0 <= max_q_len < 1 << 31):
        raise BackendError("window and max_q_len must be int32 and not negative",
                           {"window": window, "max_q_len": max_q_len})
    if Hkv == 0 or H == 0 or H % Hkv:
        raise ShapeError("query heads must be a multiple of the pool's heads", expected=f"n * {Hkv}", actual=H)
    if out is None:
        out = q.new_empty((N, H, D))
    else:
        _same("out", out, at, dt)
        os = _packed(out, "out", H, N, D)
        if _overlap(q, out):
            raise BackendError("out must not share memory with the query")
    if scale is None:
        scale = D ** -0.5 if D else 1.0
    code = _lib.dtype_code(dt)
    ws_bytes = _attention_workspace(code, B, N, H, Hkv, D, max_q_len)
    ws = kv_len.new_empty(ws_bytes // 4)
    _call("avq_paged_attention", lib.avq_paged_attention, at, code, q.data_ptr(), qs, H, key_pool.data_ptr(), kst,
          value_pool.data_ptr(), vst, Hkv, D, pages, page_size, block_table.data_ptr(), row, width, kv_len.data_ptr(),
          q_start.data_ptr(), B, N, causal, window, scale, max_q_len, out.data_ptr(), os, ws.data_ptr(), ws_bytes)
    return out


__all__ = ["ForwardDiagnostics", "PreparedCodebook", "QuantState", "append", "bcar_update", "codeword_presence",
           "dense_attention", "forward", "paged_append", "paged_attention", "pass_caps", "prepare_codebook", "quantize",
           "rotary"]
