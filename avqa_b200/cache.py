"""KV caches with the reference's interface (``src/avqa/cache.py:39-331``).

Both caches keep raw keys/values in head layout ``[B, H, S, D]`` and return
them from :meth:`lookup` in append order.  In addition each cache carries the
device quantization state of the AVQ modules that decode through it, so a
decode step quantizes only the appended token (bit-identical to the
reference's full re-quantization, see ``csrc/avq_decode.cu``).

Unlike the reference's ``PagedKVCache`` (whose pages are allocated as
``[1, H, 0, D]`` fp32 and therefore reject B > 1 and bf16 appends), pages
here are ``[B, H, page_size, D]`` device tensors in the cache dtype; decode
appends are written into the current page by the append kernel.
"""
from __future__ import annotations

from abc import ABC, abstractmethod
from collections.abc import Sequence
from contextlib import contextmanager
from dataclasses import dataclass

import torch

from avqa_b200.exceptions import BackendError, ConfigurationError, NotInitializedError, ShapeError


class KVCache(ABC):
    """Abstract KV cache."""

    def __init__(self) -> None:
        self.quant_states: dict = {}  # module key -> ops.QuantState

    @abstractmethod
    def append(self, key: torch.Tensor, value: torch.Tensor) -> None: ...

    @abstractmethod
    def lookup(self) -> tuple[torch.Tensor, torch.Tensor]: ...

    @abstractmethod
    def reset(self) -> None: ...

    @abstractmethod
    def state_dict(self) -> dict[str, torch.Tensor]: ...

    @abstractmethod
    def load_state_dict(self, state: dict[str, torch.Tensor]) -> None: ...

    @property
    @abstractmethod
    def size(self) -> int: ...


class InMemoryKVCache(KVCache):
    """Contiguous cache; keys/values concatenated along the sequence axis."""

    def __init__(self, num_heads: int = 1, head_dim_k: int = 64, head_dim_v: int = 64, max_size: int = 0,
                 device: str | torch.device = "cpu", dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        self.num_heads, self.head_dim_k, self.head_dim_v = num_heads, head_dim_k, head_dim_v
        self.max_size, self.device, self.dtype = max_size, device, dtype
        self.cache_key = torch.empty(0, num_heads, 0, head_dim_k, device=device, dtype=dtype)
        self.cache_value = torch.empty(0, num_heads, 0, head_dim_v, device=device, dtype=dtype)

    def append(self, key: torch.Tensor, value: torch.Tensor) -> None:
        if tuple(key.shape) != (*value.shape[:-1], self.head_dim_k):
            raise ShapeError(f"key/value shape mismatch: key={tuple(key.shape)}, value={tuple(value.shape)}",
                             expected=(*value.shape[:-1], self.head_dim_k), actual=tuple(key.shape))
        if self.cache_key.numel() == 0:
            self.cache_key = key.to(device=self.device, dtype=self.dtype)
            self.cache_value = value.to(device=self.device, dtype=self.dtype)
        else:
            self.cache_key = torch.cat([self.cache_key, key.to(self.cache_key.dtype)], dim=-2)
            self.cache_value = torch.cat([self.cache_value, value.to(self.cache_value.dtype)], dim=-2)
        if self.max_size > 0 and self.size > self.max_size:
            excess = self.size - self.max_size
            self.cache_key = self.cache_key[..., excess:, :].contiguous()
            self.cache_value = self.cache_value[..., excess:, :].contiguous()
            self.quant_states.clear()  # evicted keys leave the buckets: re-quantize next time

    def lookup(self) -> tuple[torch.Tensor, torch.Tensor]:
        if self.cache_key.numel() == 0 or self.cache_value.numel() == 0:
            return (torch.zeros(1, self.num_heads, 0, self.head_dim_k, dtype=self.dtype, device=self.device),
                    torch.zeros(1, self.num_heads, 0, self.head_dim_v, dtype=self.dtype, device=self.device))
        return self.cache_key, self.cache_value

    def reset(self) -> None:
        self.cache_key = torch.empty(0, self.num_heads, 0, self.head_dim_k, device=self.device, dtype=self.dtype)
        self.cache_value = torch.empty(0, self.num_heads, 0, self.head_dim_v, device=self.device, dtype=self.dtype)
        self.quant_states.clear()

    def state_dict(self) -> dict[str, torch.Tensor]:
        return {"schema_version": torch.tensor(1, dtype=torch.int32),
                "num_heads": torch.tensor(self.num_heads, dtype=torch.int32),
                "head_dim_k": torch.tensor(self.head_dim_k, dtype=torch.int32),
                "head_dim_v": torch.tensor(self.head_dim_v, dtype=torch.int32),
                "size": torch.tensor(self.size, dtype=torch.int32),
                "cache_key": self.cache_key.detach().clone(), "cache_value": self.cache_value.detach().clone()}

    def load_state_dict(self, state: dict[str, torch.Tensor]) -> None:
        for name in ("num_heads", "head_dim_k", "head_dim_v"):
            if name in state and int(state[name]) != getattr(self, name):
                raise ShapeError(f"{name} mismatch", expected=getattr(self, name), actual=int(state[name]))
        k, v = state.get("cache_key"), state.get("cache_value")
        self.quant_states.clear()
        if k is not None and v is not None and k.numel() > 0:
            self.cache_key = k.to(device=self.device, dtype=self.dtype)
            self.cache_value = v.to(device=self.device, dtype=self.dtype)
        else:
            self.reset()

    @property
    def size(self) -> int:
        return 0 if self.cache_key.numel() == 0 else int(self.cache_key.shape[-2])


class PagedKVCache(KVCache):
    """Fixed-size pages ``[B, H, page_size, D]`` on the cache device."""

    def __init__(self, page_size: int = 16, num_heads: int = 1, head_dim_k: int = 64, head_dim_v: int = 64,
                 max_pages: int = 0, device: str | torch.device = "cpu", dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        if page_size <= 0:
            raise ConfigurationError(f"page_size must be > 0, got {page_size}", {"page_size": page_size})
        self.page_size, self.num_heads = page_size, num_heads
        self.head_dim_k, self.head_dim_v = head_dim_k, head_dim_v
        self.max_pages, self.device, self.dtype = max_pages, device, dtype
        self.key_pages: list[torch.Tensor] = []
        self.value_pages: list[torch.Tensor] = []
        self.batch = 0
        self.fill = 0  # tokens in the last page

    # -- page management -------------------------------------------------------

    def allocate_page(self, batch: int) -> None:
        if self.max_pages > 0 and len(self.key_pages) >= self.max_pages:
            raise NotInitializedError(f"paged KV cache is full ({self.max_pages} pages)")
        shape_k = (batch, self.num_heads, self.page_size, self.head_dim_k)
        shape_v = (batch, self.num_heads, self.page_size, self.head_dim_v)
        self.key_pages.append(torch.zeros(shape_k, dtype=self.dtype, device=self.device))
        self.value_pages.append(torch.zeros(shape_v, dtype=self.dtype, device=self.device))
        self.batch = batch
        self.fill = 0

    def reserve(self, batch: int, n: int) -> list[tuple[int, int, int]]:
        """Claim ``n`` slots; returns ``(page, slot0, count)`` runs in order."""
        if self.key_pages and batch != self.batch:
            raise ShapeError("batch size changed inside a paged cache", expected=self.batch, actual=batch)
        runs = []
        while n > 0:
            if not self.key_pages or self.fill == self.page_size:
                self.allocate_page(batch)
            take = min(n, self.page_size - self.fill)
            runs.append((len(self.key_pages) - 1, self.fill, take))
            self.fill += take
            n -= take
        return runs

    def append(self, key: torch.Tensor, value: torch.Tensor) -> None:
        B, _, T, _ = key.shape
        cursor = 0
        for page, slot0, take in self.reserve(B, T):
            self.key_pages[page][:, :, slot0:slot0 + take] = key[:, :, cursor:cursor + take].to(self.dtype)
            self.value_pages[page][:, :, slot0:slot0 + take] = value[:, :, cursor:cursor + take].to(self.dtype)
            cursor += take

    def lookup(self) -> tuple[torch.Tensor, torch.Tensor]:
        if not self.key_pages:
            return (torch.zeros(1, self.num_heads, 0, self.head_dim_k, dtype=self.dtype, device=self.device),
                    torch.zeros(1, self.num_heads, 0, self.head_dim_v, dtype=self.dtype, device=self.device))
        ks = self.key_pages[:-1] + [self.key_pages[-1][:, :, :self.fill]]
        vs = self.value_pages[:-1] + [self.value_pages[-1][:, :, :self.fill]]
        return torch.cat(ks, dim=-2), torch.cat(vs, dim=-2)

    def reset(self) -> None:
        self.key_pages, self.value_pages = [], []
        self.fill = 0
        self.quant_states.clear()

    def state_dict(self) -> dict[str, torch.Tensor]:
        return {"schema_version": torch.tensor(1, dtype=torch.int32),
                "page_size": torch.tensor(self.page_size, dtype=torch.int32),
                "num_pages": torch.tensor(len(self.key_pages), dtype=torch.int32),
                "size": torch.tensor(self.size, dtype=torch.int32)}

    def load_state_dict(self, state: dict[str, torch.Tensor]) -> None:
        if "page_size" in state and int(state["page_size"]) != self.page_size:
            raise ShapeError("page_size mismatch", expected=self.page_size, actual=int(state["page_size"]))
        self.reset()

    @property
    def size(self) -> int:
        return 0 if not self.key_pages else (len(self.key_pages) - 1) * self.page_size + self.fill

    @property
    def num_pages(self) -> int:
        return len(self.key_pages)


@dataclass(frozen=True)
class PagedBatch:
    """One step's packed batch over a page pool: the lists that
    :func:`avqa_b200.ops.paged_append` and :func:`~avqa_b200.ops.paged_attention` take."""

    block_table: torch.Tensor  # [B, W] int32: the pages of each sequence
    kv_len: torch.Tensor  # [B] int32: tokens of each sequence, with the new ones
    q_start: torch.Tensor  # [B + 1] int32: where each sequence's new tokens begin
    max_q_len: int  # the most new tokens of a sequence
    tokens: int  # new tokens in all


class BlockKVCache(KVCache):
    """A pool of pages ``[num_pages, H, page_size, D]`` shared by sequences of
    different lengths, each with its own list of pages.

    Unlike :class:`PagedKVCache`, whose pages hold a whole batch of equal
    lengths, sequences here grow by different numbers of tokens
    (:meth:`reserve`), end one by one (:meth:`release` gives their pages back)
    and may have fewer key heads than the queries.  Appends and attention run
    on the pages in place (:meth:`attend`).  ``AVQAttention`` attends through
    it on its dense path (``execution.mode = "reference"`` or refinement off).

    ``rotary``: a :class:`~avqa_b200.rotary.RotaryEmbedding` that rotates keys
    as they are appended and queries as they attend.
    """

    def __init__(self, num_pages: int, page_size: int = 16, num_heads: int = 1, head_dim: int = 64, rotary=None,
                 device: str | torch.device = "cuda", dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        for name, n in (("num_pages", num_pages), ("page_size", page_size), ("num_heads", num_heads),
                        ("head_dim", head_dim)):
            if n <= 0:
                raise ConfigurationError(f"{name} must be > 0, got {n}", {name: n})
        if rotary is not None and rotary.head_dim != head_dim:
            raise ConfigurationError("the rotary embedding's head_dim differs from the cache's",
                                     {"head_dim": head_dim, "rotary": rotary.head_dim})
        self.num_pages, self.page_size, self.num_heads, self.head_dim = num_pages, page_size, num_heads, head_dim
        self.rotary, self.device, self.dtype = rotary, torch.device(device), dtype
        self.key_pool = torch.zeros(num_pages, num_heads, page_size, head_dim, dtype=dtype, device=device)
        self.value_pool = torch.zeros_like(self.key_pool)
        self.lengths: list[int] = []  # tokens of each sequence
        self.pages: list[list[int]] = []  # its pages, in order
        self.free_pages = list(range(num_pages - 1, -1, -1))
        self._table = torch.zeros(0, 1, dtype=torch.int32)  # the pages as the steps' table rows, on the host

    # -- sequences ---------------------------------------------------------------

    def reserve(self, new: Sequence[int]) -> PagedBatch:
        """Make room for ``new[b]`` more tokens of each sequence b (a longer
        list than before starts new sequences) and return the step's lists.
        The cache is unchanged when the pool cannot hold them.  The lists are a
        step's own: a CUDA graph captures the operators over lists made before."""
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise BackendError("a step's pages cannot be reserved while a CUDA graph is captured")
        new = [int(n) for n in new]
        if len(new) < len(self.lengths) or any(n < 0 for n in new):
            raise ShapeError("every sequence needs a number of new tokens, 0 or more", expected=len(self.lengths),
                             actual=new)
        grown = [(self.lengths[b] if b < len(self.lengths) else 0) + n for b, n in enumerate(new)]
        need = [-(-length // self.page_size) for length in grown]
        more = [n - (len(self.pages[b]) if b < len(self.pages) else 0) for b, n in enumerate(need)]
        if sum(more) > len(self.free_pages):
            raise NotInitializedError(f"paged KV cache is full ({self.num_pages} pages)",
                                      {"needed": sum(more), "free": len(self.free_pages)})
        B, W = len(new), max([1, *need])
        rows, width = self._table.shape
        if rows < B or width < W:  # only what is short grows; no sequence can hold more than the pool
            table = torch.zeros(rows if rows >= B else max(B, 2 * rows),
                                width if width >= W else min(max(W, 2 * width), self.num_pages), dtype=torch.int32)
            table[:rows, :width] = self._table
            self._table = table
        free, taken = len(self.free_pages), {}
        for b, n in enumerate(more):
            if n > 0:
                taken[b] = self.free_pages[free - n:free][::-1]
                free -= n
                self._table[b, need[b] - n:need[b]] = torch.tensor(taken[b], dtype=torch.int32)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        # one copy carries all lists; its host memory is the step's own, as the copy may still run when the next begins
        flat = torch.empty(B * W + 2 * B + 1, dtype=torch.int32, pin_memory=self.device.type == "cuda")
        flat[:B * W].view(B, W).copy_(self._table[:B, :W])
        flat[B * W:] = torch.tensor(grown + starts, dtype=torch.int32)
        flat = flat.to(self.device, non_blocking=True)
        # nothing can fail any more
        del self.free_pages[free:]
        self.pages.extend([] for _ in range(B - len(self.pages)))
        for b, pages in taken.items():
            self.pages[b].extend(pages)
        self.lengths = grown
        self.quant_states.clear()  # whatever covered the pages does no longer
        return PagedBatch(flat[:B * W].view(B, W), flat[B * W:B * W + B], flat[B * W + B:], max([0, *new]),
                          starts[-1])

    def release(self, sequence: int) -> None:
        """End a sequence: its pages return to the pool, its place stays, empty."""
        if not 0 <= sequence < len(self.lengths):
            raise ShapeError("no such sequence", expected=f"[0, {len(self.lengths)})", actual=sequence)
        self.free_pages.extend(reversed(self.pages[sequence]))
        self.pages[sequence] = []
        self.lengths[sequence] = 0
        self.quant_states.clear()

    # -- packed steps --------------------------------------------------------------

    def attend(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, new: Sequence[int],
               positions: torch.Tensor | None = None, causal: bool = True, window: int = 0,
               scale: float | None = None, rotary=None) -> torch.Tensor:
        """Append the packed new tokens ``key``/``value`` ``[N, H, D]`` (``new[b]``
        of sequence b) and attend with ``query [N, Hq, D]`` over each
        sequence's pages; returns ``[N, Hq, D]``.  See
        :func:`avqa_b200.ops.paged_append` and
        :func:`~avqa_b200.ops.paged_attention`; ``rotary`` stands in for the
        cache's own."""
        from avqa_b200 import ops
        if rotary is not None and self.rotary is not None:
            raise ConfigurationError("the cache rotates by its own embedding already")
        if sum(new) != key.shape[0]:
            raise ShapeError("the new tokens do not add up to the packed ones", expected=sum(new),
                             actual=key.shape[0])
        self._check(key, value)
        if query.dim() != 3 or query.shape[0] != key.shape[0] or query.shape[2] != self.head_dim:
            raise ShapeError("the queries must be the new tokens' own", expected=(key.shape[0], "Hq", self.head_dim),
                             actual=tuple(query.shape))
        rotary = self.rotary if rotary is None else rotary
        with self._step(new) as batch:
            lists = (self.key_pool, self.value_pool, batch.block_table, batch.kv_len, batch.q_start)
            rotated = ops.paged_append(key, value, *lists, q=query if rotary is not None else None, rotary=rotary,
                                       positions=positions)
            return ops.paged_attention(query if rotated is None else rotated, *lists, causal=causal, window=window,
                                       scale=scale, max_q_len=batch.max_q_len)

    @contextmanager
    def _step(self, new: Sequence[int]):
        """:meth:`reserve`, taken back when the step is refused."""
        lengths, counts = list(self.lengths), [len(p) for p in self.pages]
        try:
            yield self.reserve(new)
        except Exception:
            for b in range(len(self.pages) - 1, -1, -1):
                keep = counts[b] if b < len(counts) else 0
                self.free_pages.extend(reversed(self.pages[b][keep:]))
                del self.pages[b][keep:]
            del self.pages[len(counts):]
            self.lengths = lengths
            raise

    def _check(self, key: torch.Tensor, value: torch.Tensor) -> None:
        want = (self.num_heads, self.head_dim)
        if tuple(key.shape[-2:]) != want or key.shape != value.shape:
            raise ShapeError(f"key/value shape mismatch: key={tuple(key.shape)}, value={tuple(value.shape)}",
                             expected=want, actual=tuple(key.shape[-2:]))

    # -- the KVCache interface -----------------------------------------------------------

    def append(self, key: torch.Tensor, value: torch.Tensor) -> None:
        """Append ``[B, H, T, D]``, T tokens to every sequence."""
        from avqa_b200 import ops
        if key.dim() != 4 or key.shape != value.shape or (key.shape[1], key.shape[3]) != (self.num_heads, self.head_dim):
            raise ShapeError(f"key/value shape mismatch: key={tuple(key.shape)}, value={tuple(value.shape)}",
                             expected=("B", self.num_heads, "T", self.head_dim), actual=tuple(key.shape))
        B, H, T, D = key.shape
        k, v = (x.to(device=self.device, dtype=self.dtype).transpose(1, 2).reshape(B * T, H, D) for x in (key, value))
        with self._step([T] * B) as batch:
            ops.paged_append(k, v, self.key_pool, self.value_pool, batch.block_table, batch.kv_len, batch.q_start,
                             rotary=self.rotary)

    def lookup(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys (as stored: rotated) and values ``[B, H, S, D]``, when every sequence has S tokens."""
        S = self.size
        if any(n != S for n in self.lengths):
            raise ShapeError("sequences of different lengths have no common tensor", expected=S, actual=self.lengths)
        if S == 0:
            empty = torch.zeros(max(1, len(self.lengths)), self.num_heads, 0, self.head_dim, dtype=self.dtype,
                                device=self.device)
            return empty, empty.clone()
        pages = torch.tensor(self.pages, device=self.device)
        return tuple(pool[pages].transpose(1, 2).reshape(len(self.lengths), self.num_heads, -1, self.head_dim)[:, :, :S]
                     for pool in (self.key_pool, self.value_pool))

    def reset(self) -> None:
        self.lengths, self.pages = [], []
        self.free_pages = list(range(self.num_pages - 1, -1, -1))
        self.quant_states.clear()

    def state_dict(self) -> dict[str, torch.Tensor]:
        used = [p for pages in self.pages for p in pages]
        return {"schema_version": torch.tensor(1, dtype=torch.int32),
                "page_size": torch.tensor(self.page_size, dtype=torch.int32),
                "num_heads": torch.tensor(self.num_heads, dtype=torch.int32),
                "head_dim": torch.tensor(self.head_dim, dtype=torch.int32),
                "lengths": torch.tensor(self.lengths, dtype=torch.int64),
                "key_pages": self.key_pool[used].clone(), "value_pages": self.value_pool[used].clone()}

    def load_state_dict(self, state: dict[str, torch.Tensor]) -> None:
        """Hold a saved cache's sequences instead; one that does not fit is refused and changes nothing."""
        for name in ("page_size", "num_heads", "head_dim"):
            if name in state and int(state[name]) != getattr(self, name):
                raise ShapeError(f"{name} mismatch", expected=getattr(self, name), actual=int(state[name]))
        lengths = [int(n) for n in state["lengths"].tolist()]
        if any(n < 0 for n in lengths):
            raise ShapeError("a saved length is negative", expected="0 or more", actual=lengths)
        need = sum(-(-n // self.page_size) for n in lengths)
        if need > self.num_pages:
            raise NotInitializedError(f"the saved sequences do not fit the paged KV cache ({self.num_pages} pages)",
                                      {"needed": need, "pages": self.num_pages})
        want = (need, *self.key_pool.shape[1:])
        saved = []
        for name in ("key_pages", "value_pages"):
            if tuple(state[name].shape) != want:
                raise ShapeError(f"{name} do not fit the saved lengths", expected=want, actual=tuple(state[name].shape))
            saved.append(state[name].to(device=self.device, dtype=self.dtype))
        kept = self.lengths, self.pages, self.free_pages
        self.lengths, self.pages, self.free_pages = [], [], list(range(self.num_pages - 1, -1, -1))
        try:
            self.reserve(lengths)
        except Exception:  # the cache keeps what it held
            self.lengths, self.pages, self.free_pages = kept
            for b, pages in enumerate(self.pages):
                self._table[b, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            raise
        used = [p for pages in self.pages for p in pages]
        self.key_pool[used], self.value_pool[used] = saved

    @property
    def size(self) -> int:
        """Tokens of the longest sequence."""
        return max(self.lengths, default=0)


__all__ = ["BlockKVCache", "InMemoryKVCache", "KVCache", "PagedBatch", "PagedKVCache"]
