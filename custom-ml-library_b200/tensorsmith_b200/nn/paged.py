"""``PagedKVCache``: the 4-bit KV cache of a whole model, its rows made of shared pages.

tensorsmith's cache owns a preallocated block a batch row (src/tensorsmith/nn/cache.py:12-142), int8 at the
smallest.  Here every layer has a pool of pages in 4 bits, and one page table serves all layers: rows take
pages as they grow, forked rows (parallel samples, beams) share them until one writes, and freed pages return
to the pool.  ``layers`` are the per-layer views that ``TransformerLM`` takes in the place of ``KVCache``
objects; like those they are for inference only.  A step appends the same number of tokens to every row, an
emptied one included; ``engine.kv_pages_reserve`` and ``kv_append_int4`` take rows that step by numbers of their own.

The tables, lengths, reference counts and free-page counters live on the device and are changed by the
engine's page operations without a host round trip.  The host keeps the row lengths, which decide when a
page is due, and a lower bound of the free pages; only when that bound is too small for an append does it
read the true count back, and raises when the pages do not suffice.
"""

from __future__ import annotations

import numpy as np
import torch

from .. import engine
from ..tensor import Tensor, as_device, is_grad_enabled
from .cache import _torch_dtype

_COMPUTE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


class PagedKVCache:
    """A pool of 4-bit pages for ``num_layers`` layers and the rows that hold them."""

    PAGE_SIZE = 64  # tokens of a page; 16 and 32 share shorter prefixes at some cost in speed

    def __init__(self, batch_size: int, num_layers: int, num_heads: int, head_dim: int, max_seq_len: int, *,
                 num_pages: int | None = None, page_size: int = PAGE_SIZE, device="cuda", dtype="float32"):
        if min(batch_size, num_layers, num_heads, head_dim, max_seq_len) <= 0:
            raise ValueError("cache dimensions and capacity must be positive")
        self.num_heads, self.head_dim, self.value_dim = num_heads, head_dim, head_dim
        self.max_seq_len, self.page_size = max_seq_len, page_size
        engine.int4_block_bytes(head_dim, page_size)  # raises on a size the pages do not take
        self.device = as_device(device)
        if self.device.type != "cuda":
            raise ValueError("the B200 KV cache lives on a cuda device")
        self.dtype = _torch_dtype(dtype)
        if self.dtype not in _COMPUTE_DTYPES:
            raise TypeError("a 4-bit cache computes in float32, float16 or bfloat16")
        slots = -(-max_seq_len // page_size)
        self.num_pages = batch_size * slots if num_pages is None else int(num_pages)
        if self.num_pages <= 0:
            raise ValueError("a cache needs at least one page")
        dev = torch.device("cuda", self.device.index)
        self._pool = engine.int4_pool(self.num_pages, num_heads, head_dim, page_size=page_size, layers=num_layers,
                                      device=dev)
        self._refs, self._counters = engine.kv_pages_state(self.num_pages, dev)
        self._table = torch.full((batch_size, slots), -1, dtype=torch.int32, device=dev)
        self._lens = torch.zeros(batch_size, dtype=torch.int32, device=dev)
        self._before = self._lens  # the lengths before the last append
        self._host_lens = np.zeros(batch_size, dtype=np.int64)
        self._host_before = self._host_lens  # host copy of _before
        self._reserved = np.zeros(batch_size, dtype=np.int64)  # tokens the rows' own pages can hold
        self._free = self.num_pages  # a lower bound
        self.layers = [PagedLayer(self, i) for i in range(num_layers)]

    # -- rows ----------------------------------------------------------------
    @property
    def batch_size(self) -> int:
        return len(self._host_lens)

    @property
    def length(self) -> int:
        """The longest row's tokens."""
        return int(self._host_lens.max())

    @property
    def lengths(self) -> np.ndarray:
        """Tokens of every row (host copy)."""
        return self._host_lens.copy()

    @property
    def seq_lens(self) -> torch.Tensor:
        """Device int32 [B] lengths."""
        return self._lens

    @property
    def positions(self) -> torch.Tensor:
        """Device int32 [B] position of the first token of the last append."""
        return self._before

    @property
    def page_table(self) -> torch.Tensor:
        """Device int32 [B, slots]: the page of each ``page_size`` tokens of a row, -1 for none."""
        return self._table

    def free_pages(self) -> int:
        """Pages that no row holds (reads the device's count)."""
        self._free = int(self._counters[0])
        return self._free

    @property
    def memory_bytes(self) -> int:
        return self._pool.numel()

    def _rows(self, rows) -> np.ndarray:
        raw = rows._data if isinstance(rows, Tensor) else rows
        host = raw.detach().cpu().numpy() if isinstance(raw, torch.Tensor) else np.asarray(raw)
        if host.ndim != 1 or host.size == 0 or host.dtype.kind not in "iu":
            raise ValueError("rows must be a nonempty vector of integers")
        return host.astype(np.int64)

    def fork(self, rows) -> None:
        """Row i becomes a copy of the present row ``rows[i]`` (any number of rows; -1: an empty one).  The copies
        share their pages; whoever first writes to a shared, partly filled page gets its own."""
        index = self._rows(rows)
        if (index < -1).any() or (index >= self.batch_size).any():
            raise ValueError("row out of range")
        self._settled()
        dev_index = torch.as_tensor(index.astype(np.int32), device=self._table.device)
        self._table, self._lens = engine.kv_pages_fork(self._table, self._lens, dev_index, self._refs, self._counters,
                                                       page_size=self.page_size)
        self._before = self._lens
        self._host_lens = self._host_before = np.where(index < 0, 0, self._host_lens[index])
        # full pages stay; the partly filled one may be shared now, reserved ones behind it went back
        self._reserved = self._host_lens // self.page_size * self.page_size
        for layer in self.layers:
            layer.length = self.length

    def reorder(self, indices) -> None:
        """Reorder or duplicate rows for fixed-width beam search."""
        index = self._rows(indices)
        if index.shape != (self.batch_size,):
            raise ValueError("beam indices must be one integer per cache batch row")
        if (index < 0).any() or (index >= self.batch_size).any():
            raise ValueError("beam index out of range")
        self.fork(index)

    def free(self, rows) -> None:
        """Empty the given rows; pages that nobody else holds return to the pool."""
        index = np.arange(self.batch_size)
        gone = self._rows(rows)
        if (gone < 0).any() or (gone >= self.batch_size).any():
            raise ValueError("row out of range")
        index[gone] = -1
        self.fork(index)

    def compact(self) -> None:
        """Move the live pages to the start of the pool."""
        self._settled()
        engine.kv_pages_compact(self._pool, self._table, self._refs, self._counters)

    def reset(self) -> None:
        """Empty every row."""
        for layer in self.layers:
            layer.length = self.length
        self.fork(np.full(self.batch_size, -1))

    def truncate(self, length) -> None:
        """Forget the tokens past ``length``, one number for all rows or one a row.  A step that only some layers
        have appended is forgotten in every row."""
        if np.ndim(length):
            host = self._rows(length)
            if host.shape != self._host_lens.shape or (host < 0).any() or (host > self._host_lens).any():
                raise ValueError("truncate lengths must be between zero and every row's length")
        elif not 0 <= length <= self.length:
            raise ValueError("truncate length must be between zero and the current length")
        else:
            host = length
        whole = self._host_before if self._unfinished() else self._host_lens
        self._host_lens = self._host_before = np.minimum(whole, host)
        dev = self._table.device
        lens = torch.as_tensor(self._host_lens.astype(np.int32), device=dev)
        # a fork onto themselves lets the rows drop the pages past their tokens, which others may share
        rows = torch.arange(self.batch_size, dtype=torch.int32, device=dev)
        self._table, self._lens = engine.kv_pages_fork(self._table, lens, rows, self._refs, self._counters,
                                                       page_size=self.page_size)
        self._before = self._lens
        self._reserved = self._host_lens // self.page_size * self.page_size
        for layer in self.layers:
            layer.length = self.length

    def _unfinished(self) -> bool:
        """Whether some layer has not yet appended the tokens of the last step."""
        return any(layer.length != self.length for layer in self.layers)

    def _settled(self) -> None:
        if self._unfinished():
            raise RuntimeError("every layer must append a step's tokens before the rows change")

    # -- appends ---------------------------------------------------------------
    def _begin(self, steps: int) -> None:
        """Pages for ``steps`` more tokens of every row, and the lengths with them."""
        stop = self._host_lens + steps
        if (stop > self._reserved).any():
            size = self.page_size
            # at most: the missing pages of every row, and a copy of its partly filled one
            held = -(-np.maximum(self._reserved, self._host_lens) // size)
            copies = (self._host_lens % size != 0) & (self._reserved < self._host_lens)
            need = int((np.maximum(-(-stop // size) - held, 0) + copies).sum())
            if need > self._free and need > self.free_pages() and not self._fits(steps):
                raise ValueError(f"cache has {self._free} free pages, {need} are needed")
            engine.kv_pages_reserve(self._pool, self._table, self._lens, steps, self._refs, self._counters,
                                    page_size=size)
            self._free -= need
            self._reserved = -(-stop // size) * size
        self._before, self._lens = self._lens, self._lens + steps
        self._host_before, self._host_lens = self._host_lens, stop

    def _fits(self, steps: int) -> bool:
        """The exact need against the free pages, read from the device: copies of pages that several writers share
        leave one of them the page itself."""
        size, table, refs = self.page_size, self._table.cpu().numpy(), self._refs.cpu().numpy()
        need, writers = 0, {}
        for r, n in enumerate(self._host_lens):
            need += int((table[r, -(-n // size): -(-(n + steps) // size)] < 0).sum())
            if n % size:
                writers.setdefault(int(table[r, n // size]), []).append(r)
        need += sum(len(rows) - (int(refs[page]) == len(rows)) for page, rows in writers.items())
        return need <= self._free

    def __repr__(self):
        return (f"PagedKVCache(rows={self.batch_size}, length={self.length}, capacity={self.max_seq_len}, "
                f"pages={self.num_pages} x {self.page_size}, layers={len(self.layers)}, device='{self.device}')")


class PagedLayer:
    """One layer of a ``PagedKVCache``, with the interface of ``KVCache`` that the attention module uses."""

    quantized = True

    def __init__(self, cache: PagedKVCache, index: int):
        self.cache, self.index, self.length = cache, index, 0

    batch_size = property(lambda self: self.cache.batch_size)
    num_heads = property(lambda self: self.cache.num_heads)
    head_dim = property(lambda self: self.cache.head_dim)
    value_dim = property(lambda self: self.cache.value_dim)
    max_seq_len = property(lambda self: self.cache.max_seq_len)
    device = property(lambda self: self.cache.device)
    dtype = property(lambda self: self.cache.dtype)

    @property
    def pool(self) -> torch.Tensor:
        return self.cache._pool[self.index]

    def append(self, key: Tensor, value: Tensor) -> None:
        """Quantise a [B, H, steps, D] chunk behind every row's tokens.

        The first layer to append a step reserves its pages; the others write the same tokens."""
        self._append(key, value, None)

    def append_rotary(self, key: Tensor, value: Tensor, *, base: float = 10000.0, rotary_dim: int | None = None) -> None:
        """``append`` with the keys rotated at their cache positions first (nn/transformer.py:139-142)."""
        dim = self.head_dim if rotary_dim is None else rotary_dim
        if dim <= 0 or dim % 2 or dim > self.head_dim or base <= 0 or not np.isfinite(base):
            raise ValueError("RoPE requires a positive even rotary dimension and valid positions/base")
        self._append(key, value, dict(base=base, rotary_dim=dim))

    def _append(self, key: Tensor, value: Tensor, rotary) -> None:
        cache = self.cache
        if key.device != cache.device or value.device != cache.device:
            raise ValueError("cache and key/value tensors must be on the same device")
        if is_grad_enabled() and (key.requires_grad or value.requires_grad):
            raise RuntimeError("KVCache is inference-only; use no_grad() for differentiable inputs")
        if key.ndim != 4 or key.shape[:2] != (cache.batch_size, cache.num_heads) or key.shape[-1] != cache.head_dim:
            raise ValueError("key shape does not match cache configuration")
        if value.shape != key.shape:
            raise ValueError("value shape does not match cache configuration")
        if rotary is not None:
            engine.dtype_code(key.dtype)  # raises on a type that cannot be rotated, before the step begins
        steps = key.shape[2]
        if self.length == cache.length:
            if steps == 0 or cache.length + steps > cache.max_seq_len:
                raise ValueError(f"cache capacity {cache.max_seq_len} exceeded or empty append")
            cache._begin(steps)
        elif self.length + steps != cache.length:
            raise ValueError("every layer must append the same tokens")
        raw = key._data
        if rotary is not None:
            raw = engine.rope(raw, positions=cache._before, **rotary)
        # rounded to the cache's compute type first, as tensorsmith's int8 cache does (nn/cache.py:68)
        raw, val = (t if t.dtype == cache.dtype else t.to(cache.dtype) for t in (raw, value._data))
        engine.kv_append_int4(raw, val, self.pool, cache._table, page_size=cache.page_size, positions=cache._before)
        self.length += steps

    def attend(self, query: Tensor, *, scale: float | None = None, is_causal: bool = True) -> Tensor:
        """Attention of ``query`` [B, Hq, Tq, D], the newest Tq tokens of every row, over the row's pages."""
        cache = self.cache
        if query.ndim != 4 or query.shape[0] != cache.batch_size or query.shape[-1] != cache.head_dim:
            raise ValueError("query shape does not match cache configuration")
        if query.shape[1] % cache.num_heads or query.device != cache.device:
            raise ValueError("query heads must be a multiple of the cache heads, on the cache device")
        if query.dtype != cache.dtype:
            raise TypeError("query dtype must be the cache compute dtype")
        if is_grad_enabled() and query.requires_grad:
            raise RuntimeError("KVCache is inference-only; use no_grad() for differentiable inputs")
        if self.length != cache.length or self.length == 0 or query.shape[2] > self.length:
            raise ValueError("the cache must already hold the query tokens")
        out, _ = engine.attention_int4(query._data, self.pool, cache._table, cache._lens, page_size=cache.page_size,
                                       max_len=self.length, is_causal=is_causal, scale=scale)
        return Tensor(out, device=cache.device)

    def get(self) -> tuple[Tensor, Tensor]:
        """Dequantised keys and values [B, H, length, D]; zero past a row's tokens."""
        cache = self.cache
        keys, values = engine.kv_gather_int4(self.pool, cache._table, self.length, page_size=cache.page_size,
                                             dtype=cache.dtype, kv_lens=cache._lens)
        return Tensor(keys, device=cache.device), Tensor(values, device=cache.device)

    def truncate(self, length) -> None:
        """``PagedKVCache.truncate``: in every layer, as they share the rows."""
        if np.ndim(length) or length != self.cache.length:
            self.cache.truncate(length)

    def __len__(self):
        return self.length
