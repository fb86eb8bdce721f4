"""The paged 4-bit KV cache in NumPy: storage format, attention over it, page operations.

Written from the definitions in include/ts_attn.h; loops are fine here.
"""

from __future__ import annotations

import numpy as np

SCALE_MIN, SCALE_MAX = 2.0**-20, 9216.0


def int4_scale(amax: np.ndarray) -> np.ndarray:
    """max|x| / 7 rounded up to 5 significant bits, within [2^-20, 9216]."""
    s = np.minimum(amax.astype(np.float32) / np.float32(7), np.float32(SCALE_MAX))
    mant, exp = np.frexp(s.astype(np.float64))  # s = mant * 2^exp, mant in [0.5, 1)
    up = np.ldexp(np.ceil(mant * 32) / 32, exp)
    return np.clip(up, SCALE_MIN, SCALE_MAX)


def quantize_int4(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """``x`` [..., D] -> (n int8 [..., D] in [-7, 7], scales float64 [..., D / 32])."""
    g = x.astype(np.float32).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    scale = int4_scale(np.nanmax(np.abs(np.where(np.isnan(g), 0, g)), axis=-1))
    with np.errstate(invalid="ignore"):
        n = np.rint(np.clip(g / scale[..., None].astype(np.float32), -7, 7))
    n = np.where(np.isnan(g), 0, n).astype(np.int8)
    return n.reshape(x.shape), scale


def dequantize_int4(n: np.ndarray, scale: np.ndarray) -> np.ndarray:
    return (n.astype(np.float64).reshape(scale.shape + (32,)) * scale[..., None]).reshape(n.shape)


def pack_block(k: np.ndarray, ks: np.ndarray, v: np.ndarray, vs: np.ndarray) -> np.ndarray:
    """One page's block (uint8) of one head from n [page, D] and scales [page, D / 32] of K and V."""
    parts = []
    for n, s in ((k, ks), (v, vs)):
        page, dim = n.shape
        groups = dim // 32
        words = np.zeros((page, dim // 8), np.uint32)
        for c in range(dim):
            g, t, e = c // 32, c % 32 // 8, c % 8
            words[:, t * groups + g] |= (n[:, c].astype(np.int64) + 8).astype(np.uint32) << np.uint32(4 * e)
        parts += [words.view(np.uint8).ravel(), s.astype(np.float16).view(np.uint8).ravel()]
    return np.concatenate(parts)


def unpack_block(block: np.ndarray, page: int, dim: int) -> tuple[np.ndarray, np.ndarray]:
    """(keys, values) float64 [page, D] that a block stands for."""
    out = []
    groups, half = dim // 32, block.size // 2
    for part in (block[:half], block[half:]):
        words = np.ascontiguousarray(part[: page * dim // 2]).view(np.uint32).reshape(page, dim // 8)
        scale = np.ascontiguousarray(part[page * dim // 2:]).view(np.float16).reshape(page, groups).astype(np.float64)
        x = np.empty((page, dim))
        for c in range(dim):
            g, t, e = c // 32, c % 32 // 8, c % 8
            x[:, c] = ((words[:, t * groups + g] >> np.uint32(4 * e)) & 15).astype(np.float64) - 8
            x[:, c] *= scale[:, g]
        out.append(x)
    return out[0], out[1]


def attention_int4(q, keys, values, lens, *, is_causal=True, scale=None):
    """fp64 attention of ``q`` [B, Hq, Tq, D] over rows' own keys / values (lists of [Hkv, len_b, D]).

    Returns (out, lse, spread): ``spread`` = sum_j p_ij |v_jc|, what a rounding of p can move."""
    b, hq, tq, d = q.shape
    scale = d**-0.5 if scale is None else scale
    out, lse, spread = np.zeros(q.shape), np.full((b, hq, tq), -np.inf), np.zeros(q.shape)
    for r in range(b):
        n = int(lens[r])
        for h in range(hq):
            hk = h // (hq // keys[r].shape[0])
            for i in range(tq):
                seen = min(n, n - tq + i + 1) if is_causal else n
                if seen <= 0:
                    continue
                s = keys[r][hk, :seen] @ q[r, h, i].astype(np.float64) * scale
                m = s.max()
                p = np.exp(s - m)
                lse[r, h, i] = m + np.log(p.sum())
                p /= p.sum()
                out[r, h, i] = p @ values[r][hk, :seen]
                spread[r, h, i] = p @ np.abs(values[r][hk, :seen])
    return out, lse, spread


class PagesOracle:
    """Tables, counts and pages of a paged cache, one step at a time in Python integers."""

    def __init__(self, table, lens, refs, pool, page_size):
        self.table, self.lens, self.refs = np.array(table), np.array(lens), np.array(refs)
        self.pool, self.page_size = np.array(pool), page_size  # [layers, pages, ...]

    def fork(self, index):
        rows = []
        for src in index:
            row = np.full(self.table.shape[1], -1, self.table.dtype)
            if src >= 0:
                used = -(-int(self.lens[src]) // self.page_size)
                row[:used] = self.table[src, :used]
            rows.append(row)
        for page in np.concatenate(rows):
            if page >= 0:
                self.refs[page] += 1
        for page in self.table.ravel():
            if page >= 0:
                self.refs[page] -= 1
        self.lens = np.array([self.lens[s] if s >= 0 else 0 for s in index], self.lens.dtype)
        self.table = np.stack(rows)

    def reserve(self, steps):
        """True when the pages sufficed; steps: one number a row."""
        size = self.page_size
        writes = {}  # shared partial page -> the rows that write to it
        for r, n in enumerate(steps):
            if n > 0 and self.lens[r] % size:
                writes.setdefault(int(self.table[r, self.lens[r] // size]), []).append(r)
        wanted = []  # (row, slot, page to copy)
        for r, n in enumerate(steps):
            first = int(self.lens[r]) // size
            if n > 0 and self.lens[r] % size:
                page = int(self.table[r, first])
                others = self.refs[page] - len(writes[page])
                if others > 0 or r != writes[page][-1]:
                    wanted.append((r, first, page))
            for slot in range(-(-int(self.lens[r]) // size), -(-(int(self.lens[r]) + int(n)) // size)):
                if slot >= self.table.shape[1]:
                    return False
                if self.table[r, slot] < 0:
                    wanted.append((r, slot, -1))
        free = np.nonzero(self.refs == 0)[0]
        if len(wanted) > len(free):
            return False
        copies = []
        for (r, slot, page), own in zip(wanted, free):
            if page >= 0:
                copies.append((page, own))
                self.refs[page] -= 1
            self.table[r, slot] = own
            self.refs[own] = 1
        for page, own in copies:
            self.pool[:, own] = self.pool[:, page]
        return True

    def compact(self):
        live = int((self.refs > 0).sum())
        movers = [p for p in range(len(self.refs)) if self.refs[p] > 0 and p >= live][::-1]
        holes = [p for p in range(live) if self.refs[p] == 0]
        for a, b in zip(movers, holes):
            self.pool[:, b] = self.pool[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.table[self.table == a] = b
