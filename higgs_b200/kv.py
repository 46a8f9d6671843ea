"""Python handles over the native KV page pool and radix prefix cache
(higgs_block_pool_* / higgs_prefix_cache_* in include/higgs_cuda.h)."""
from __future__ import annotations

import ctypes

import numpy as np

from . import ffi

PAGE = 16


def _i32p(a: np.ndarray):
    return a.ctypes.data_as(ctypes.c_void_p)


class BlockPool:
    """Refcounted KV page ids [0, num_pages)."""

    def __init__(self, num_pages: int):
        h = ffi.P()
        ffi.call("higgs_block_pool_create", num_pages, ctypes.byref(h))
        self.handle = h.value
        self.num_pages = num_pages

    def __del__(self):
        try:
            ffi.load().higgs_block_pool_destroy(self.handle)
        except Exception:
            pass

    @property
    def num_free(self) -> int:
        return int(ffi.load().higgs_block_pool_num_free(self.handle))

    def alloc(self, n: int) -> np.ndarray:
        out = np.empty(n, np.int32)
        ffi.call("higgs_block_pool_alloc", self.handle, n, _i32p(out))
        return out

    def retain(self, pages) -> None:
        p = np.ascontiguousarray(pages, dtype=np.int32)
        ffi.call("higgs_block_pool_retain", self.handle, _i32p(p), p.size)

    def release(self, pages) -> None:
        p = np.ascontiguousarray(pages, dtype=np.int32)
        ffi.call("higgs_block_pool_release", self.handle, _i32p(p), p.size)

    def refcount(self, page: int) -> int:
        return int(ffi.load().higgs_block_pool_refcount(self.handle, page))

    def fork(self, pages, length: int) -> tuple[np.ndarray, tuple[int, int] | None]:
        """(pages of a second owner of the sequence, the (source, destination) pair of pages to copy
        or None): whole pages are shared, a partly filled last one is replaced by a fresh one."""
        ffi.fits_int(length)
        p = np.ascontiguousarray(pages, dtype=np.int32)
        out = np.empty(-(-max(length, 0) // PAGE), np.int32)
        pair = np.empty(2, np.int32)
        ffi.call("higgs_block_pool_fork", self.handle, _i32p(p), p.size, length, _i32p(out), _i32p(pair),
                 _i32p(pair[1:]))
        return out, None if pair[0] < 0 else (int(pair[0]), int(pair[1]))

    def compact(self, max_moves: int | None = None) -> tuple[np.ndarray, np.ndarray]:
        """Packs allocated pages into the lowest ids; the moves (sources, destinations), whose
        pages the caller copies and renames."""
        m = self.num_pages if max_moves is None else min(max_moves, self.num_pages)
        moves = np.empty((2, max(m, 1)), np.int32)
        n = ctypes.c_int(0)
        ffi.call("higgs_block_pool_compact", self.handle, m, _i32p(moves[0]), _i32p(moves[1]), ctypes.byref(n))
        return moves[0, :n.value].copy(), moves[1, :n.value].copy()

    def move(self, src, dst) -> None:
        """Moves the counts of allocated pages src[i] to free pages dst[i]; move(dst, src) takes
        back the moves that compact returned."""
        s = np.ascontiguousarray(src, dtype=np.int32)
        d = np.ascontiguousarray(dst, dtype=np.int32)
        if s.size != d.size:
            raise ValueError("move: lists of different lengths")
        ffi.call("higgs_block_pool_move", self.handle, _i32p(s), _i32p(d), s.size)


class PrefixCache:
    """PrefixCache (prompt_cache.rs:41-311) over whole KV pages."""

    def __init__(self, pool: BlockPool, max_entries: int = 8):
        h = ffi.P()
        ffi.call("higgs_prefix_cache_create", pool.handle, max_entries, ctypes.byref(h))
        self.handle = h.value
        self.pool = pool  # keeps the pool alive

    def __del__(self):
        try:
            ffi.load().higgs_prefix_cache_destroy(self.handle)
        except Exception:
            pass

    def __len__(self) -> int:
        return int(ffi.load().higgs_prefix_cache_len(self.handle))

    def clear(self) -> None:
        ffi.call("higgs_prefix_cache_clear", self.handle)

    def lookup(self, tokens) -> tuple[int, np.ndarray]:
        """(matched_tokens, pages); the returned pages are retained for the caller."""
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        out = np.empty(max(1, t.size // PAGE), np.int32)
        m = ctypes.c_int(0)
        ffi.call("higgs_prefix_cache_lookup", self.handle, _i32p(t), t.size, _i32p(out), out.size,
                 ctypes.byref(m))
        return m.value, out[: m.value // PAGE].copy()

    def store(self, tokens, pages) -> None:
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        p = np.ascontiguousarray(pages, dtype=np.int32)
        ffi.call("higgs_prefix_cache_store", self.handle, _i32p(t), t.size, _i32p(p), p.size)

    def remap(self, src, dst) -> None:
        """Renames pages src[i] -> dst[i] in every entry (after BlockPool.compact)."""
        s = np.ascontiguousarray(src, dtype=np.int32)
        d = np.ascontiguousarray(dst, dtype=np.int32)
        if s.size != d.size:
            raise ValueError("remap: lists of different lengths")
        ffi.call("higgs_prefix_cache_remap", self.handle, _i32p(s), _i32p(d), s.size)

    def uses(self, pages) -> np.ndarray:
        """How many references to each of the pages the entries hold."""
        p = np.ascontiguousarray(pages, dtype=np.int32)
        out = np.empty(p.size, np.int32)
        ffi.call("higgs_prefix_cache_uses", self.handle, _i32p(p), p.size, _i32p(out))
        return out
