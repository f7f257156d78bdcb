"""A cache of stream states in pages: streams branch, end and move together without copying more than they must.

    from yggdrasil_b200 import StateCache
    cache = StateCache.empty(pages=4096, streams=1024, like=model.init_state(1))   # a page: one stream's state
    cache.grow([0, 1])                    # streams 0 and 1 get their first page (zeros)
    cache.fork([0, 0, 1], [2, 3, 4])      # 2 and 3 go on from 0, 4 from 1
    state = cache.read([2, 3, 4])         # (3, layers, n), for model.step
    cache.write([2, 3, 4], new_state)
    cache.free([0, 1])
    live = cache.compact()                # the live pages are cache.pages[:live] now
    cache.status()                        # raises if a call met a bad index or had no room

`table[s, :length[s]]` are the pages of stream s (-1 beyond). The last one is its live state, its own; those before are
snapshots (`grow` leaves one behind), which forks share: `refs[p]` counts the table entries that hold page p. A fork may
go back to a snapshot (`depth`). Everything stays on the device, on the current stream; the kernels are
csrc/ygg_pages.cu. Calls on one cache are ordered by their stream; a cache used on several streams at once is the
caller's to order. A cache has to live as long as the CUDA graphs that captured calls on it. Pages hold values: a batch or
pages that ask for a gradient are refused.
"""
from __future__ import annotations

import threading
import weakref

import numpy as np
import torch

from . import _native, _ops

_SLOTS = 1024
_lock = threading.Lock()
_pools: dict = {}   # device index -> _Pool


class _Chunk:
    """The words of _SLOTS caches, each handed out once: three of status (pinned host memory, which the device can write) and
    a 64-bit one for a cache's barriers (device memory), all zero."""

    def __init__(self, index):
        self.status = torch.zeros((_SLOTS, 4), dtype=torch.int32).pin_memory()
        self.sync = torch.zeros(_SLOTS, dtype=torch.int64, device=torch.device("cuda", index))
        self.status_at, self.sync_at = self.status.data_ptr(), self.sync.data_ptr()
        torch.cuda.current_stream(index).synchronize()   # zero for a cache on any stream

    def renew(self, index):
        torch.cuda.synchronize(index)
        self.status.zero_()
        self.sync.zero_()
        torch.cuda.current_stream(index).synchronize()


class _Hold:
    """Kept by the caches of a chunk: it tells whether any is left."""


class _Pool:
    """A device's chunks. A cache may go while calls on it are on their way, on whatever stream: its words stay, and serve
    again only when no cache of their chunk is left and the device has been waited for (once in _SLOTS caches at most). The
    next chunk is got ready early, outside graph captures, so that a cache can be made inside one."""

    def __init__(self, index):
        self.index, self.chunk, self.hold, self.spare, self.old = index, None, None, None, []
        self.used = self.until = 0   # words handed out of the chunk, and up to when without a further look

    def fresh(self):
        for i, (chunk, held) in enumerate(self.old):
            if held() is None:
                chunk.renew(self.index)
                del self.old[i]
                return chunk
        return _Chunk(self.index)

    def look(self):
        if self.chunk is None or self.used == _SLOTS:
            chunk = self.spare or self.fresh()
            if self.chunk is not None:
                self.old.append((self.chunk, weakref.ref(self.hold)))
            self.chunk, self.hold, self.spare = chunk, _Hold(), None
            self.used, self.until = 0, _SLOTS // 2
        elif torch.cuda.is_current_stream_capturing():
            self.until = self.used + 1
        else:
            self.spare, self.until = self.fresh(), _SLOTS


def _words(index):
    """Words of a cache's own: their chunk, which of them, and what to keep as long as the cache lives."""
    with _lock:
        pool = _pools.get(index)
        if pool is None:
            pool = _pools[index] = _Pool(index)
        if pool.used >= pool.until:
            pool.look()
        pool.used += 1
        return pool.chunk, pool.used - 1, pool.hold


class StateCache:
    def __init__(self, pages, table, length, refs):
        """Around tensors that hold a cache already (updated in place): pages (P, ...) of any type, table (S, M), length
        (S,) and refs (P,) int32, contiguous, on one CUDA device."""
        self._h = None
        if isinstance(pages, torch.Tensor) and pages.is_cuda:
            chunk, self._at, self._hold = _words(pages.get_device())
            self._status, self._sync = chunk.status, chunk.sync
            self._h = _ops.cache(pages, table, length, refs, chunk.status_at + 16 * self._at, chunk.sync_at + 8 * self._at)
        if self._h is None:
            raise ValueError("a cache needs contiguous tensors on one CUDA device: pages (P, ...), table (S, M) int32, "
                             "length (S,) int32 and refs (P,) int32")
        self.pages, self.table, self.length, self.refs = pages, table, length, refs
        self.device = pages.device

    @classmethod
    def empty(cls, pages, streams, per_stream=1, like=None, shape=None, dtype=None, device=None):
        """A cache without live pages. A page has `shape` and `dtype` (on `device`), or those of a state `like`
        (1, layers, n) as model.init_state(1) gives it."""
        if like is not None:
            shape, dtype, device = like.shape[1:], like.dtype, like.device
        if pages < 1 or streams < 1 or per_stream < 1 or shape is None:
            raise ValueError("a cache needs pages, streams, a table row and the shape of a page")
        device = torch.device(device if device is not None else "cuda")
        if device.type != "cuda":
            raise ValueError(f"device {device}: the cache lives on a CUDA device")
        ints = lambda *size, v=0: torch.full(size, v, dtype=torch.int32, device=device)  # noqa: E731
        return cls(torch.empty((pages, *shape), dtype=dtype, device=device), ints(streams, per_stream, v=-1),
                   ints(streams), ints(pages))

    def _ids(self, ids, what, limit):
        """Indices as a contiguous int32 tensor on the device; host indices are range-checked (negative: padding)."""
        if isinstance(ids, torch.Tensor) and ids.is_cuda:
            if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64) or ids.device != self.device:
                raise ValueError(f"{what} must be a row of int32 or int64 on {self.device}")
            return (ids if ids.dtype == torch.int32 else ids.clamp(-1, 2 ** 31 - 1).int()).contiguous()
        host = np.asarray(ids)
        if host.ndim != 1 or (host.size and host.dtype.kind not in "iu"):
            raise ValueError(f"{what} must be a row of integers")
        if host.size and host.max() >= limit:
            raise ValueError(f"{what}: {int(host.max())} out of range [0, {limit})")
        host = np.maximum(host.astype(np.int64), -1)   # as below -2^31 on the device: padding, whatever its low 32 bits say
        return torch.as_tensor(host.astype(np.int32)).to(self.device)

    def _streams(self, ids, what="streams"):
        return self._ids(ids, what, self.table.shape[0])

    def fork(self, parents, children, depth=None):
        """Stream children[i], which must hold no pages, goes on from parents[i]: it shares the parent's pages but the
        last, which is copied into a new page. depth[i]: only the parent's first depth[i] pages (at least 1), so that
        the child goes on from an earlier snapshot. A parent without pages leaves its child without."""
        if children is None or _ops.cache_fork(self._h, parents, children, depth) is None:
            p, c = self._streams(parents, "parents"), self._streams(children, "children")
            d = None if depth is None else self._ids(depth, "depth", 1 << 31)
            if p.shape != c.shape or (d is not None and d.shape != p.shape):
                raise ValueError("one child, and one depth, for each parent")
            _ops.cache_fork(self._h, p, c, d)

    def grow(self, streams):
        """Each stream gets one more page, a copy of its last (zeros for its first); the page before it stays as a
        snapshot."""
        if _ops.cache_fork(self._h, streams, None, None) is None:
            _ops.cache_fork(self._h, self._streams(streams), None, None)

    def free(self, streams):
        """The streams let go of their pages; pages that nothing holds any more are free."""
        if _ops.cache_free(self._h, streams) is None:
            _ops.cache_free(self._h, self._streams(streams))

    def compact(self):
        """Moves the live pages to the front and renumbers the tables. Returns their number as an int32 tensor () on the
        device: pages[:live] is one contiguous batch."""
        return _ops.cache_compact(self._h)

    def read(self, streams):
        """The live states of streams as a new batch (len(streams), ...); zeros for a stream without pages."""
        batch = _ops.cache_read(self._h, streams)
        return batch if batch is not None else _ops.cache_read(self._h, self._streams(streams))

    def write(self, streams, batch):
        """batch[i] becomes the live state of streams[i], a stream that holds pages; no stream named twice, and the batch
        no part of the pages themselves."""
        if _ops.cache_write(self._h, streams, batch) is None:
            s = self._streams(streams)
            want = (s.shape[0], *self.pages.shape[1:])
            if not isinstance(batch, torch.Tensor) or batch.dtype != self.pages.dtype or batch.device != self.device \
                    or batch.shape != want:
                raise ValueError(f"batch must be {self.pages.dtype} {want} on {self.device}")
            _ops.cache_write(self._h, s, batch.contiguous())

    def copy(self, source, target):
        """Page target[i] becomes a copy of page source[i]; a target is named once, and is no source of the call."""
        if _ops.cache_copy(self._h, source, target) is None:
            count = self.pages.shape[0]
            a, b = self._ids(source, "source", count), self._ids(target, "target", count)
            if a.shape != b.shape:
                raise ValueError("one target for each source")
            _ops.cache_copy(self._h, a, b)

    def status(self, clear=True):
        """Raise if a call since the last clear met a bad index (ValueError) or had no page or table entry left
        (RuntimeError); what such a call could do it did. Waits for the current stream. A cache whose blocks once gave up
        waiting for each other (YggError with YGG_E_TIMEOUT) stays unusable: clear does not clear that."""
        torch.cuda.current_stream(self.device).synchronize()
        words = self._status[self._at]
        bad, full, late, _ = words.tolist()
        if clear:
            words[:2].zero_()
        if late:
            raise _native.YggError(_native.YGG_E_TIMEOUT, "StateCache: not to be used any more")
        if bad:
            raise ValueError("a stream or page was out of range, a child held pages or was named twice, or a table named a "
                             "page that is not the cache's")
        if full:
            raise _native.YggError(_native.YGG_E_CAPACITY, "StateCache", "no free page, or a full table row")
