"""The paged 4-bit KV cache of include/cactus_hip.h from Python: the cache
descriptor as a ctypes structure, and an owner of its device buffers."""
from __future__ import annotations

import ctypes
import numbers

import numpy as np

from . import DeviceBuffer, call, hip

NO_PAGES = 1       # CACTUS_HIP_KV4_NO_PAGES
BAD_REQUEST = 2    # CACTUS_HIP_KV4_BAD_REQUEST


class CacheDesc(ctypes.Structure):
    """cactus_hip_kv4_cache: pass `desc.ref` as the entry points' cache."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("pages", "table", "lens", "refs", "state")] + \
               [(n, ctypes.c_size_t) for n in ("layers", "kv_heads", "head_dim", "page_size", "num_pages", "max_seqs",
                                               "max_pages")]

    @property
    def ref(self):
        return ctypes.byref(self)


class _List(DeviceBuffer):
    """A list of slots, counts or pages that a call uploaded."""


class KV4Cache:
    """Pages, tables and workspace of one cache, set up by cactus_hip_kv4_reset.

    The methods take device pointers (DeviceBuffer.ptr, or any integer) where
    the entry points do; slot and page lists may be sequences of ints, which
    are uploaded first (the call then waits for the stream).  `stream` is a
    Stream's handle.  Scratch memory is kept per stream: calls on two streams, also
    from two threads, may overlap as the entry points say.  In a capture give
    pointers, and make the same call once before it, so that the scratch memory is
    there; a graph that may overlap eager calls needs the entry points and a
    workspace of its own."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, page_size: int, num_pages: int, max_seqs: int,
                 max_pages: int, stream=None):
        self.desc = CacheDesc(layers=layers, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size,
                              num_pages=num_pages, max_seqs=max_seqs, max_pages=max_pages)
        n = ctypes.c_size_t()
        call("cactus_hip_kv4_bytes", self.desc.ref, ctypes.byref(n))
        self._buf = {"pages": DeviceBuffer(n.value), "table": DeviceBuffer(4 * max_seqs * max_pages),
                     "lens": DeviceBuffer(4 * max_seqs), "refs": DeviceBuffer(4 * num_pages), "state": DeviceBuffer(16)}
        for name, b in self._buf.items():
            setattr(self.desc, name, b.ptr)
        self._work = {}
        self.reset(stream)

    def _lst(self, v, n: int, stream=None):
        """A device pointer as it is; a sequence of n ints or more uploaded, for the call that it is made for."""
        if v is None or isinstance(v, numbers.Integral):
            return None if v is None else int(v)
        a = np.asarray(v)
        if a.ndim != 1 or len(a) < n:
            raise ValueError(f"a list of {n} integers is needed")
        if n == 0:
            return None
        if a.dtype.kind not in "iu":
            raise TypeError("a list of integers is needed")
        if a.min() < -(1 << 31) or a.max() >= 1 << 31:
            raise OverflowError("a list of 32-bit integers is needed")
        return _List.from_numpy(a.astype(np.int32), stream)

    @staticmethod
    def _pairs(src, dst) -> int:
        if len(src) != len(dst):
            raise ValueError(f"{len(src)} sources, {len(dst)} destinations")
        return len(src)

    def _call(self, name, *args, stream=None):
        # uploaded lists belong to this call, whatever other threads do, and go once it has read them
        lists = [a for a in args if isinstance(a, _List)]
        try:
            call(name, self.desc.ref, *(a.ptr if isinstance(a, _List) else a for a in args), stream)
        finally:
            if lists:
                call("cactus_hip_stream_sync", stream)

    def workspace(self, nbytes: int, stream=None):
        """At least nbytes of scratch memory for calls on `stream`, the first 4096 bytes zero."""
        work = self._work.setdefault(stream or 0, [])
        last = work[-1] if work else None
        if last is None or last.nbytes < nbytes:
            # a smaller one stays: a captured graph may hold its address
            last = DeviceBuffer(max(nbytes, 4096))
            call("cactus_hip_memset", last.ptr, 0, 4096, stream)
            work.append(last)
        return last.ptr, last.nbytes

    def reset(self, stream=None):
        self._call("cactus_hip_kv4_reset", stream=stream)

    def status(self, stream=None) -> int:
        s = ctypes.c_int()
        call("cactus_hip_kv4_status", self.desc.ref, ctypes.byref(s), stream)
        return s.value

    def extend(self, batch: int, count: int = 0, seqs=None, counts=None, stream=None):
        self._call("cactus_hip_kv4_extend", self._lst(seqs, batch, stream), self._lst(counts, batch, stream), batch, count,
                   stream=stream)

    def append(self, layer: int, k: int, v: int, batch: int, seq_len: int, kv_stride: int | None = None, seqs=None,
               counts=None, stream=None):
        stride = kv_stride or self.desc.kv_heads * self.desc.head_dim
        self._call("cactus_hip_kv4_append_f16", layer, self._lst(seqs, batch, stream), self._lst(counts, batch, stream), k, v,
                   batch, seq_len, stride, stream=stream)

    def read(self, layer: int, k: int, v: int, batch: int, seq_len: int, seqs=None, starts=None, counts=None, stream=None):
        self._call("cactus_hip_kv4_read_f16", layer, self._lst(seqs, batch, stream), self._lst(starts, batch, stream),
                   self._lst(counts, batch, stream), k, v, batch, seq_len, stream=stream)

    def attention(self, layer: int, q: int, o: int, batch: int, seq_len: int, num_q_heads: int, scale: float = 0.0,
                  window: int = 0, sink: int = 0, causal: bool = True, q_stride: int | None = None, seqs=None,
                  counts=None, stream=None):
        need = hip().cactus_hip_attention_kv4_workspace(self.desc.ref, batch, seq_len, num_q_heads)
        work, size = self.workspace(need, stream)
        stride = q_stride or num_q_heads * self.desc.head_dim
        self._call("cactus_hip_attention_kv4_f16", layer, self._lst(seqs, batch, stream), self._lst(counts, batch, stream), q,
                   stride, o, batch, seq_len, num_q_heads, scale, window, sink, int(causal), work, size, stream=stream)

    def fork(self, src, dst, n: int | None = None, stream=None):
        n = self._pairs(src, dst) if n is None else n
        work, size = self.workspace(hip().cactus_hip_kv4_pages_workspace(self.desc.ref, n), stream)
        self._call("cactus_hip_kv4_fork", self._lst(src, n, stream), self._lst(dst, n, stream), n, work, size, stream=stream)

    def free(self, seqs, n: int | None = None, stream=None):
        n = len(seqs) if n is None else n
        self._call("cactus_hip_kv4_free", self._lst(seqs, n, stream), n, stream=stream)

    def compact(self, stream=None):
        work, size = self.workspace(hip().cactus_hip_kv4_pages_workspace(self.desc.ref, 0), stream)
        self._call("cactus_hip_kv4_compact", work, size, stream=stream)

    def copy_pages(self, src, dst, n: int | None = None, stream=None):
        n = self._pairs(src, dst) if n is None else n
        self._call("cactus_hip_kv4_copy_pages", self._lst(src, n, stream), self._lst(dst, n, stream), n, stream=stream)

    def tables(self, stream=None) -> dict:
        """Host copies of table, lens, refs and state."""
        d = self.desc
        shapes = {"table": (d.max_seqs, d.max_pages), "lens": (d.max_seqs,), "refs": (d.num_pages,), "state": (4,)}
        return {n: self._buf[n].to_numpy(np.int32, s, stream) for n, s in shapes.items()}
