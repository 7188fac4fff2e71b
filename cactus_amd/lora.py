"""Low-rank adapters of include/cactus_hip.h from Python: an owner of the
device buffers of one projection's adapters."""
from __future__ import annotations

import numpy as np

from . import DeviceBuffer, call

MAX_RANK = 256


class LoraAdapters:
    """Adapters of one projection [N][K]: up to `count` of them, of any rank up to `rank` (a multiple of 8; lower
    ranks are padded with zeros).  An adapter that was never set adds nothing.  `stream` is a Stream's handle; the
    constructor waits for it, so that calls may follow on any stream."""

    def __init__(self, count: int, rank: int, K: int, N: int, stream=None):
        if rank % 8 or not 8 <= rank <= MAX_RANK:
            raise ValueError(f"rank is a multiple of 8 from 8 to {MAX_RANK}")
        if K % 8 or N % 8 or K < 0 or N < 0:
            raise ValueError("K and N are multiples of 8")
        self.count, self.rank, self.K, self.N = count, rank, K, N
        self._A, self._B, self._scales = DeviceBuffer(2 * count * rank * K), DeviceBuffer(2 * count * N * rank), DeviceBuffer(4 * count)
        for b in (self._A, self._B, self._scales):
            call("cactus_hip_memset", b.ptr, 0, b.nbytes, stream)
        call("cactus_hip_stream_sync", stream)      # calls on other streams are not ordered behind the fills

    def set(self, i: int, A, B, scale: float = 1.0, stream=None):
        """A [r][K] and B [N][r], r at most the rank: y += scale * B (A x).  Waits for the stream."""
        A, B = np.asarray(A, np.float16), np.asarray(B, np.float16)
        if not 0 <= i < self.count:
            raise IndexError(f"no adapter {i}")
        if A.ndim != 2 or A.shape[1] != self.K or not A.shape[0] <= self.rank or B.shape != (self.N, A.shape[0]):
            raise ValueError(f"A [r][{self.K}] and B [{self.N}][r] with r up to {self.rank} are needed")
        r = self.rank - A.shape[0]
        for buf, a in ((self._A, np.pad(A, ((0, r), (0, 0)))), (self._B, np.pad(B, ((0, 0), (0, r)))), (self._scales, np.float32([scale]))):
            a = np.ascontiguousarray(a)
            if a.nbytes:
                call("cactus_hip_memcpy_h2d", buf.ptr + i * a.nbytes, a.ctypes.data, a.nbytes, stream)

    def add(self, x: int, base: int, y: int, adapters: int, batch: int, seq_len: int = 1, counts: int | None = None,
            x_stride: int | None = None, base_stride: int | None = None, y_stride: int | None = None, stream=None):
        """Device pointers as cactus_hip_lora_add_f16 takes them; y may be base."""
        call("cactus_hip_lora_add_f16", x, x_stride or self.K, self._A.ptr, self._B.ptr, self._scales.ptr, self.count, self.rank,
             adapters, counts, base, base_stride or self.N, y, y_stride or (base_stride if y == base else None) or self.N, batch,
             seq_len, self.K, self.N, stream)
