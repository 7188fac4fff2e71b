"""The rules on logits of include/cactus_hip.h from Python: the settings'
descriptor as a ctypes structure, and an owner of its device buffers."""
from __future__ import annotations

import ctypes

import numpy as np

from . import DeviceBuffer, call, hip

MAX_BIAS = 1024      # CACTUS_HIP_LOGITS_MAX_BIAS


class RulesDesc(ctypes.Structure):
    """cactus_hip_logits_rules: pass `desc.ref` as the entry points' rules."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("history", "history_lens", "repetition", "frequency", "presence", "bias_tokens",
                                               "bias_values", "bias_counts", "masks", "mask_ids")] + \
               [(n, ctypes.c_size_t) for n in ("history_stride", "bias_stride", "num_masks", "mask_stride", "max_seqs")]

    @property
    def ref(self):
        return ctypes.byref(self)


class LogitsRules:
    """Settings of max_seqs sequences: tokens seen so far with their penalties, up to max_bias
    biases, and one of num_masks masks over the vocabulary.  The setters upload one slot's
    part and wait for the stream; a slot starts with none of them.  `stream` is a Stream's handle."""

    def __init__(self, max_seqs: int, vocab: int, max_history: int = 0, max_bias: int = 0, num_masks: int = 0, stream=None):
        if max_bias > MAX_BIAS:
            raise ValueError(f"at most {MAX_BIAS} biases")
        self.vocab, words = vocab, -(-vocab // 32)
        self.desc = RulesDesc(history_stride=max_history, bias_stride=max_bias, num_masks=num_masks, mask_stride=words,
                              max_seqs=max_seqs)
        self._buf, self._work = {}, {}
        start = {}
        if max_history:
            start.update(history=np.full((max_seqs, max_history), -1, np.int32), history_lens=np.zeros(max_seqs, np.int32),
                         repetition=np.ones(max_seqs, np.float32), frequency=np.zeros(max_seqs, np.float32),
                         presence=np.zeros(max_seqs, np.float32))
        if max_bias:
            start.update(bias_tokens=np.full((max_seqs, max_bias), -1, np.int32),
                         bias_values=np.zeros((max_seqs, max_bias), np.float32), bias_counts=np.zeros(max_seqs, np.int32))
        if num_masks:
            start.update(masks=np.full((num_masks, words), 0xFFFFFFFF, np.uint32), mask_ids=np.full(max_seqs, -1, np.int32))
        for name, a in start.items():
            self._buf[name] = DeviceBuffer.from_numpy(a, stream)
            setattr(self.desc, name, self._buf[name].ptr)

    def _put(self, name: str, slot: int, values, dtype, stride: int, stream, rows: int | None = None):
        a = np.asarray(values)
        if np.issubdtype(dtype, np.integer) and a.size and (a.dtype.kind not in "iu" or a.min() < np.iinfo(dtype).min or a.max() > np.iinfo(dtype).max):
            raise TypeError(f"{name}: 32-bit integers are needed")
        a = np.ascontiguousarray(a, dtype)
        if not 0 <= slot < (self.desc.max_seqs if rows is None else rows):
            raise IndexError(f"no slot or mask {slot}")
        if name not in self._buf or a.size > stride:
            raise ValueError(f"{name}: room for {stride if name in self._buf else 0} values, {a.size} given")
        if a.size:
            call("cactus_hip_memcpy_h2d", self._buf[name].ptr + 4 * slot * stride, a.ctypes.data, a.nbytes, stream)
        return a.size

    def set_history(self, slot: int, tokens, stream=None):
        n = self._put("history", slot, tokens, np.int32, self.desc.history_stride, stream)
        self._put("history_lens", slot, [n], np.int32, 1, stream)

    def set_penalties(self, slot: int, repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0, stream=None):
        for name, v in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
            self._put(name, slot, [v], np.float32, 1, stream)

    def set_bias(self, slot: int, tokens, values, stream=None):
        if len(tokens) != len(values):
            raise ValueError(f"{len(tokens)} tokens, {len(values)} values")
        n = self._put("bias_tokens", slot, tokens, np.int32, self.desc.bias_stride, stream)
        self._put("bias_values", slot, values, np.float32, self.desc.bias_stride, stream)
        self._put("bias_counts", slot, [n], np.int32, 1, stream)

    def set_mask(self, mask: int, allowed, stream=None):
        """allowed: a truth value per token."""
        a = np.asarray(allowed, bool)
        if a.shape != (self.vocab,):
            raise ValueError(f"{self.vocab} truth values are needed")
        bits = np.packbits(np.pad(a, (0, -len(a) % 32)), bitorder="little").view(np.uint32)
        self._put("masks", mask, bits, np.uint32, self.desc.mask_stride, stream, self.desc.num_masks)

    def use_mask(self, slot: int, mask: int, stream=None):
        """Mask number `mask` for the slot; -1: none."""
        self._put("mask_ids", slot, [mask], np.int32, 1, stream)

    def apply(self, logits: int, out: int, batch: int, best: int | None = None, fp32: bool = False, stride: int | None = None,
              out_stride: int | None = None, seqs: int | None = None, stream=None):
        """Device pointers as the entry points take them.  The best tokens' scratch memory is kept per stream:
        in a capture make the same call once before it; a graph that may overlap eager calls
        needs the entry points and a workspace of its own."""
        work, size = None, 0
        if best is not None:
            size = hip().cactus_hip_logits_rules_workspace(batch)
            kept = self._work.setdefault(stream or 0, [])
            last = kept[-1] if kept else None
            if last is None or last.nbytes < size:
                # a smaller one stays: a captured graph may hold its address
                last = DeviceBuffer(size)
                call("cactus_hip_memset", last.ptr, 0, size, stream)
                kept.append(last)
            work, size = last.ptr, last.nbytes
        call("cactus_hip_logits_rules_f32" if fp32 else "cactus_hip_logits_rules_f16", self.desc.ref, seqs, logits,
             stride or self.vocab, out, out_stride or self.vocab, best, batch, self.vocab, work, size, stream)
