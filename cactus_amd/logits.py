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
        self._buf, self._part, self._work = {}, {}, {}
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
            self._part[name] = a.dtype.type, a.shape[1] if a.ndim > 1 else 1
            setattr(self.desc, name, self._buf[name].ptr)

    def _put(self, slot: int, stream, rows: int | None = None, **parts):
        """Uploads a slot's (or a mask's) part of each named array; checks all of them first."""
        if not 0 <= slot < (self.desc.max_seqs if rows is None else rows):
            raise IndexError(f"no slot or mask {slot}")
        ready = []
        for name, values in parts.items():
            kind, stride = self._part.get(name, (None, 0))
            a = np.asarray(values)
            if kind is None or a.size > stride:
                raise ValueError(f"{name}: room for {stride} values, {a.size} given")
            if a.size and kind != np.float32 and (a.dtype.kind not in "iu" or a.min() < np.iinfo(kind).min or a.max() > np.iinfo(kind).max):
                raise TypeError(f"{name}: 32-bit integers are needed")
            if a.size and kind == np.float32 and a.dtype.kind not in "fiub":
                raise TypeError(f"{name}: numbers are needed")
            ready.append((self._buf[name].ptr + 4 * slot * stride, np.ascontiguousarray(a, kind)))
        for ptr, a in ready:
            if a.size:
                call("cactus_hip_memcpy_h2d", ptr, a.ctypes.data, a.nbytes, stream)

    def set_history(self, slot: int, tokens, stream=None):
        self._put(slot, stream, history=tokens, history_lens=[np.size(tokens)])

    def set_penalties(self, slot: int, repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0, stream=None):
        self._put(slot, stream, repetition=[repetition], frequency=[frequency], presence=[presence])

    def set_bias(self, slot: int, tokens, values, stream=None):
        if np.size(tokens) != np.size(values):
            raise ValueError(f"{np.size(tokens)} tokens, {np.size(values)} values")
        self._put(slot, stream, bias_tokens=tokens, bias_values=values, bias_counts=[np.size(tokens)])

    def set_mask(self, mask: int, allowed, stream=None):
        """allowed: a truth value per token."""
        a = np.asarray(allowed, bool)
        if a.shape != (self.vocab,):
            raise ValueError(f"{self.vocab} truth values are needed")
        bits = np.packbits(np.pad(a, (0, -len(a) % 32)), bitorder="little").view(np.uint32)
        self._put(mask, stream, self.desc.num_masks, masks=bits)

    def use_mask(self, slot: int, mask: int, stream=None):
        """Mask number `mask` for the slot; -1: none; num_masks or more: no token is allowed."""
        self._put(slot, stream, mask_ids=[mask])

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
