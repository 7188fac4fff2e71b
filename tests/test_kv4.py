"""The paged 4-bit KV cache without a GPU: refusals before any launch, sizes,
and the restatement's own quantization."""
import ctypes
import gc

import numpy as np
import pytest

from _kv4 import code_at, quantize, scale_at, values


@pytest.fixture(scope="module")
def lib():
    import cactus_amd
    return cactus_amd.hip()


def desc(**kw):
    from cactus_amd.kv4 import CacheDesc
    shape = dict(layers=2, kv_heads=2, head_dim=128, page_size=64, num_pages=8, max_seqs=4, max_pages=4)
    ptrs = dict(pages=1 << 20, table=1 << 21, lens=1 << 22, refs=1 << 23, state=1 << 24)   # never dereferenced
    return CacheDesc(**{**shape, **ptrs, **kw})


def refused(lib, rc, text):
    assert rc == -1
    assert text in lib.cactus_hip_last_error(), lib.cactus_hip_last_error()


BAD = [(dict(head_dim=96), b"head_dim"), (dict(head_dim=0), b"head_dim"), (dict(page_size=48), b"page_size"),
       (dict(page_size=8), b"page_size"), (dict(page_size=8192), b"page_size"), (dict(kv_heads=0), b"kv_heads"),
       (dict(layers=0), b"layers"), (dict(num_pages=0), b"num_pages"), (dict(num_pages=1 << 40), b"num_pages"),
       (dict(max_seqs=0), b"max_seqs"), (dict(max_seqs=70000), b"max_seqs"), (dict(max_pages=1 << 26), b"max_pages")]


@pytest.mark.parametrize("change,text", BAD + [(dict(pages=None), b"null buffer"), (dict(table=None), b"null buffer"),
                                               (dict(state=None), b"null buffer"), (dict(pages=(1 << 20) + 64), b"aligned")])
def test_every_call_checks_the_cache(lib, change, text):
    c = desc(**change).ref
    p = 4096
    refused(lib, lib.cactus_hip_kv4_reset(c, None), text)
    refused(lib, lib.cactus_hip_kv4_extend(c, None, None, 1, 1, None), text)
    refused(lib, lib.cactus_hip_kv4_append_f16(c, 0, None, None, p, p, 1, 1, 256, None), text)
    refused(lib, lib.cactus_hip_kv4_read_f16(c, 0, None, None, None, p, p, 1, 1, None), text)
    refused(lib, lib.cactus_hip_attention_kv4_f16(c, 0, None, None, p, 256, p, 1, 1, 2, 0.0, 0, 0, 1, p, 1 << 30, None), text)
    refused(lib, lib.cactus_hip_kv4_fork(c, p, p, 1, p, 1 << 30, None), text)
    refused(lib, lib.cactus_hip_kv4_free(c, None, 1, None), text)
    refused(lib, lib.cactus_hip_kv4_compact(c, p, 1 << 30, None), text)
    refused(lib, lib.cactus_hip_kv4_copy_pages(c, p, p, 1, None), text)
    refused(lib, lib.cactus_hip_kv4_status(c, p, None), text)


@pytest.mark.parametrize("change,text", BAD)
def test_sizes_check_the_shape(lib, change, text):
    c = desc(**change).ref
    n = ctypes.c_size_t()
    refused(lib, lib.cactus_hip_kv4_bytes(c, ctypes.byref(n)), text)
    assert lib.cactus_hip_kv4_pages_workspace(c, 1) == 0
    assert lib.cactus_hip_attention_kv4_workspace(c, 1, 1, 2) == 0


def test_null_cache_and_sizes(lib):
    n = ctypes.c_size_t()
    refused(lib, lib.cactus_hip_kv4_bytes(None, ctypes.byref(n)), b"null")
    refused(lib, lib.cactus_hip_kv4_bytes(desc().ref, None), b"null")
    assert lib.cactus_hip_kv4_bytes(desc().ref, ctypes.byref(n)) == 0
    assert n.value == 2 * 8 * 2 * 64 * 128 * 9 // 8
    assert lib.cactus_hip_kv4_pages_workspace(desc().ref, 3) >= 4096
    assert lib.cactus_hip_attention_kv4_workspace(desc().ref, 1, 1, 4) >= 4096


def test_refused_arguments(lib):
    c, p, big = desc().ref, 4096, 1 << 30
    refused(lib, lib.cactus_hip_kv4_append_f16(c, 2, None, None, p, p, 1, 1, 256, None), b"layer")
    refused(lib, lib.cactus_hip_kv4_append_f16(c, 0, None, None, None, p, 1, 1, 256, None), b"null")
    refused(lib, lib.cactus_hip_kv4_append_f16(c, 0, None, None, p, p + 8, 1, 1, 256, None), b"aligned")
    refused(lib, lib.cactus_hip_kv4_append_f16(c, 0, None, None, p, p, 1, 1, 260, None), b"aligned")
    refused(lib, lib.cactus_hip_kv4_append_f16(c, 0, None, None, p, p, 1, 1, 248, None), b"kv_stride")
    refused(lib, lib.cactus_hip_kv4_append_f16(c, 0, None, None, p, p, 5, 1, 256, None), b"slots")
    refused(lib, lib.cactus_hip_kv4_read_f16(c, 0, None, None, None, p, p + 2, 1, 1, None), b"aligned")
    refused(lib, lib.cactus_hip_kv4_extend(c, None, None, 5, 1, None), b"slots")
    refused(lib, lib.cactus_hip_kv4_extend(c, None, None, 1, 1 << 31, None), b"count")
    att = lib.cactus_hip_attention_kv4_f16
    refused(lib, att(c, 0, None, None, None, 256, p, 1, 1, 2, 0.0, 0, 0, 1, p, big, None), b"null")
    refused(lib, att(c, 0, None, None, p, 384, p, 1, 1, 3, 0.0, 0, 0, 1, p, big, None), b"num_q_heads")
    refused(lib, att(c, 0, None, None, p, 128, p, 1, 1, 2, 0.0, 0, 0, 1, p, big, None), b"q_stride")
    refused(lib, att(c, 0, None, None, p + 2, 256, p, 1, 1, 2, 0.0, 0, 0, 1, p, big, None), b"aligned")
    refused(lib, att(c, 0, None, None, p, 256, p + 8, 1, 1, 2, 0.0, 0, 0, 1, p, big, None), b"aligned")
    refused(lib, att(c, 0, None, None, p, 256, p, 1, 1, 2, 0.0, 0, 0, 1, None, big, None), b"workspace")
    refused(lib, att(c, 0, None, None, p, 256, p, 1, 1, 2, 0.0, 0, 0, 1, p + 128, big, None), b"workspace")
    refused(lib, att(c, 0, None, None, p, 256, p, 1, 1, 2, 0.0, 0, 0, 1, p, 64, None), b"workspace")
    refused(lib, att(c, 0, None, None, p, 256, p, 1, 1 << 30, 2, 0.0, 0, 0, 1, p, big, None), b"seq_len")
    refused(lib, att(c, 2, None, None, p, 256, p, 1, 1, 2, 0.0, 0, 0, 1, p, big, None), b"layer")
    refused(lib, lib.cactus_hip_kv4_fork(c, None, p, 1, p, big, None), b"null")
    refused(lib, lib.cactus_hip_kv4_fork(c, p, p, 5, p, big, None), b"slots")
    refused(lib, lib.cactus_hip_kv4_fork(c, p, p, 1, p, 4096, None), b"workspace")
    refused(lib, lib.cactus_hip_kv4_compact(c, p, 4096, None), b"workspace")
    refused(lib, lib.cactus_hip_kv4_copy_pages(c, p, None, 1, None), b"null")
    refused(lib, lib.cactus_hip_kv4_copy_pages(c, p, p, 9, None), b"pages")
    refused(lib, lib.cactus_hip_kv4_status(c, None, None), b"null")
    # more stages of keys than the kernels count: 128 and, with dims of 256 and many rows, 64 keys each
    for change, rows in ((dict(head_dim=256), 65), (dict(head_dim=64), 65), (dict(head_dim=256), 1)):
        wide = desc(page_size=16, max_pages=1 << 20, kv_heads=1, **change).ref
        batch = (8192 if change["head_dim"] == 256 else 16384) if rows > 1 else 16384
        assert att(wide, 0, None, None, p, 256, p, batch, rows, 1, 0.0, 0, 0, 1, p, big, None) == -2
        assert b"too large" in lib.cactus_hip_last_error()
    # nothing to do is no error and no launch
    assert lib.cactus_hip_kv4_append_f16(c, 0, None, None, None, None, 0, 1, 256, None) == 0
    assert att(c, 0, None, None, None, 0, None, 1, 0, 2, 0.0, 0, 0, 1, None, 0, None) == 0
    assert lib.cactus_hip_kv4_extend(c, None, None, 0, 1, None) == 0
    assert lib.cactus_hip_kv4_fork(c, None, None, 0, None, 0, None) == 0
    assert lib.cactus_hip_kv4_free(c, None, 0, None) == 0
    assert lib.cactus_hip_kv4_copy_pages(c, None, None, 0, None) == 0


def test_lists_of_the_python_owner():
    from cactus_amd.kv4 import KV4Cache
    c = KV4Cache.__new__(KV4Cache)
    assert c._lst(None, 3) is None and c._lst([], 0) is None
    assert c._lst(np.int64(1 << 40), 3) == 1 << 40         # a pointer, whatever the integer's type
    for bad in ([0], [[0, 1], [2, 3]], [0.5, 1, 2], [1, 2, 1 << 31]):      # too short, not a list, not numbers of slots
        with pytest.raises((ValueError, TypeError, OverflowError)):
            c._lst(bad, 2)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_layout_gives_every_code_and_scale_a_place_of_its_own(d):
    nibbles = {code_at(d, k, i, v) for k in range(16) for i in range(d) for v in (False, True)}
    scales = {scale_at(d, k, g, v) + b for k in range(16) for g in range(d // 32) for v in (False, True) for b in (0, 1)}
    assert len(nibbles) == 2 * 16 * d and len(scales) == 2 * 16 * (d // 32) * 2
    assert {b for b, _ in nibbles} | scales == set(range(18 * d)) and not {b for b, _ in nibbles} & scales


def test_the_quantized_values_are_exact_fp16_numbers_near_the_input():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((400, 64)) * np.exp(3 * rng.standard_normal((400, 1)))).astype(np.float16)
    x[0], x[1], x[2] = 0, 65504, np.float16(2.0 ** -24)
    c, s = quantize(x)
    y = values(c, s).reshape(x.shape)
    assert np.abs(c).max() == 7
    np.testing.assert_array_equal(y, y.astype(np.float16).astype(np.float64))
    # half a step, and what the rounded scale leaves of the largest value (2^-9 of it, or half of 2^-24 per code)
    g = np.abs(x.astype(np.float64)).reshape(400, -1, 32).max(-1).repeat(32, -1)
    bound = np.repeat(s.astype(np.float64), 32, -1).reshape(x.shape) / 2 + g * 2.0 ** -9 + 7 * 2.0 ** -25
    assert (np.abs(y - x) <= bound).all()


class Memory:
    """Stands in for the library: which allocations live, and which lists the queued work of each stream reads."""

    def __init__(self, monkeypatch):
        import cactus_amd
        self.live, self.queued, self.wrong, self.hooks = set(), {}, [], {}
        self.next, self.uploads = 1 << 20, 0
        monkeypatch.setattr(cactus_amd, "call", self.call)
        monkeypatch.setattr("cactus_amd.kv4.call", self.call)
        monkeypatch.setattr(cactus_amd, "hip", lambda: self)
        monkeypatch.setattr("cactus_amd.kv4.hip", lambda: self)

    def call(self, name, *args):
        if name == "cactus_hip_malloc":
            self.next += 4096
            args[0]._obj.value = self.next
            self.live.add(self.next)
        elif name == "cactus_hip_kv4_bytes":
            args[1]._obj.value = 4096
        elif name == "cactus_hip_stream_sync":
            self.queued[args[0]] = set()
        elif name in ("cactus_hip_kv4_extend", "cactus_hip_kv4_fork"):
            lists = set(args[1:3])
            if not lists <= self.live:
                self.wrong.append(f"{name} given freed lists on stream {args[-1]}")
            self.queued.setdefault(args[-1], set()).update(lists)
            if name in self.hooks:
                self.hooks.pop(name)()
            if name == "cactus_hip_kv4_fork":
                raise RuntimeError("refused behind its first launch")
        self.uploads += name == "cactus_hip_memcpy_h2d"
        if self.uploads == 2 and "second upload" in self.hooks:
            self.hooks.pop("second upload")()

    def cactus_hip_free(self, p):
        self.live.discard(p)
        self.wrong += [f"list freed under stream {s}" for s, lists in self.queued.items() if p in lists]

    def cactus_hip_kv4_pages_workspace(self, cache, n):
        return 8192


@pytest.mark.parametrize("when", ["second upload", "cactus_hip_kv4_extend"])
def test_lists_of_a_call_outlive_another_threads_call(monkeypatch, when):
    """A second thread's whole call falls between this one's upload, launch and wait."""
    import threading
    from cactus_amd.kv4 import KV4Cache
    mem = Memory(monkeypatch)
    c = KV4Cache(1, 1, 64, 16, 8, 4, 4)

    def other():
        t = threading.Thread(target=lambda: c.extend(2, seqs=[2, 3], counts=[1, 1], stream=7))
        t.start()
        t.join()

    mem.hooks[when] = other
    held = len(mem.live)
    c.extend(2, seqs=[0, 1], counts=[1, 1], stream=5)
    assert mem.wrong == [] and len(mem.live) == held


def test_lists_of_a_call_that_fails_go_when_the_stream_is_done(monkeypatch):
    from cactus_amd.kv4 import KV4Cache
    mem = Memory(monkeypatch)
    c = KV4Cache(1, 1, 64, 16, 8, 4, 4)
    c.workspace(8192, 5)
    held = len(mem.live)
    with pytest.raises(RuntimeError):
        c.fork([0, 1], [2, 3], stream=5)
    gc.collect()                               # the exception's frames
    assert mem.wrong == [] and len(mem.live) == held and not mem.queued[5]


def test_pairs_of_different_lengths_are_refused(monkeypatch):
    from cactus_amd.kv4 import KV4Cache
    mem = Memory(monkeypatch)
    c = KV4Cache(1, 1, 64, 16, 8, 4, 4)
    held = set(mem.live)
    for call in (c.fork, c.copy_pages):
        for src, dst in (([0], [1, 2]), ([0, 1], [2])):
            with pytest.raises(ValueError):
                call(src, dst)
    gc.collect()
    assert mem.live == held and mem.queued == {}
