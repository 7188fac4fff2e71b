"""Rotated appends, adapters per request and rules on logits without a GPU:
refusals before any launch, sizes, the Python owners' checks, and the restatements."""
import ctypes

import numpy as np
import pytest

import _serving as S


@pytest.fixture(scope="module")
def lib():
    import cactus_amd
    return cactus_amd.hip()


def refused(lib, rc, text):
    assert rc == -1
    assert text in lib.cactus_hip_last_error(), lib.cactus_hip_last_error()


# ------------------------------------------------------------------ rotated append
def cache(**kw):
    from cactus_amd.kv4 import CacheDesc
    shape = dict(layers=2, kv_heads=2, head_dim=128, page_size=64, num_pages=8, max_seqs=4, max_pages=4)
    ptrs = dict(pages=1 << 20, table=1 << 21, lens=1 << 22, refs=1 << 23, state=1 << 24)   # never dereferenced
    return CacheDesc(**{**shape, **ptrs, **kw})


def append(lib, desc=None, layer=0, **kw):
    a = dict(seqs=None, counts=None, q=4096, q_stride=512, q_out=8192, heads=4, k=4096, v=4096, kv_stride=256, q_norm=None,
             k_norm=None, eps=1e-6, table=4096, positions=256, batch=2, seq_len=3)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.cactus_hip_kv4_append_rope_f16((desc or cache()).ref, layer, *a.values(), None)


@pytest.mark.parametrize("kw,text", [
    (dict(k=None), b"null pointer"), (dict(v=None), b"null pointer"), (dict(q=None), b"null pointer"),
    (dict(q_out=None), b"null pointer"), (dict(table=None), b"null pointer"), (dict(q=4104), b"aligned"),
    (dict(q_out=4100), b"aligned"), (dict(k=4098), b"aligned"), (dict(v=4104), b"aligned"), (dict(kv_stride=260), b"aligned"),
    (dict(q_stride=516), b"aligned"), (dict(q_norm=8), b"aligned"), (dict(k_norm=4100), b"aligned"), (dict(table=4104), b"aligned"),
    (dict(kv_stride=248), b"kv_stride"), (dict(q_stride=504), b"q_stride"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"), (dict(positions=255), b"table_positions"),
    (dict(batch=5), b"slots"), (dict(seq_len=1 << 28), b"seq_len"), (dict(heads=16385), b"num_q_heads"),
    (dict(q=4096, q_out=4096, q_stride=520), b"in place")])
def test_append_refusals(lib, kw, text):
    refused(lib, append(lib, **kw), text)


def test_append_checks_the_cache_and_the_layer(lib):
    refused(lib, append(lib, cache(head_dim=96)), b"head_dim")
    refused(lib, append(lib, cache(lens=None)), b"null buffer")
    refused(lib, append(lib, layer=2), b"layer")
    assert append(lib, batch=0) == 0 and append(lib, seq_len=0) == 0


def test_rope_table_refusals(lib):
    for kw, text in (((4096, 10, 63, 1e4), b"head_dim"), ((4096, 10, 0, 1e4), b"head_dim"), ((4096, 10, 64, 0.0), b"theta"),
                     ((4096, 10, 64, float("nan")), b"theta"), ((4096, 1 << 31, 64, 1e4), b"positions"),
                     ((None, 10, 64, 1e4), b"null")):
        refused(lib, lib.cactus_hip_rope_table_f32(*kw, None), text)
    assert lib.cactus_hip_rope_table_f32(None, 0, 64, 1e4, None) == 0


def test_rotation_restated():
    """A rotation keeps lengths, position 0 changes nothing, and scores depend on distances alone."""
    rng = np.random.default_rng(1)
    t = S.rope_table(50, 64, 1e4)
    q, k = rng.standard_normal((2, 64))
    y, _ = S.rotated(q, None, 0, t[0])
    assert np.array_equal(y, q)
    at = lambda x, p: S.rotated(x, None, 0, t[p])[0]  # noqa: E731
    assert np.allclose(at(q, 17) @ at(k, 5), at(q, 40) @ at(k, 28), atol=64 * 2.0 ** -22 * np.abs(q).max() * np.abs(k).max())


def test_cache_owner_waits_for_what_it_sets_up(monkeypatch):
    """Tables and rotations that the owner makes are there when it returns them: other streams' calls are not ordered
    behind the kernels that fill them."""
    from cactus_amd import kv4
    sent = []

    class Buffer:
        def __init__(self, n):
            self.nbytes, self.ptr = n, 1 << 20
    monkeypatch.setattr(kv4, "DeviceBuffer", Buffer)
    monkeypatch.setattr(kv4, "call", lambda name, *a: sent.append((name, a)))
    waits = ("cactus_hip_stream_sync", "cactus_hip_kv4_status")      # (the status waits for the stream)
    for stream in (None, 77):
        sent.clear()
        c = kv4.KV4Cache(1, 1, 64, 16, 8, 4, 4, stream)
        names = [n for n, a in sent if a[-1] == stream]
        assert "cactus_hip_kv4_reset" in names and names[-1] in waits
        sent.clear()
        c.rope_table(1e4, stream)
        names = [n for n, a in sent if a[-1] == stream]
        assert "cactus_hip_rope_table_f32" in names and names[-1] in waits


# ------------------------------------------------------------------ adapters
def lora(lib, **kw):
    a = dict(x=4096, x_stride=64, A=4096, B=4096, scales=None, n=3, rank=16, ids=4096, counts=None, base=4096, base_stride=128,
             y=8192, y_stride=128, batch=2, seq_len=3, K=64, N=128)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.cactus_hip_lora_add_f16(*a.values(), None)


@pytest.mark.parametrize("kw,text", [
    (dict(rank=0), b"rank"), (dict(rank=12), b"rank"), (dict(rank=264), b"rank"), (dict(K=60, x_stride=60), b"multiples of 8"),
    (dict(N=100), b"multiples of 8"), (dict(K=1 << 24, x_stride=1 << 24), b"2^24"), (dict(x=None), b"null pointer"),
    (dict(A=None), b"null pointer"), (dict(B=None), b"null pointer"), (dict(ids=None), b"null pointer"),
    (dict(base=None), b"null pointer"), (dict(y=None), b"null pointer"), (dict(x=4098), b"aligned"), (dict(A=4104), b"aligned"),
    (dict(B=4104), b"aligned"), (dict(base=4104), b"aligned"), (dict(y=4104), b"aligned"), (dict(x_stride=68), b"aligned"),
    (dict(x_stride=56), b"stride"), (dict(base_stride=120), b"stride"), (dict(y_stride=120), b"stride"),
    (dict(y=4096, y_stride=136), b"in place"), (dict(batch=65536), b"batch"), (dict(seq_len=1 << 24), b"seq_len"),
    (dict(n=1 << 24), b"num_adapters"), (dict(batch=65535, seq_len=1 << 20), b"batch times seq_len")])
def test_lora_refusals(lib, kw, text):
    refused(lib, lora(lib, **kw), text)


@pytest.mark.parametrize("S", [1, 3, 100])
def test_lora_without_inputs_needs_its_second_weights(lib, S):
    """K 0: A and x may be missing, but the outputs' product still reads B."""
    refused(lib, lora(lib, K=0, x_stride=0, x=None, A=None, B=None, seq_len=S), b"null pointer")


@pytest.mark.parametrize("S", [1, 3, 100])
@pytest.mark.parametrize("base", [4096, 16384])
def test_lora_refuses_outputs_in_place_of_x(lib, S, base):
    """Workgroups that share a row read all of x: one would overwrite what another still reads."""
    refused(lib, lora(lib, K=64, N=64, x=4096, y=4096, base=base, x_stride=64, base_stride=64, y_stride=64, seq_len=S), b"place of x")


def test_lora_without_rows_does_nothing(lib):
    assert lora(lib, batch=0) == 0 and lora(lib, seq_len=0) == 0 and lora(lib, N=0) == 0


# ------------------------------------------------------------------ rules on logits
def call_rules(lib, half=True, change=(), **kw):
    from cactus_amd.logits import RulesDesc
    r = dict(history=4096, history_lens=4096, repetition=4096, frequency=4096, presence=4096, bias_tokens=4096, bias_values=4096,
             bias_counts=4096, masks=4096, mask_ids=4096, history_stride=10, bias_stride=5, num_masks=2, mask_stride=4, max_seqs=6)
    r.update(change)
    a = dict(seqs=None, logits=4096, stride=100, out=8192, out_stride=100, best=4096, batch=3, vocab=100, work=4096, size=48)
    assert set(kw) <= set(a)
    a.update(kw)
    return (lib.cactus_hip_logits_rules_f16 if half else lib.cactus_hip_logits_rules_f32)(RulesDesc(**r).ref, *a.values(), None)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("change,kw,text", [
    (dict(max_seqs=0), {}, b"max_seqs"), (dict(history_stride=1 << 20), {}, b"history_stride"),
    (dict(bias_stride=1025), {}, b"bias_stride"), (dict(bias_values=None), {}, b"without values"),
    (dict(mask_stride=3), {}, b"mask_stride"), (dict(mask_ids=None, num_masks=5), {}, b"mask"), ({}, dict(batch=65536, size=1 << 21), b"65535"),
    ({}, dict(vocab=1 << 28, stride=1 << 28, out_stride=1 << 28), b"mask_stride"), ({}, dict(logits=None), b"null pointer"),
    ({}, dict(out=None), b"null pointer"), ({}, dict(stride=99), b"stride"), ({}, dict(out_stride=99), b"stride"),
    ({}, dict(out=8194), b"misaligned"), ({}, dict(logits=4097), b"misaligned"), ({}, dict(work=None), b"workspace"),
    ({}, dict(work=4104), b"workspace"), ({}, dict(size=47), b"workspace"), ({}, dict(out=4096, stride=104), b"in place")])
def test_rules_refusals(lib, half, change, kw, text):
    refused(lib, call_rules(lib, half, change, **kw), text)


def test_rules_more_refusals(lib):
    refused(lib, call_rules(lib, True, dict(masks=None), vocab=1 << 28, stride=1 << 28, out_stride=1 << 28), b"vocab")
    refused(lib, call_rules(lib, True, out=4096), b"in place")        # FP16 rows cannot become FP32 where they are
    refused(lib, lib.cactus_hip_logits_rules_f16(None, None, 4096, 1, 4096, 1, None, 1, 1, None, 0, None), b"null rules")
    assert call_rules(lib, batch=0) == 0 and call_rules(lib, vocab=0) == 0
    assert lib.cactus_hip_logits_rules_workspace(3) == 48


def test_rules_owner_checks(monkeypatch):
    from cactus_amd import logits as L
    sent = []

    class Buffer:
        def __init__(self, n):
            self.nbytes, self.ptr = n, 1 << 20

        @classmethod
        def from_numpy(cls, a, stream=None):
            return cls(a.nbytes)
    monkeypatch.setattr(L, "DeviceBuffer", Buffer)
    monkeypatch.setattr(L, "call", lambda name, *a: sent.append((name, *a)))
    r = L.LogitsRules(4, 50, max_history=8, max_bias=2, num_masks=1)
    r.set_history(3, [1, 2, 3])
    assert sent[0][1] == (1 << 20) + 4 * 3 * 8 and sent[0][3] == 12
    for bad in (lambda: r.set_history(4, [1]), lambda: r.set_mask(1, [True] * 50), lambda: r.use_mask(-1, 0)):
        with pytest.raises(IndexError):
            bad()
    for bad in (lambda: r.set_history(0, range(9)), lambda: r.set_bias(0, [1, 2, 3], [0, 0, 0]), lambda: r.set_bias(0, [1], []),
                lambda: r.set_mask(0, [True] * 49), lambda: L.LogitsRules(1, 50, max_bias=1025),
                lambda: L.LogitsRules(1, 50).set_history(0, [1])):
        with pytest.raises(ValueError):
            bad()


def test_rules_owner_keeps_scratch_memory_once_it_is_zero(monkeypatch):
    """A workspace is kept for later calls only behind its fill: not where that fails, and not for another
    thread's call in between."""
    from cactus_amd import logits as L

    class Buffer:
        made = 0

        def __init__(self, n):
            Buffer.made += 1
            self.nbytes, self.ptr = n, Buffer.made << 20
    monkeypatch.setattr(L, "DeviceBuffer", Buffer)
    monkeypatch.setattr(L, "hip", lambda: type("Lib", (), {"cactus_hip_logits_rules_workspace": staticmethod(lambda n: 16 * n)}))
    filled, used, during = set(), [], []

    def call(name, *a):
        if name == "cactus_hip_memset":
            if during:
                during.pop()()
            filled.add(a[0])
        else:
            used.append(a[-3])
            assert used[-1] in filled, "scratch memory that is not zero"
    monkeypatch.setattr(L, "call", call)

    def fail():
        raise RuntimeError("refused")
    r = L.LogitsRules(4, 50)
    during.append(fail)
    with pytest.raises(RuntimeError):
        r.apply(4096, 8192, 4, 4096)
    r.apply(4096, 8192, 4, 4096)
    during.append(lambda: r.apply(4096, 8192, 8, 4096, stream=5))
    r.apply(4096, 8192, 8, 4096, stream=5)
    r.apply(4096, 8192, 2, 4096, stream=5)
    assert len(used) == 4


def test_rules_owner_takes_integers(monkeypatch):
    from cactus_amd import logits as L

    class Buffer:
        def __init__(self, n):
            self.nbytes, self.ptr = n, 1 << 20

        @classmethod
        def from_numpy(cls, a, stream=None):
            return cls(a.nbytes)
    monkeypatch.setattr(L, "DeviceBuffer", Buffer)
    monkeypatch.setattr(L, "call", lambda name, *a: None)
    r = L.LogitsRules(4, 50, max_history=8, max_bias=2)
    for bad in ([1.5], np.array([1 << 32]), [1 << 31], [True]):
        with pytest.raises(TypeError):
            r.set_history(0, bad)
        with pytest.raises(TypeError):
            r.set_bias(0, bad, [1.0])
    r.set_history(0, [])
    r.set_history(0, np.arange(8, dtype=np.uint8))


def test_rules_owner_changes_a_setting_whole_or_not_at_all(monkeypatch):
    """Every part of a setting is checked before the first is uploaded."""
    from cactus_amd import logits as L
    sent = []

    class Buffer:
        def __init__(self, n):
            self.nbytes, self.ptr = n, 1 << 20

        @classmethod
        def from_numpy(cls, a, stream=None):
            return cls(a.nbytes)
    monkeypatch.setattr(L, "DeviceBuffer", Buffer)
    monkeypatch.setattr(L, "call", lambda name, *a: sent.append((name, *a)))
    r = L.LogitsRules(4, 50, max_history=8, max_bias=6, num_masks=1)
    for bad in (lambda: r.set_bias(0, [1, 2], ["a", "b"]), lambda: r.set_bias(0, [1], [None]), lambda: r.set_bias(0, [[1, 2, 3]], [1.0]),
                lambda: r.set_bias(0, [1, 2], [[1.0, 2.0], [3.0, 4.0]]), lambda: r.set_bias(0, [1, 2, 3], np.float32(1)),
                lambda: r.set_history(0, ["a"]), lambda: r.set_penalties(0, 1.1, 0.5, "none"),
                lambda: r.set_penalties(0, 1.1, None), lambda: r.set_penalties(0, [1.0, 2.0]), lambda: r.use_mask(0, [0, 0])):
        with pytest.raises((TypeError, ValueError)):
            bad()
        assert sent == []
    r.set_bias(1, np.array([3, 4]), (0.5, -1))
    assert [c[3] for c in sent] == [8, 8, 4]
    sent.clear()
    r.set_penalties(1, 2, np.float64(0.5))
    r.set_bias(1, [], [])
    r.set_history(1, [[1, 2, 3]])
    assert [c[3] for c in sent] == [4] * 4 + [12, 4]
    L.LogitsRules(0, 50, max_history=8, max_bias=6, num_masks=0)


def test_lora_owner_checks(monkeypatch):
    from cactus_amd import lora as L
    sent = []

    class Buffer:
        def __init__(self, n):
            self.nbytes, self.ptr = n, 1 << 20
    monkeypatch.setattr(L, "DeviceBuffer", Buffer)
    monkeypatch.setattr(L, "call", lambda name, *a: sent.append((name, *a)))
    a = L.LoraAdapters(3, 16, 32, 24)
    sent.clear()
    a.set(2, np.ones((4, 32)), np.ones((24, 4)), 0.5)
    assert [(s[1] - (1 << 20), s[3]) for s in sent] == [(2 * 16 * 32 * 2, 16 * 32 * 2), (2 * 16 * 24 * 2, 16 * 24 * 2), (8, 4)]
    with pytest.raises(IndexError):
        a.set(3, np.ones((4, 32)), np.ones((24, 4)))
    for A, B in (((17, 32), (24, 17)), ((4, 31), (24, 4)), ((4, 32), (24, 5)), ((4, 32), (23, 4)), ((32,), (24, 1))):
        with pytest.raises(ValueError):
            a.set(0, np.ones(A), np.ones(B))
    for bad in ((3, 12, 32, 24), (3, 0, 32, 24), (3, 264, 32, 24), (3, 8, 30, 24), (3, 8, 32, 20)):
        with pytest.raises(ValueError):
            L.LoraAdapters(*bad)


def test_lora_owner_waits_for_its_first_weights(monkeypatch):
    """The zeros that the adapters start with are there when the owner is: a call on another stream, the
    upload of an adapter among them, is not ordered behind a fill that is still on its way."""
    from cactus_amd import lora as L
    sent = []

    class Buffer:
        def __init__(self, n):
            self.nbytes, self.ptr = n, 1 << 20
    monkeypatch.setattr(L, "DeviceBuffer", Buffer)
    monkeypatch.setattr(L, "call", lambda name, *a: sent.append((name, a)))
    for stream in (None, 77):
        sent.clear()
        L.LoraAdapters(3, 16, 32, 24, stream)
        fills = [i for i, (name, a) in enumerate(sent) if name == "cactus_hip_memset" and a[-1] == stream]
        assert len(fills) == 3
        assert sent[-1] == ("cactus_hip_stream_sync", (stream,)) and fills[-1] < len(sent) - 1


def test_rules_restated():
    x = np.array([2.0, -2.0, 1.0, 0.0, 3.0], np.float32)
    y, best = S.rules(x, hist=[0, 1, 1, -1, 7], rep=2.0, freq=0.5, pres=0.25, bias=[(3, 4.0), (3, -1.0), (9, 1.0)])
    assert y.tolist() == [0.25, -5.25, 1.0, 3.0, 3.0] and best == 3
    y, best = S.rules(x, mask=np.array([1, 1, 0, 0, 0], bool))
    assert y.tolist() == [2.0, -2.0, -np.inf, -np.inf, -np.inf] and best == 0
    assert S.rules(x, mask=np.zeros(5, bool))[1] == 0
    assert S.rules([np.nan, -0.0, 0.0])[1] == 1
