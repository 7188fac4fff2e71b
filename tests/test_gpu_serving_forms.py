"""The forms that the rotated append and the adapters take: sizes that the rules of their
dispatch send to each, against the plain restatements."""
import ctypes
import re
from pathlib import Path

import numpy as np
import pytest

import _serving as S
from test_gpu_serving_ops import Rope, Step, adapters, check_lora, dev, f16, run_lora

pytestmark = pytest.mark.gpu

EPS = float(np.float32(1e-6))       # what the kernels are given of it
CSRC = Path(__file__).resolve().parent.parent / "cactus_amd" / "csrc"


def rule(source, name):
    """A constant of a kernel's dispatch: the sizes below are held against it, so that they keep reaching
    what they are meant for."""
    return int(re.search(rf"\b{name} = (\d+)", (CSRC / source).read_text()).group(1))


# ------------------------------------------------------------------ rotated append
def tiled(B, n):
    return n >= rule("kv4_rope.hip", "ROPE_TILE_SEQ") and B * n >= rule("kv4_rope.hip", "ROPE_TILE_ROWS")


def waves(B, n, Hq, H, d):
    return B * -(-n // 16) * (d // 64 * (Hq + H) + H)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [65, 80])
def test_tiles_with_queries_in_place(hip_ready, d, n):
    rng = np.random.default_rng(d)
    c = Rope(hip_ready, 1, 2, d, 16, 40, 3, 8)
    assert tiled(2, n)
    c.extend([0, 2], [n, n - 1])
    c.append([0, 2], [n, n - 1], *c.rows(rng, 2, n, 4), *c.norms(rng), EPS, in_place=True)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("Hq,H", [(0, 1), (0, 3), (1, 1), (5, 1), (12, 3), (8, 8)])
def test_tiles_of_few_and_odd_heads(hip_ready, Hq, H, d):
    rng = np.random.default_rng(Hq + H + d)
    n = 45
    c = Rope(hip_ready, 1, H, d, 16, 40, 3, 8)
    assert tiled(3, n)
    c.extend([0, 1, 2], [5, 0, 20])
    c.extend([0, 1, 2], [n, n, n])
    c.append([0, 1, 2], [n] * 3, *c.rows(rng, 3, n, Hq), *c.norms(rng), EPS)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q_normed", [True, False])
def test_tiles_with_one_norm_of_two(hip_ready, q_normed, d):
    rng = np.random.default_rng(3)
    n = 130
    c = Rope(hip_ready, 1, 2, d, 16, 40, 3, 12)
    assert tiled(1, n)
    c.extend([0], [n])
    w = next(c.norms(rng))
    c.append([0], [n], *c.rows(rng, 1, n, 4), w if q_normed else None, None if q_normed else w, eps=2.0 ** -7)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_tiles_of_requests_that_write_nothing(hip_ready, d):
    rng = np.random.default_rng(d)
    n = 66
    c = Rope(hip_ready, 1, 2, d, 16, 60, 6, 12)
    assert tiled(2, n)
    c.extend([0, 1, 3], [n - 2, 70, 33])              # slots 0 and 3 have fewer tokens than rows
    c.append([0, -1, 6, 1, 1 << 30], [n] * 5, *c.rows(rng, 5, n, 2))
    c.append([3, 1], [n, 0], *c.rows(rng, 2, n, 2))
    # a page that the table does not name: the query is rotated all the same
    c.cpu.table[3, 1] = -1
    c.gpu._buf["table"].upload(c.cpu.table)
    c.append([3, 1], [33, n], *c.rows(rng, 2, n, 2), *c.norms(rng), EPS)
    c.gpu.extend(1, seqs=[99], counts=[1])
    c.append([1, 0], [n, 1], *c.rows(rng, 2, n, 2), write=False)
    assert c.gpu.status() == 2


def extremes(rng, d, q, k, v):
    for x in (q, k, v):
        x[0, 0, 0], x[0, 1, 0] = 0, 65504
        x[0, 0, 1] = np.float16(2.0 ** -24) * rng.integers(-9, 10, d)
        x[0, 0, 2, 7], x[0, 1, 3, d - 1], x[1, 2, 4, 3] = np.nan, np.inf, -np.inf
        x[1, 0, 5] *= np.float16(2.0 ** -12)
        x[1, 1, 6] = np.where(np.arange(d) % 32 == 5, 60000, 1)
        x[1, 1, 7] = (np.arange(d) % 14 - 6.5)
        x[1, 1, 7, ::32] = 7
        x[1, 40:44, 2] *= np.float16(2.0 ** -18)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("normed", [False, True])
def test_tiles_of_extreme_values(hip_ready, d, normed):
    rng = np.random.default_rng(d)
    n = 70
    c = Rope(hip_ready, 1, 8, d, 16, 40, 3, 8)
    assert tiled(2, n)
    c.extend([0, 1], [n + 5, n])
    q, k, v = c.rows(rng, 2, n, 8)
    extremes(rng, d, q, k, v)
    c.append([0, 1], [n, n], q, k, v, *(c.norms(rng) if normed else (None, None)), EPS)


def test_tiles_at_far_positions(hip_ready):
    rng = np.random.default_rng(2)
    c = Rope(hip_ready, 1, 1, 64, 4096, 70, 2, 40, theta=1e6)
    assert tiled(2, 70)
    c.extend([0, 1], [163840, 100000])
    c.append([0, 1], [70, 70], *c.rows(rng, 2, 70, 2), *c.norms(rng), EPS)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_and_tiles_meet(hip_ready, d):
    """On either side of both borders of the rule between a wave per row and tiles."""
    rng = np.random.default_rng(d)
    rows, seq = rule("kv4_rope.hip", "ROPE_TILE_ROWS"), rule("kv4_rope.hip", "ROPE_TILE_SEQ")
    sizes = [(-(-rows // seq), seq), (-(-rows // seq) - 1, seq), (-(-rows // (seq - 1)), seq - 1), (1, rows - 1), (1, rows)]
    assert [tiled(*s) for s in sizes] == [True, False, False, False, True]
    for B, n in sizes:
        c = Rope(hip_ready, 1, 1, d, 16, 60, 24, 12)
        c.extend(list(range(B)), rng.integers(0, 20, B).tolist())
        c.extend(list(range(B)), [n] * B)
        c.append(list(range(B)), [n] * B, *c.rows(rng, B, n, 2), *c.norms(rng), EPS)


@pytest.mark.parametrize("d,B,n", [(64, 8, 257), (128, 5, 257), (256, 4, 176)])
@pytest.mark.parametrize("Hq,normed,in_place", [(33, True, False), (32, False, False), (33, False, True), (32, True, True)])
def test_waves_of_two_heads(hip_ready, d, B, n, Hq, normed, in_place):
    """Ragged prompts of so many waves that each takes two heads: with 33 query heads one takes the last of them and
    the first key head, with 32 the last wave has one key head; of 15 KV heads the last wave has one's values."""
    rng = np.random.default_rng(d + Hq)
    H = 15
    assert tiled(B, n) and waves(B, n, Hq, H, d) >= rule("kv4_rope.hip", "ROPE_TWO_HEADS")
    c = Rope(hip_ready, 1, H, d, 16, 200, B, 20)
    counts = [n, n - 1, n // 2 + 3, n - 16, 1, n, 0, n // 3][:B]
    c.extend(list(range(B)), [3, 0, 16, 31, 15, 7, 1, 40][:B])
    c.extend(list(range(B)), counts)
    q, k, v = c.rows(rng, B, n, Hq)
    extremes(rng, d, q, k, v)
    c.append(list(range(B)), counts, q, k, v, *(c.norms(rng) if normed else (None, None)), EPS, pad=0 if in_place else 16, in_place=in_place)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_two_heads_of_keys_alone(hip_ready, d):
    rng = np.random.default_rng(d)
    B, H = 8, 15
    n = {64: 560, 128: 370, 256: 225}[d]
    assert tiled(B, n) and waves(B, n, 0, H, d) >= rule("kv4_rope.hip", "ROPE_TWO_HEADS")
    c = Rope(hip_ready, 1, H, d, 64, 90, B, 10)
    c.extend(list(range(B)), [n] * B)
    c.append(list(range(B)), [n] * B, *c.rows(rng, B, n, 0), None, next(c.norms(rng)), EPS)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("normed", [False, True])
def test_single_rows_queries_are_rounded_once(hip_ready, d, normed):
    """Where a wave has one row, queries are computed in 64 bits: the FP16 value next to the formula's, but where that
    lies so close to the middle of two that 64 bits cannot tell.

    Of |a cos| + |b sin|, the sum of d squares (d / 64 + 6 roundings, half of them in the root), its
    root, and four products and a sum err by less than 32 of 2^-53: 2^-48."""
    rng = np.random.default_rng(d)
    B, n, Hq = 20, 6, 16
    assert not tiled(B, n)
    c = Rope(hip_ready, 1, 1, d, 16, 200, B, 8)
    lens = rng.integers(n, 100, B).tolist()
    c.extend(list(range(B)), lens)
    q, k, v = c.rows(rng, B, n, Hq)
    q_norm, k_norm = c.norms(rng) if normed else (None, None)
    b = [dev(hip_ready, a) for a in (q, k, v)] + [hip_ready.DeviceBuffer(q.nbytes)]
    w = [None if a is None else dev(hip_ready, a) for a in (q_norm, k_norm)]
    c.gpu.append_rope(0, b[0].ptr, b[3].ptr, Hq, b[1].ptr, b[2].ptr, B, n, c.dtable.ptr, len(c.table), None, None,
                      *(a and a.ptr for a in w), EPS)
    got = b[3].to_numpy(np.float16, q.shape)
    for i in range(B):
        for r in range(n):
            y, err = S.rotated(q[i, r], q_norm, EPS, c.table[lens[i] - n + r])
            e = err / ((d / 2 + 12) * S.E32) * 2.0 ** -48
            assert ((y - e).astype(np.float16) <= got[i, r]).all() and (got[i, r] <= (y + e).astype(np.float16)).all()


# ------------------------------------------------------------------ adapters
def tiles32(b, n):
    return n > 16 and b * -(-n // 32) >= rule("lora.hip", "LORA_TILE2")


def requests(rng, b, n):
    """Ragged rows, some requests without any or with more than there are; adapters 0 to 3, a third of them none."""
    counts = rng.integers(1, n + 1, b)
    counts[[1, 4, 7]] = 0, n + 9, -2
    ids = rng.integers(-2, 4, b)
    ids[:3] = 3, 0, -1
    return counts.tolist(), ids.tolist()


@pytest.mark.parametrize("r", [8, 16, 24, 32, 40, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("in_place", [False, True])
def test_lora_prompts_in_tiles_of_32_rows(hip_ready, r, in_place):
    """Several steps of K per wave and more than one round of outputs per workgroup, both with a remainder."""
    rng = np.random.default_rng(r)
    b, n, K, N = 33, 50, 1160, 1544
    assert tiles32(b, n)
    A, B, s = adapters(rng, 4, r, K, N)
    x, base = f16(rng, b, n, K), f16(rng, b, n, N)
    counts, ids = requests(rng, b, n)
    for i, m in enumerate(counts):
        x[i, max(m, 0):] = np.nan            # not read: no row that is there is touched by them
    got = run_lora(hip_ready, x, A, B, s, ids, counts, base, (8, 16, 24), in_place)
    check_lora(got, x, A, B, s, ids, counts, base, in_place)


@pytest.mark.parametrize("r", [8, 16, 48, 64, 128, 200])
def test_lora_more_tiles_than_workgroups_at_a_time(hip_ready, r):
    """Every workgroup takes all outputs of its rows."""
    rng = np.random.default_rng(r)
    b, n, K, N = 90, 70, 72, 1032
    assert tiles32(b, n) and b * -(-n // 32) > rule("lora.hip", "LORA_WGS")
    A, B, s = adapters(rng, 4, r, K, N)
    x, base = f16(rng, b, n, K), f16(rng, b, n, N)
    counts, ids = requests(rng, b, n)
    check_lora(run_lora(hip_ready, x, A, B, s, ids, counts, base), x, A, B, s, ids, counts, base)


@pytest.mark.parametrize("r", [16, 32, 64, 128, 256])
def test_lora_32_row_tiles_keep_nan_and_infinity_in_their_rows(hip_ready, r):
    rng = np.random.default_rng(r)
    b, n, K, N = 32, 50, 136, 200
    assert tiles32(b, n)
    A, B, s = adapters(rng, 2, r, K, N)
    x, base = f16(rng, b, n, K), f16(rng, b, n, N)
    ids = [i % 2 for i in range(b)]
    clean = run_lora(hip_ready, x, A, B, s, ids, None, base)
    check_lora(clean, x, A, B, s, ids, None, base)
    for bad in (np.nan, np.inf, -np.inf):
        y = x.copy()
        y[0, 17, 5], y[5, 31, 135], y[31, 49, 0] = bad, bad, bad
        got = run_lora(hip_ready, y, A, B, s, ids, None, base)
        for i, j in ((0, 17), (5, 31), (31, 49)):
            assert not np.isfinite(got[i, j]).any()
            got[i, j] = clean[i, j]
        np.testing.assert_array_equal(got, clean)


@pytest.mark.parametrize("r", [8, 64])
def test_lora_32_row_tiles_ranges(hip_ready, r):
    """The ranks' values pass FP16's range on both sides."""
    rng = np.random.default_rng(r)
    b, n, K, N = 32, 40, 264, 72
    assert tiles32(b, n)
    for ax, aa, ab, s in ((2.0 ** -14, 2.0 ** -14, 1.0, 1.0), (200.0, 200.0, 2.0 ** -12, 2.0 ** -8), (3000.0, 3000.0, 2.0 ** -24, 2.0 ** -10),
                          (0.0, 1.0, 1.0, 1.0)):
        A, B = f16(rng, 2, r, K, scale=aa), f16(rng, 2, N, r, scale=ab)
        x, base = f16(rng, b, n, K, scale=ax), f16(rng, b, n, N, scale=1e-3)
        sc, ids = np.array([s, -s], np.float32), [i % 2 for i in range(b)]
        check_lora(run_lora(hip_ready, x, A, B, sc, ids, None, base), x, A, B, sc, ids, None, base)


def test_lora_tiles_of_16_and_32_rows_meet(hip_ready):
    rng = np.random.default_rng(1)
    K, N, most = 104, 136, rule("lora.hip", "LORA_TILE2")
    A, B, s = adapters(rng, 4, 32, K, N)
    sizes = [(most - 1, 17), (most, 17), (most, 16), (most // 2, 33), (most // 2 - 1, 64), (1, 32 * most), (1, 32 * (most - 1))]
    assert [tiles32(*z) for z in sizes] == [False, True, False, True, False, True, False]
    for b, n in sizes:
        x, base, ids = f16(rng, b, n, K), f16(rng, b, n, N), rng.integers(-1, 4, b).tolist()
        check_lora(run_lora(hip_ready, x, A, B, s, ids, None, base), x, A, B, s, ids, None, base)


@pytest.mark.parametrize("r,N", [(8, 16392), (16, 8200), (24, 8200), (64, 4104), (128, 4104), (256, 4104)])
@pytest.mark.parametrize("in_place", [False, True])
def test_lora_single_rows_in_several_rounds(hip_ready, r, N, in_place):
    """So many requests that a workgroup's waves take outputs more than once, with a remainder."""
    rng = np.random.default_rng(r)
    b, K = 130, 1544
    pieces = 1 << (r // 8 - 1).bit_length()
    assert -(-N // (512 // pieces)) > 8 * -(-rule("lora.hip", "LORA_WGS") // b), "one round"
    A, B, s = adapters(rng, 5, r, K, N)
    x, base = f16(rng, b, 1, K), f16(rng, b, 1, N)
    ids = rng.integers(-1, 6, b).tolist()
    counts = rng.integers(-1, 3, b).tolist()
    got = run_lora(hip_ready, x, A, B, s, ids, counts, base, (8, 16, 24), in_place)
    check_lora(got, x, A, B, s, ids, counts, base, in_place)


# ------------------------------------------------------------------ a step of prompts
def test_captured_prompts(hip_ready):
    """Prompts as a graph, replayed while the sequences grow, an eager step on another stream at the same time:
    both have what they have alone."""
    cm, B, n = hip_ready, 33, 40
    a, e = (Step(cm, B, np.random.default_rng(16)) for _ in range(2))
    assert tiled(B, n) and tiles32(B, n)
    rng = np.random.default_rng(17)
    st = cm.Stream()
    ba, be = a.buffers(n), e.buffers(n)

    def rows(counts):
        x = f16(rng, B, n, a.HID)
        for b in (ba, be):
            b["x"].upload(x)
            b["counts"].upload(np.int32(counts))
            for k in ("qkv", "q", "o"):
                b[k].upload(np.zeros(b[k].nbytes // 2, np.float16))
    rows([n] * B)
    for s, b in ((a, ba), (e, be)):            # once before the capture, so that scratch memory is there
        s.run(b, n, st.handle)
        st.sync()
    graph = ctypes.c_void_p()
    cm.call("cactus_hip_graph_capture_begin", st.handle)
    a.run(ba, n, st.handle)
    cm.call("cactus_hip_graph_capture_end", st.handle, ctypes.byref(graph))
    for i in range(3):
        rows(rng.integers(0, n + 1, B))
        cm.call("cactus_hip_graph_launch", graph, st.handle)
        e.run(be, n, None)
        st.sync()
        cm.call("cactus_hip_stream_sync", None)
        assert a.cache.status(st.handle) == 0 and e.cache.status() == 0
        for k in ("qkv", "q", "o"):
            size = ba[k].nbytes // 2
            np.testing.assert_array_equal(ba[k].to_numpy(np.uint16, size), be[k].to_numpy(np.uint16, size), err_msg=f"replay {i}: {k}")
        for name, v in a.cache.tables().items():
            np.testing.assert_array_equal(v, e.cache.tables()[name])
        size = a.cache._buf["pages"].nbytes
        np.testing.assert_array_equal(a.cache._buf["pages"].to_numpy(np.uint8, size), e.cache._buf["pages"].to_numpy(np.uint8, size))
    cm.call("cactus_hip_graph_destroy", graph)
