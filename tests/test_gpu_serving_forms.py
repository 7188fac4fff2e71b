"""The forms that the rotated append takes: sizes that the rules of its dispatch send to
each, against the plain restatements."""
import re
from pathlib import Path

import numpy as np
import pytest

import _serving as S
from test_gpu_serving_ops import Rope, dev

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
