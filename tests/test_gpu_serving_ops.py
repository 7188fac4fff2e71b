"""Rotated appends, adapters per request and rules on logits on the GPU against
their plain restatements, and a step that runs them together."""
import ctypes

import numpy as np
import pytest

import _serving as S
from _kv4 import Model, attention, quantize, values

pytestmark = pytest.mark.gpu

MARK = np.float16(-77.25)      # what rows hold that have to stay


def dev(cm, a):
    return cm.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def f16(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float16)


# ------------------------------------------------------------------ rotated append
class Rope:
    """A KV4Cache, its model and a table; fresh pages hold 0xFF bytes (NaN scales)."""

    def __init__(self, cm, layers=1, kv_heads=2, head_dim=64, page_size=16, num_pages=40, max_seqs=6, max_pages=12, theta=1e4):
        from cactus_amd.kv4 import KV4Cache
        self.cm, self.d = cm, head_dim
        shape = (layers, kv_heads, head_dim, page_size, num_pages, max_seqs, max_pages)
        self.gpu, self.cpu = KV4Cache(*shape), Model(*shape)
        self.gpu._buf["pages"].upload(self.cpu.pages)
        self.table = S.rope_table(page_size * max_pages, head_dim, theta)
        self.dtable = dev(cm, self.table)

    def extend(self, seqs, counts):
        assert self.cpu.extend(seqs, counts) == 0
        self.gpu.extend(len(seqs), seqs=seqs, counts=counts)
        assert self.gpu.status() == 0

    def append(self, seqs, counts, q, k, v, q_norm=None, k_norm=None, eps=1e-6, layer=0, pad=0, in_place=False, write=True):
        """q [B][S][Hq][d], k, v [B][S][H][d] side by side in rows with `pad` more values; checks q_out, pages and tables."""
        cm, d = self.cm, self.d
        B, n, Hq = q.shape[:3]
        H = k.shape[2]
        rows = np.full((B * n, (Hq + 2 * H) * d + pad), np.float16(np.nan))
        rows[:, :(Hq + 2 * H) * d] = np.concatenate((q, k, v), 2).reshape(B * n, -1)
        buf, q_out = dev(cm, rows), dev(cm, np.full((B, n, Hq, d), MARK))
        if in_place:
            q_out = dev(cm, q)
        dn = [None if w is None else dev(cm, w) for w in (q_norm, k_norm)]
        stride, pn = rows.shape[1], [None if w is None else w.ptr for w in dn]
        self.gpu.append_rope(layer, (q_out.ptr if in_place else buf.ptr) if Hq else None, q_out.ptr if Hq else None, Hq,
                             buf.ptr + 2 * Hq * d, buf.ptr + 2 * (Hq + H) * d, B, n, self.dtable.ptr, len(self.table),
                             None if in_place else stride, stride, *pn, eps, list(seqs), list(counts))
        got = q_out.to_numpy(np.float16, (B, n, Hq, d)) if Hq else np.zeros((B, n, 0, d), np.float16)
        want = q.copy() if in_place else np.full(q.shape, MARK)
        for b, (s, m) in enumerate(zip(seqs, counts)):
            there = 0 <= s < self.cpu.max_seqs and write
            for r in range(n):
                pos = int(self.cpu.lens[s]) - m + r if there else -1
                if r >= m or pos < 0:
                    np.testing.assert_array_equal(got[b, r].view(np.uint16), want[b, r].view(np.uint16), err_msg=f"row {b} {r} stays")
                    continue
                y, err = S.rotated(q[b, r], q_norm, eps, self.table[pos])
                fine = np.isfinite(y) & (np.abs(y) < 65504)
                with np.errstate(over="ignore"):
                    np.testing.assert_array_equal(got[b, r][~fine], y[~fine].astype(np.float16))
                off = np.abs(got[b, r][fine].astype(np.float64) - y[fine]) - (S.half_step(y) + err)[fine]
                assert (off <= 0).all(), f"query {b} {r}: {off.max()} over the bound"
                with np.errstate(over="ignore"):
                    key = S.rotated(k[b, r], k_norm, eps, self.table[pos])[0].astype(np.float16)
                if self.cpu.table[s, pos // self.cpu.ps] >= 0:
                    self.cpu.write(layer, s, pos, key, v[b, r])
        self.check()

    def check(self):
        t = self.gpu.tables()
        for name in ("table", "lens", "refs"):
            np.testing.assert_array_equal(t[name], getattr(self.cpu, name), err_msg=name)
        np.testing.assert_array_equal(self.gpu._buf["pages"].to_numpy(np.uint8, self.cpu.pages.shape), self.cpu.pages)

    def rows(self, rng, B, n, Hq, scale=1.0):
        H = self.cpu.H
        return f16(rng, B, n, Hq, self.d, scale=scale), f16(rng, B, n, H, self.d, scale=scale), f16(rng, B, n, H, self.d, scale=scale)

    def norms(self, rng):
        return ((1 + 0.3 * rng.standard_normal(self.d)).astype(np.float16) for _ in range(2))


def test_rope_table(hip_ready):
    for d, theta, n in ((64, 1e4, 1000), (128, 1e6, 40000), (256, 5e5, 77), (6, 3.5, 10)):
        buf = hip_ready.DeviceBuffer(4 * n * d)
        hip_ready.call("cactus_hip_rope_table_f32", buf.ptr, n, d, theta, None)
        got = buf.to_numpy(np.float32, (n, 2, d // 2))
        theta = float(np.float32(theta))
        want = S.rope_table(n, d, theta).astype(np.float64)
        # half a step of FP32, and the angle p f's own rounding in 64 bits (a few 2^-52 of at most n)
        assert (np.abs(got - want) <= 2.0 ** -24 * np.abs(want) * 2 + 2.0 ** -48 * n).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("ps,n,lens", [(16, 1, [0, 15, 16, 17]), (16, 37, [0, 3, 29, 0]), (64, 70, [0, 63, 1, 40]),
                                       (256, 5, [250, 0, 14, 12]), (32, 16, [16, 0, 32, 8]), (16, 17, [15, 16, 1, 0])])
@pytest.mark.parametrize("normed", [False, True])
def test_rows_are_rotated_and_written(hip_ready, d, ps, n, lens, normed):
    rng = np.random.default_rng(d + ps + n)
    c = Rope(hip_ready, 2, 3, d, ps, 40, 6, 12)
    c.extend([4, 0, 2, 1], lens)
    counts, seqs = [n, max(1, n // 2), 0, max(1, n - 1)], [2, 4, 0, 1]
    c.extend(seqs, counts)
    q_norm, k_norm = c.norms(rng) if normed else (None, None)
    c.append(seqs, counts, *c.rows(rng, 4, n, 6), q_norm, k_norm, layer=1, pad=8)


@pytest.mark.parametrize("Hq,H", [(0, 1), (1, 1), (5, 1), (12, 3), (8, 8)])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_head_counts(hip_ready, Hq, H, n):
    rng = np.random.default_rng(Hq + H + n)
    c = Rope(hip_ready, 1, H, 64, 16, 40, 3, 8)
    c.extend([0, 1, 2], [5, 0, 20])
    c.extend([0, 1, 2], [n, n, n])
    c.append([0, 1, 2], [n] * 3, *c.rows(rng, 3, n, Hq), *c.norms(rng))


@pytest.mark.parametrize("q_normed", [True, False])
def test_one_norm_of_two(hip_ready, q_normed):
    rng = np.random.default_rng(3)
    for n in (2, 33):
        c = Rope(hip_ready, 1, 2, 128, 16, 40, 3, 8)
        c.extend([0], [n])
        w = next(c.norms(rng))
        c.append([0], [n], *c.rows(rng, 1, n, 4), w if q_normed else None, None if q_normed else w, eps=1e-2)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [2, 40])
def test_queries_in_place(hip_ready, d, n):
    rng = np.random.default_rng(d)
    c = Rope(hip_ready, 1, 2, d, 16, 40, 3, 8)
    c.extend([0, 2], [n, n - 1])
    c.append([0, 2], [n, n - 1], *c.rows(rng, 2, n, 4), *c.norms(rng), in_place=True)


@pytest.mark.parametrize("n", [1, 6, 50])
def test_requests_that_write_nothing(hip_ready, n):
    """Slots out of range, rows without a token, pages that are not there; and a status that holds all back."""
    rng = np.random.default_rng(n)
    c = Rope(hip_ready, 1, 2, 64, 16, 60, 6, 12)
    c.extend([0, 1, 3], [max(1, n - 2), 70, 33])      # slot 0 has fewer tokens than rows
    c.append([0, -1, 6, 1, 1 << 30], [n] * 5, *c.rows(rng, 5, n, 2))
    # a page that the table does not name: the query is rotated all the same
    c.cpu.table[3, 2] = -1
    c.gpu._buf["table"].upload(c.cpu.table)
    c.append([3, 1], [min(n, 33), n], *c.rows(rng, 2, n, 2))
    c.gpu.extend(1, seqs=[99], counts=[1])
    c.append([1, 0], [n, 1], *c.rows(rng, 2, n, 2), write=False)
    assert c.gpu.status() == 2


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("normed", [False, True])
def test_extreme_values(hip_ready, n, normed):
    rng = np.random.default_rng(n)
    for d in (64, 128, 256):
        c = Rope(hip_ready, 1, 8, d, 16, 40, 3, 8)
        c.extend([0, 1], [n + 5, n])
        q, k, v = c.rows(rng, 2, n, 8)
        for x in (q, k, v):
            x[0, 0, 0], x[0, 1, 0] = 0, 65504
            x[0, 0, 1] = np.float16(2.0 ** -24) * rng.integers(-9, 10, d)
            x[0, 0, 2, 7], x[0, 1, 3, d - 1], x[1, 2, 4, 3] = np.nan, np.inf, -np.inf
            x[1, 0, 5] *= np.float16(2.0 ** -12)
            x[1, 1, 6] = np.where(np.arange(d) % 32 == 5, 60000, 1)
            x[1, 1, 7] = (np.arange(d) % 14 - 6.5)
            x[1, 1, 7, ::32] = 7
        q_norm, k_norm = c.norms(rng) if normed else (None, None)
        c.append([0, 1], [n, n], q, k, v, q_norm, k_norm)


def test_far_positions_and_long_tables(hip_ready):
    """Positions whose angles an FP32 product would have off by hundredths."""
    rng = np.random.default_rng(2)
    c = Rope(hip_ready, 1, 1, 64, 4096, 70, 2, 40, theta=1e6)
    c.extend([0, 1], [163840, 100000])
    for n in (1, 20):
        c.append([0, 1], [n, n], *c.rows(rng, 2, n, 2), *c.norms(rng))


@pytest.mark.parametrize("n", [1, 5, 64, 100])
def test_unturned_rows_are_an_append(hip_ready, n):
    """Without norms and with no angle the pages are byte for byte kv4_append's."""
    rng = np.random.default_rng(n)
    pages = []
    for rope in (False, True):
        rng = np.random.default_rng(n)
        c = Rope(hip_ready, 1, 2, 128, 16, 40, 3, 12)
        c.table[:, 0], c.table[:, 1] = 1, 0
        c.dtable = dev(hip_ready, c.table)
        c.extend([0, 1], [7, 30])
        c.extend([0, 1], [n, n])
        q, k, v = c.rows(rng, 2, n, 2)
        if rope:
            c.append([0, 1], [n, n], q, k, v)
        else:
            dk, dv = dev(hip_ready, k), dev(hip_ready, v)
            c.gpu.append(0, dk.ptr, dv.ptr, 2, n, seqs=[0, 1])
        pages.append(c.gpu._buf["pages"].to_numpy(np.uint8, c.cpu.pages.shape))
    np.testing.assert_array_equal(*pages)


# ------------------------------------------------------------------ adapters
def run_lora(cm, x, A, B, scales, ids, counts, base, pad=(0, 0, 0), in_place=False):
    """x [b][S][K], base [b][S][N]; pad: values more per row of x, base, y. -> y [b][S][N]"""
    b, n, K = x.shape
    N, r = B.shape[1:]

    def rows(a, extra, fill):
        t = np.full((b * n, a.shape[-1] + extra), np.float16(fill))
        t[:, :a.shape[-1]] = a.reshape(b * n, -1)
        return dev(cm, t)
    dx, db = rows(x, pad[0], np.nan), rows(base, pad[1], np.nan)
    dy = db if in_place else dev(cm, np.full((b * n, N + pad[2]), MARK))
    ys = N + (pad[1] if in_place else pad[2])
    dA, dB, dids = dev(cm, A), dev(cm, B), dev(cm, np.asarray(ids, np.int32))
    ds = None if scales is None else dev(cm, np.asarray(scales, np.float32))
    dc = None if counts is None else dev(cm, np.asarray(counts, np.int32))
    cm.call("cactus_hip_lora_add_f16", dx.ptr, K + pad[0], dA.ptr, dB.ptr, ds and ds.ptr, len(A), r, dids.ptr, dc and dc.ptr,
            db.ptr, N + pad[1], dy.ptr, ys, b, n, K, N, None)
    y = dy.to_numpy(np.float16, (b * n, ys))
    tail = y[:, N:].view(np.uint16)
    assert (tail == np.float16(np.nan if in_place else MARK).view(np.uint16)).all(), "values behind a row changed"
    return y[:, :N].reshape(b, n, N)


def check_lora(got, x, A, B, scales, ids, counts, base, in_place=False):
    for i, a in enumerate(ids):
        m = x.shape[1] if counts is None else min(max(counts[i], 0), x.shape[1])
        stay = base[i, m:] if in_place else np.full_like(base[i, m:], MARK)
        np.testing.assert_array_equal(got[i, m:].view(np.uint16), stay.view(np.uint16), err_msg=f"request {i}: rows that stay")
        if not 0 <= a < len(A):
            np.testing.assert_array_equal(got[i, :m].view(np.uint16), base[i, :m].view(np.uint16), err_msg=f"request {i}: no adapter")
            continue
        s = 1.0 if scales is None else float(np.float32(scales[a]))
        y, err = S.lora(x[i, :m], A[a], B[a], s, base[i, :m])
        off = np.abs(got[i, :m].astype(np.float64) - y) - err
        assert (off <= 0).all(), f"request {i}: {off.max()} over the bound"


def adapters(rng, n, r, K, N):
    return f16(rng, n, r, K, scale=K ** -0.5), f16(rng, n, N, r, scale=r ** -0.5), 0.25 + rng.random(n).astype(np.float32)


@pytest.mark.parametrize("r", [8, 16, 24, 32, 40, 64, 128, 256])
@pytest.mark.parametrize("b,n,K,N", [(1, 1, 64, 40), (3, 1, 520, 264), (2, 17, 72, 136), (3, 40, 256, 128)])
def test_lora_sizes(hip_ready, r, b, n, K, N):
    rng = np.random.default_rng(r + K)
    A, B, s = adapters(rng, 4, r, K, N)
    x, base = f16(rng, b, n, K), f16(rng, b, n, N, scale=0.1)
    ids = rng.integers(0, 4, b)
    check_lora(run_lora(hip_ready, x, A, B, s, ids, None, base), x, A, B, s, ids, None, base)


@pytest.mark.parametrize("b,n,K,N,r", [(1, 1, 8, 8, 8), (1, 1, 16, 4096, 16), (1, 2, 4096, 8, 8), (1, 300, 1000, 1048, 16),
                                       (70, 1, 1024, 2048, 16), (2, 130, 2048, 520, 64), (5, 65, 24, 72, 24), (1, 513, 40, 16, 8),
                                       (1, 1, 11008, 200, 16), (9, 1, 64, 11008, 32)])
def test_lora_shapes(hip_ready, b, n, K, N, r):
    rng = np.random.default_rng(b + n + K)
    A, B, s = adapters(rng, 3, r, K, N)
    x, base = f16(rng, b, n, K), f16(rng, b, n, N)
    ids = rng.integers(-1, 3, b)
    check_lora(run_lora(hip_ready, x, A, B, s, ids, None, base), x, A, B, s, ids, None, base)


@pytest.mark.parametrize("n", [1, 5, 16, 33, 70])
@pytest.mark.parametrize("in_place", [False, True])
def test_lora_requests(hip_ready, n, in_place):
    """Rows that are not there, requests without an adapter, numbers outside, one adapter for several, strides."""
    rng = np.random.default_rng(n)
    A, B, s = adapters(rng, 3, 16, 200, 328)
    ids = [2, -1, 0, 3, 0, 1, -(1 << 31), (1 << 31) - 1, 2]
    counts = [n, n, max(0, n - 1), n, 0, n // 2, n, 1, -3]
    x, base = f16(rng, 9, n, 200), f16(rng, 9, n, 328)
    for c in (counts, [n + 1] * 9):
        for i, m in enumerate(c):
            x[i, max(m, 0):] = np.nan        # not read: no row of the request is touched by them
        got = run_lora(hip_ready, x, A, B, s, ids, c, base, (8, 16, 24), in_place)
        check_lora(got, x, A, B, s, ids, c, base, in_place)
        x = f16(rng, 9, n, 200)


def test_lora_without_scales_adapters_or_inputs(hip_ready):
    rng = np.random.default_rng(0)
    A, B, _ = adapters(rng, 2, 8, 64, 64)
    x, base = f16(rng, 2, 3, 64), f16(rng, 2, 3, 64)
    check_lora(run_lora(hip_ready, x, A, B, None, [1, 0], None, base), x, A, B, None, [1, 0], None, base)
    got = run_lora(hip_ready, x, A[:0], B[:0], None, [1, 0], None, base)
    np.testing.assert_array_equal(got, base)
    got = run_lora(hip_ready, x[..., :0], A[..., :0], B, None, [1, 0], None, base)      # K = 0: nothing to add
    np.testing.assert_array_equal(got, base)


@pytest.mark.parametrize("n", [1, 20, 80])
@pytest.mark.parametrize("r", [8, 64])
def test_lora_ranges(hip_ready, n, r):
    """Subnormal and huge weights and activations: the middle's values pass FP16's range on both sides."""
    rng = np.random.default_rng(n + r)
    K, N = 264, 72
    for ax, aa, ab, s in ((2.0 ** -14, 2.0 ** -14, 1.0, 1.0), (200.0, 200.0, 2.0 ** -12, 2.0 ** -8), (1.0, 2.0 ** -20, 60.0, 2.0 ** 12),
                          (100.0, 1.0, 2.0 ** -22, 3.0), (3000.0, 3000.0, 2.0 ** -24, 2.0 ** -10), (0.0, 1.0, 1.0, 1.0)):
        A, B = f16(rng, 2, r, K, scale=aa), f16(rng, 2, N, r, scale=ab)
        x, base = f16(rng, 2, n, K, scale=ax), f16(rng, 2, n, N, scale=1e-3)
        sc = np.array([s, -s], np.float32)
        check_lora(run_lora(hip_ready, x, A, B, sc, [0, 1], None, base), x, A, B, sc, [0, 1], None, base)


@pytest.mark.parametrize("n", [1, 2, 20, 80])
def test_lora_keeps_nan_and_infinity_in_their_rows(hip_ready, n):
    rng = np.random.default_rng(n)
    K, N, r = 136, 72, 16
    A, B, s = adapters(rng, 2, r, K, N)
    x, base = f16(rng, 2, n, K), f16(rng, 2, n, N)
    clean = run_lora(hip_ready, x, A, B, s, [0, 1], None, base)
    for bad in (np.nan, np.inf, -np.inf):
        y, z = x.copy(), base.copy()
        y[0, n // 2, 5], z[1, 0, 7] = bad, bad
        got = run_lora(hip_ready, y, A, B, s, [0, 1], None, z)
        for i in range(2):
            for j in range(n):
                if (i, j) == (0, n // 2):
                    # every output has a part of the bad value: no number comes of it where the product is not 0
                    assert not np.isfinite(got[i, j]).any()
                    if np.isinf(bad):
                        with np.errstate(invalid="ignore"):
                            h = A[0, :, 5].astype(np.float64) * bad
                            want = B[0].astype(np.float64) @ h * float(s[0])
                        np.testing.assert_array_equal(got[i, j].astype(np.float64), want)
                elif (i, j) == (1, 0):
                    np.testing.assert_array_equal(got[i, j, 7], np.float16(bad))
                    np.testing.assert_array_equal(np.delete(got[i, j], 7), np.delete(clean[i, j], 7))
                else:
                    np.testing.assert_array_equal(got[i, j], clean[i, j])


# ------------------------------------------------------------------ rules on logits
def run_rules(cm, x, V, seqs=None, hist=None, lens=None, pen=None, bias=None, bias_counts=None, masks=None, mask_ids=None,
              max_seqs=None, stride=None, out_stride=None, in_place=False, best=True, offset=0, passes=1):
    """x [rows][V] FP16 or FP32; the other arrays as the settings hold them. Checks against the restatement."""
    from cactus_amd.logits import RulesDesc
    n, half = len(x), x.dtype == np.float16
    max_seqs = max_seqs or n
    stride, out_stride = stride or V, out_stride or V
    if in_place:
        out_stride = stride
    keep = {k: dev(cm, v) for k, v in dict(
        history=hist, history_lens=lens, repetition=pen and np.float32(pen[0]), frequency=pen and np.float32(pen[1]),
        presence=pen and np.float32(pen[2]), bias_tokens=bias and bias[0], bias_values=bias and bias[1], bias_counts=bias_counts,
        masks=masks, mask_ids=mask_ids, seqs=None if seqs is None else np.int32(seqs)).items() if v is not None}
    desc = RulesDesc(max_seqs=max_seqs, **{k: b.ptr for k, b in keep.items() if k != "seqs"})
    desc.history_stride = 0 if hist is None else hist.shape[1]
    desc.bias_stride = 0 if bias is None else bias[0].shape[1]
    desc.num_masks, desc.mask_stride = (0, 0) if masks is None else masks.shape
    rows = np.full(n * stride + offset, x.dtype.type(np.nan))
    rows[offset:].reshape(n, stride)[:, :V] = x
    mark = np.float32(-77.25)
    dx, do = dev(cm, rows), dev(cm, np.full(n * out_stride + offset, mark))
    db, work = dev(cm, np.full(n, 0xABCDEF, np.uint32)), dev(cm, np.zeros(4 * n, np.uint32))
    pin, pout = dx.ptr + offset * x.itemsize, do.ptr + 4 * offset
    for _ in range(passes):
        cm.call("cactus_hip_logits_rules_f16" if half else "cactus_hip_logits_rules_f32", desc.ref,
                keep["seqs"].ptr if "seqs" in keep else None, pin, stride, pin if in_place else pout, out_stride,
                db.ptr if best else None, n, V, work.ptr if best else None, 16 * n if best else 0, None)
    assert (work.to_numpy(np.uint32, 4 * n) == 0).all()
    got = (dx if in_place else do).to_numpy(np.float32, n * out_stride + offset)
    assert (got[:offset].view(np.uint32) == np.float32(np.nan if in_place else mark).view(np.uint32)).all()
    got, top = got[offset:].reshape(n, out_stride), db.to_numpy(np.uint32, n)
    rest = got[:, V:]
    assert np.isnan(rest).all() if in_place else (rest == mark).all(), "values behind a row changed"
    for i in range(n):
        s = i if seqs is None else seqs[i]
        if not 0 <= s < max_seqs:
            assert top[i] == 0xABCDEF
            np.testing.assert_array_equal(got[i, :V], x[i] if in_place else np.full(V, mark))
            continue
        h = () if hist is None else hist[s] if lens is None else hist[s, :max(0, lens[s])]
        bl = () if bias is None else zip(bias[0][s][:None if bias_counts is None else max(0, bias_counts[s])], bias[1][s])
        mid = None if masks is None else s if mask_ids is None else mask_ids[s]
        m = None
        if mid is not None and mid >= 0:
            m = np.zeros(V, bool) if mid >= len(masks) else np.unpackbits(masks[mid].view(np.uint8), bitorder="little")[:V] > 0
        want, b = S.rules(x[i], h, *(p[s] for p in pen) if pen else (), bias=list(bl), mask=m)
        np.testing.assert_array_equal(got[i, :V], want, err_msg=f"row {i}")
        if best:
            assert top[i] == b, f"row {i}"
    return got[:, :V], top


def settings(rng, slots, V, H=40, nb=9, masks=3):
    t = rng.integers(-3, V + 3, (slots, H)).astype(np.int32)
    t[:, ::3] = t[:, :1]                    # the same token many times
    lens = rng.integers(0, H + 1, slots).astype(np.int32)
    lens[0], lens[-1] = 0, H + 5            # (beyond the list: all of it)
    pen = [1 + rng.random(slots), rng.random(slots), rng.random(slots)]
    bt = rng.integers(-2, V + 2, (slots, nb)).astype(np.int32)
    bt[:, 1::3] = bt[:, :1]                 # entries that name a token again
    bt[:, 2] = t[:, 0]                      # a penalized token with a bias
    bv = (3 * rng.standard_normal((slots, nb))).astype(np.float32)
    mk = rng.integers(0, 1 << 32, (masks, -(-V // 32) + 1), dtype=np.uint64).astype(np.uint32)
    return dict(hist=t, lens=np.minimum(lens, H), pen=pen, bias=(bt, bv), bias_counts=rng.integers(0, nb + 1, slots).astype(np.int32),
                masks=mk, mask_ids=rng.integers(-1, masks, slots).astype(np.int32))


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 4096, 4097, 8200, 32003, 70001])
@pytest.mark.parametrize("kind", [np.float16, np.float32])
def test_rules(hip_ready, V, kind):
    rng = np.random.default_rng(V)
    x = (4 * rng.standard_normal((5, V))).astype(kind)
    run_rules(hip_ready, x, V, **settings(rng, 5, V), passes=2)


@pytest.mark.parametrize("kind", [np.float16, np.float32])
@pytest.mark.parametrize("stride,out_stride,offset", [(0, 0, 0), (5, 0, 1), (8, 8, 0), (0, 3, 3), (2, 4, 2), (6, 2, 7)])
def test_rules_strides_and_alignment(hip_ready, kind, stride, out_stride, offset):
    rng = np.random.default_rng(stride)
    for V in (7, 640, 5001):
        x = (4 * rng.standard_normal((3, V))).astype(kind)
        run_rules(hip_ready, x, V, **settings(rng, 3, V), stride=V + stride, out_stride=V + out_stride, offset=offset)


@pytest.mark.parametrize("part", ["hist", "bias", "masks", "none"])
def test_rules_one_at_a_time(hip_ready, part):
    rng = np.random.default_rng(4)
    for V in (1000, 9001):
        s = settings(rng, 4, V)
        keys = {"hist": ("hist", "lens", "pen"), "bias": ("bias", "bias_counts"), "masks": ("masks", "mask_ids"), "none": ()}[part]
        x = (4 * rng.standard_normal((4, V))).astype(np.float16)
        run_rules(hip_ready, x, V, **{k: s[k] for k in keys})
        run_rules(hip_ready, x, V, **{k: s[k] for k in keys[:1]}, **({"max_seqs": 3, "seqs": [2, 0, 2, 1]} if part == "masks" else {}))
        run_rules(hip_ready, x, V, **{k: s[k] for k in keys}, best=False)


def test_rules_slots(hip_ready):
    """Rows of any slots, the same one twice, slots that do not exist."""
    rng = np.random.default_rng(6)
    V = 6001
    x = (4 * rng.standard_normal((7, V))).astype(np.float32)
    s = settings(rng, 9, V)
    s["mask_ids"][4] = 3                    # a mask that does not exist: nothing is allowed
    for in_place in (False, True):
        run_rules(hip_ready, x, V, **s, seqs=[8, 2, -1, 2, 9, 4, 1 << 30], max_seqs=9, in_place=in_place)


def test_rules_values(hip_ready):
    rng = np.random.default_rng(7)
    V = 5000
    for kind in (np.float16, np.float32):
        x = (4 * rng.standard_normal((9, V))).astype(kind)
        x[0] = -np.inf
        x[1] = np.nan
        x[2, ::7], x[2, 3] = np.nan, np.inf
        x[3] = np.where(np.arange(V) % 2, 0.0, -0.0)
        x[4] = -np.inf
        x[4, 4321] = np.finfo(kind).min
        x[5] = 1.5                            # all the same: the first that is left
        x[6, [17, 4999]] = 60000
        x[7] = -np.abs(x[7])
        s = settings(rng, 9, V)
        run_rules(hip_ready, x, V, **s)
        run_rules(hip_ready, x, V)
        s["pen"] = [np.ones(9), np.zeros(9), np.zeros(9)]
        s["masks"][:] = 0
        s["masks"][1, 100] = 1 << 5
        run_rules(hip_ready, x, V, **s)


def test_rules_long_histories_and_lists(hip_ready):
    rng = np.random.default_rng(8)
    V = 20011
    s = settings(rng, 3, V, H=70000, nb=1024)
    s["hist"][1] = 77
    s["bias"][0][2] = 5                       # 1024 entries for one token
    run_rules(hip_ready, (4 * rng.standard_normal((3, V))).astype(np.float16), V, **s)


def test_rules_tokens_at_the_ends_of_32_bits(hip_ready):
    """Outside the vocabulary by as much as there is, in histories on either side of the entries that are read early."""
    rng = np.random.default_rng(18)
    ends = np.int32([-(1 << 31), -(1 << 31) + 1, -(1 << 31) + 8192, (1 << 31) - 1, (1 << 31) - 8192, -8192, -1])
    for V, H in ((5, 7), (20011, 40), (9001, 5000)):
        s = settings(rng, 2, V, H=H)
        s["hist"][:, rng.permutation(H)[:max(7, H // 3)]] = np.resize(ends, max(7, H // 3))
        s["lens"][:] = H
        s["bias"][0][:, 3:7] = ends[:4]
        s["bias_counts"][:] = 9
        for kind in (np.float16, np.float32):
            run_rules(hip_ready, (4 * rng.standard_normal((2, V))).astype(kind), V, **s)


def test_rules_many_rows(hip_ready):
    rng = np.random.default_rng(9)
    for n, V in ((300, 1111), (40, 30000)):
        x = (4 * rng.standard_normal((n, V))).astype(np.float16)
        run_rules(hip_ready, x, V, **settings(rng, n, V), passes=3)


def test_rules_owner(hip_ready):
    from cactus_amd.logits import LogitsRules
    rng = np.random.default_rng(10)
    V = 1234
    x = (4 * rng.standard_normal((2, V))).astype(np.float16)
    r = LogitsRules(3, V, max_history=10, max_bias=4, num_masks=2)
    r.set_history(2, [5, 5, 9])
    r.set_penalties(2, 1.5, 0.25, 0.5)
    r.set_bias(2, [9, 100], [2.0, -3.0])
    allowed = rng.random(V) < 0.5
    r.set_mask(1, allowed)
    r.use_mask(2, 1)
    seqs = dev(hip_ready, np.int32([2, 0]))
    dx, do, db = dev(hip_ready, x), hip_ready.DeviceBuffer(8 * V), hip_ready.DeviceBuffer(8)
    r.apply(dx.ptr, do.ptr, 2, db.ptr, seqs=seqs.ptr)
    got, top = do.to_numpy(np.float32, (2, V)), db.to_numpy(np.uint32, 2)
    for i, want in enumerate((S.rules(x[0], [5, 5, 9], 1.5, 0.25, 0.5, [(9, 2.0), (100, -3.0)], allowed), S.rules(x[1]))):
        np.testing.assert_array_equal(got[i], want[0])
        assert top[i] == want[1]


# ------------------------------------------------------------------ far offsets
def test_lora_behind_4_gb(hip_ready):
    """An adapter whose weights lie behind 2^32 bytes, and rows that do."""
    rng = np.random.default_rng(11)
    cm = hip_ready
    r, K, N, n = 256, 16384, 16384, 520                       # 8 MB of each per adapter
    A, B, _ = adapters(rng, 1, r, K, N)
    dA, dB = cm.DeviceBuffer(n * A.nbytes), cm.DeviceBuffer(n * B.nbytes)
    for buf, a in ((dA, A), (dB, B)):
        cm.call("cactus_hip_memcpy_h2d", buf.ptr + (n - 1) * a.nbytes, a.ctypes.data, a.nbytes, None)
    ids = dev(cm, np.int32([n - 1, n - 1]))
    for S, stride in ((1, 1 << 31), (20, 1 << 27)):
        x, base = f16(rng, 2, S, K), f16(rng, 2, S, N)
        big = cm.DeviceBuffer((2 * S - 1) * stride * 2 + 2 * (K + N))          # rows of x and of y, far from each other
        for b in range(2):
            for i in range(S):
                row = np.concatenate((x[b, i], base[b, i]))
                cm.call("cactus_hip_memcpy_h2d", big.ptr + (b * S + i) * stride * 2, row.ctypes.data, row.nbytes, None)
        y_at = big.ptr + 2 * K
        cm.call("cactus_hip_lora_add_f16", big.ptr, stride, dA.ptr, dB.ptr, None, n, r, ids.ptr, None, y_at, stride, y_at, stride,
                2, S, K, N, None)
        got = np.zeros((2, S, N), np.float16)
        for b in range(2):
            for i in range(S):
                cm.call("cactus_hip_memcpy_d2h", got[b, i].ctypes.data, y_at + (b * S + i) * stride * 2, 2 * N, None)
        check_lora(got, x, A, B, None, [0, 0], None, base)
        big.free()


def test_rules_behind_4_gb(hip_ready):
    rng = np.random.default_rng(12)
    cm, V, stride, n = hip_ready, 5003, (1 << 29) + 4, 4
    from cactus_amd.logits import RulesDesc
    x = (4 * rng.standard_normal((n, V))).astype(np.float32)
    big = cm.DeviceBuffer(((n - 1) * stride + V) * 4)
    for i in range(n):
        cm.call("cactus_hip_memcpy_h2d", big.ptr + 4 * i * stride, x[i].ctypes.data, x[i].nbytes, None)
    best, work = cm.DeviceBuffer(4 * n), dev(cm, np.zeros(4 * n, np.uint32))
    mask = rng.integers(0, 1 << 32, -(-V // 32), dtype=np.uint64).astype(np.uint32)
    dm, di = dev(cm, mask), dev(cm, np.zeros(n, np.int32))
    d = RulesDesc(max_seqs=n, masks=dm.ptr, mask_ids=di.ptr, num_masks=1, mask_stride=len(mask))
    cm.call("cactus_hip_logits_rules_f32", d.ref, None, big.ptr, stride, big.ptr, stride, best.ptr, n, V, work.ptr, 16 * n, None)
    got = np.zeros(V, np.float32)
    for i in range(n):
        cm.call("cactus_hip_memcpy_d2h", got.ctypes.data, big.ptr + 4 * i * stride, 4 * V, None)
        want, b = S.rules(x[i], mask=np.unpackbits(mask.view(np.uint8), bitorder="little")[:V] > 0)
        np.testing.assert_array_equal(got, want)
        assert best.to_numpy(np.uint32, n)[i] == b


@pytest.mark.parametrize("n", [1, 200])
def test_append_on_pages_behind_4_gb(hip_ready, n):
    rng = np.random.default_rng(13)
    cm, d, H, ps, pages = hip_ready, 256, 8, 4096, 480        # 9.4 MB per page
    from cactus_amd.kv4 import KV4Cache
    c = KV4Cache(1, H, d, ps, pages, 2, 2)
    c.extend(1, n)
    t = c.tables()
    t["table"][0, 0] = pages - 1
    c._buf["table"].upload(t["table"])
    table = S.rope_table(2 * ps, d, 1e6)
    dt, q, k, v = dev(cm, table), f16(rng, 1, n, 4, d), f16(rng, 1, n, H, d), f16(rng, 1, n, H, d)
    dq, dk, dv, do = dev(cm, q), dev(cm, k), dev(cm, v), cm.DeviceBuffer(q.nbytes)
    c.append_rope(0, dq.ptr, do.ptr, 4, dk.ptr, dv.ptr, 1, n, dt.ptr, 2 * ps)
    ok, ov = cm.DeviceBuffer(k.nbytes), cm.DeviceBuffer(v.nbytes)
    c.read(0, ok.ptr, ov.ptr, 1, n)
    key = np.stack([S.rotated(k[0, i], None, 0, table[i])[0] for i in range(n)]).astype(np.float16)
    for buf, want in ((ok, key), (ov, v[0])):
        np.testing.assert_array_equal(buf.to_numpy(np.float16, want.shape).astype(np.float64), values(*quantize(want)).reshape(want.shape))


# ------------------------------------------------------------------ streams, graphs, a whole step
def test_calls_on_two_streams(hip_ready):
    """Calls that overlap, each with its own workspace and outputs, give what they give alone."""
    from cactus_amd.logits import RulesDesc
    rng = np.random.default_rng(14)
    cm, V, rows = hip_ready, 30011, 24
    x = (4 * rng.standard_normal((2, rows, V))).astype(np.float16)
    s = settings(rng, rows, V)
    keep = [dev(cm, a) for a in (s["hist"], s["lens"], *(np.float32(p) for p in s["pen"]), *s["bias"], s["bias_counts"])]
    d = RulesDesc(max_seqs=rows, history_stride=s["hist"].shape[1], bias_stride=s["bias"][0].shape[1],
                  **dict(zip(("history", "history_lens", "repetition", "frequency", "presence", "bias_tokens", "bias_values", "bias_counts"),
                             (b.ptr for b in keep))))
    streams = [cm.Stream(), cm.Stream()]
    bufs = [(dev(cm, x[i]), cm.DeviceBuffer(4 * rows * V), cm.DeviceBuffer(4 * rows), dev(cm, np.zeros(4 * rows, np.uint32))) for i in range(2)]
    A, B, sc = adapters(rng, 3, 16, 512, 1024)
    xs, base = f16(rng, 2, 9, 40, 512), f16(rng, 2, 9, 40, 1024)
    w = [dev(cm, a) for a in (A, B, sc)]
    ids = dev(cm, np.int32([0, 1, 2, -1, 0, 1, 2, 0, 1]))
    lb = [(dev(cm, xs[i]), dev(cm, base[i]), cm.DeviceBuffer(base[i].nbytes)) for i in range(2)]
    for _ in range(20):
        for i in (0, 1):
            a, o, b, work = bufs[i]
            cm.call("cactus_hip_logits_rules_f16", d.ref, None, a.ptr, V, o.ptr, V, b.ptr, rows, V, work.ptr, 16 * rows, streams[i].handle)
            a, z, y = lb[i]
            cm.call("cactus_hip_lora_add_f16", a.ptr, 512, w[0].ptr, w[1].ptr, w[2].ptr, 3, 16, ids.ptr, None, z.ptr, 1024, y.ptr,
                    1024, 9, 40, 512, 1024, streams[i].handle)
    for i in (0, 1):
        streams[i].sync()
        got, top = bufs[i][1].to_numpy(np.float32, (rows, V)), bufs[i][2].to_numpy(np.uint32, rows)
        for r in range(rows):
            want, b = S.rules(x[i, r], s["hist"][r, :s["lens"][r]], *(p[r] for p in s["pen"]),
                              list(zip(s["bias"][0][r, :s["bias_counts"][r]], s["bias"][1][r])))
            np.testing.assert_array_equal(got[r], want)
            assert top[r] == b
        check_lora(lb[i][2].to_numpy(np.float16, (9, 40, 1024)), xs[i], A, B, sc, [0, 1, 2, -1, 0, 1, 2, 0, 1], None, base[i])


class Step:
    """A layer and the head of a small model for many sequences: the projections that requests share with their
    adapters, the rotated append, attention over the pages, the logits and their rules."""
    HID, HQ, H, D, V, R = 256, 4, 2, 64, 3001, 8

    def __init__(self, cm, B, rng):
        from cactus_amd.kv4 import KV4Cache
        from cactus_amd.logits import LogitsRules
        from cactus_amd.lora import LoraAdapters
        self.cm, self.B = cm, B
        n = (self.HQ + 2 * self.H) * self.D
        self.qkv_w = rng.integers(-127, 128, (n, self.HID)).astype(np.int8)
        self.qkv_s = (0.001 + 0.001 * rng.random((n, self.HID // 32))).astype(np.float16)
        self.head = f16(rng, self.V, self.HQ * self.D, scale=0.2)
        self.norms = [(1 + 0.3 * rng.standard_normal(self.D)).astype(np.float16) for _ in range(2)]
        self.A, self.Bw, self.sc = adapters(rng, 3, self.R, self.HID, n)
        self.lora = LoraAdapters(3, self.R, self.HID, n)
        for i in range(3):
            self.lora.set(i, self.A[i], self.Bw[i], self.sc[i])
        self.ids = [i % 4 - 1 for i in range(B)]
        self.cache = KV4Cache(1, self.H, self.D, 16, 12 * B, B, 10)
        cm.call("cactus_hip_memset", self.cache._buf["pages"].ptr, 0, self.cache._buf["pages"].nbytes, None)
        self.table = S.rope_table(160, self.D, 1e4)
        self.rules = LogitsRules(B, self.V, 20, 3, 2)
        self.hist = [rng.integers(0, self.V, i % 20) for i in range(B)]
        self.allowed = rng.random(self.V) < 0.3
        for i in range(B):
            self.rules.set_history(i, self.hist[i])
            self.rules.set_penalties(i, 1.3, 0.2, 0.1)
        self.rules.set_bias(0, [5, 5], [3.0, 1.0])
        self.rules.set_mask(1, self.allowed)
        self.rules.use_mask(B - 1, 1)
        self.d = {k: dev(cm, v) for k, v in dict(w=self.qkv_w, s=self.qkv_s, head=self.head, qn=self.norms[0], kn=self.norms[1],
                                                 table=self.table, ids=np.int32(self.ids)).items()}

    def buffers(self, S_):
        n, B = (self.HQ + 2 * self.H) * self.D, self.B
        size = dict(x=2 * B * S_ * self.HID, proj=2 * B * S_ * n, qkv=2 * B * S_ * n, q=2 * B * S_ * self.HQ * self.D,
                    o=2 * B * S_ * self.HQ * self.D, logits=2 * B * self.V, out=4 * B * self.V, best=4 * B, counts=4 * B)
        return {k: self.cm.DeviceBuffer(v) for k, v in size.items()}

    def run(self, b, S_, stream=None):
        cm, B, HQ, H, D = self.cm, self.B, self.HQ, self.H, self.D
        n = (HQ + 2 * H) * D
        self.cache.extend(B, 0, None, b["counts"].ptr, stream)
        cm.call("cactus_hip_matmul_int8_f16act_noalloc", b["x"].ptr, self.d["w"].ptr, self.d["s"].ptr, b["proj"].ptr, B * S_, self.HID, n, 32, stream)
        self.lora.add(b["x"].ptr, b["proj"].ptr, b["qkv"].ptr, self.d["ids"].ptr, B, S_, b["counts"].ptr, stream=stream)
        self.cache.append_rope(0, b["qkv"].ptr, b["q"].ptr, HQ, b["qkv"].ptr + 2 * HQ * D, b["qkv"].ptr + 2 * (HQ + H) * D, B, S_,
                               self.d["table"].ptr, 160, n, n, self.d["qn"].ptr, self.d["kn"].ptr, 1e-6, None, b["counts"].ptr, stream)
        self.cache.attention(0, b["q"].ptr, b["o"].ptr, B, S_, HQ, counts=b["counts"].ptr, stream=stream)
        if S_ == 1:
            cm.call("cactus_hip_matmul_f16", b["o"].ptr, self.d["head"].ptr, b["logits"].ptr, B, HQ * D, self.V, stream)
            self.rules.apply(b["logits"].ptr, b["out"].ptr, B, b["best"].ptr, stream=stream)


def test_a_step_of_many_sequences(hip_ready):
    """Prompts of different lengths, then single tokens: every stage against its restatement."""
    rng = np.random.default_rng(15)
    B = 7
    s = Step(hip_ready, B, rng)
    HQ, H, D = s.HQ, s.H, s.D
    cpu = Model(1, H, D, 16, 12 * B, B, 10)
    s.cache._buf["pages"].upload(cpu.pages)
    for S_, counts in ((40, [40, 3, 17, 0, 25, 1, 33]), (1, [1] * B), (3, [3, 1, 2, 0, 3, 3, 1]), (1, [1, 1, 0, 1, 1, 1, 1])):
        b = s.buffers(S_)
        x = f16(rng, B, S_, s.HID)
        b["x"].upload(x)
        b["counts"].upload(np.int32(counts))
        b["q"].upload(np.zeros((B, S_, HQ, D), np.float16))
        b["o"].upload(np.zeros((B, S_, HQ, D), np.float16))
        b["qkv"].upload(np.zeros((B, S_, (HQ + 2 * H) * D), np.float16))
        s.run(b, S_)
        assert s.cache.status() == 0 and cpu.extend(list(range(B)), counts) == 0
        proj, qkv = (b[k].to_numpy(np.float16, (B, S_, HQ + 2 * H, D)) for k in ("proj", "qkv"))
        q, o = (b[k].to_numpy(np.float16, (B, S_, HQ, D)) for k in ("q", "o"))
        for i, m in enumerate(counts):
            n = (HQ + 2 * H) * D
            flat, before = qkv[i, :m].reshape(m, n), proj[i, :m].reshape(m, n)
            if s.ids[i] < 0:
                np.testing.assert_array_equal(flat, before)
            elif m:
                y, err = S.lora(x[i, :m], s.A[s.ids[i]], s.Bw[s.ids[i]], float(np.float32(s.sc[s.ids[i]])), before)
                assert (np.abs(flat - y) <= err).all()
            for r in range(m):
                pos = int(cpu.lens[i]) - m + r
                y, err = S.rotated(qkv[i, r, :HQ], s.norms[0], 1e-6, s.table[pos])
                assert (np.abs(q[i, r] - y) <= S.half_step(y) + err).all()
                key = S.rotated(qkv[i, r, HQ:HQ + H], s.norms[1], 1e-6, s.table[pos])[0].astype(np.float16)
                cpu.write(0, i, pos, key, qkv[i, r, HQ + H:])
            if m:
                (kc, ks), (vc, vs) = cpu.read(0, i)
                want, tol = attention(q[i, :m], kc, ks, vc, vs, len(kc), D ** -0.5)
                assert (np.abs(o[i, :m] - want) <= tol).all()
        np.testing.assert_array_equal(s.cache._buf["pages"].to_numpy(np.uint8, cpu.pages.shape), cpu.pages)
        if S_ == 1:
            logits, out, best = b["logits"].to_numpy(np.float16, (B, s.V)), b["out"].to_numpy(np.float32, (B, s.V)), b["best"].to_numpy(np.uint32, B)
            for i in range(B):
                want, top = S.rules(logits[i], s.hist[i], 1.3, 0.2, 0.1, [(5, 3.0), (5, 1.0)] if i == 0 else [], s.allowed if i == B - 1 else None)
                np.testing.assert_array_equal(out[i], want)
                assert best[i] == top


def test_a_captured_step(hip_ready):
    """The step as a graph, replayed while the sequences grow, other work in between: what the eager step gives."""
    cm, B = hip_ready, 5
    a, e = (Step(cm, B, np.random.default_rng(16)) for _ in range(2))
    rng = np.random.default_rng(17)
    st = cm.Stream()
    ba, be, prompt = a.buffers(1), e.buffers(1), f16(rng, B, 20, a.HID)
    for s in (a, e):
        b = s.buffers(20)
        b["x"].upload(prompt)
        b["counts"].upload(np.int32([20, 1, 7, 16, 13]))
        s.run(b, 20, st.handle)
        st.sync()
    # one eager step before the capture, so that scratch memory is there
    xs = f16(rng, 9, B, 1, a.HID)
    for s, b in ((a, ba), (e, be)):
        b["counts"].upload(np.int32([1] * B))
        b["x"].upload(xs[0])
        s.run(b, 1, st.handle)
        st.sync()
    graph = ctypes.c_void_p()
    cm.call("cactus_hip_graph_capture_begin", st.handle)
    a.run(ba, 1, st.handle)
    cm.call("cactus_hip_graph_capture_end", st.handle, ctypes.byref(graph))
    for i, counts in enumerate([[1] * 5, [1, 0, 1, 1, 1], [1] * 5, [0, 0, 0, 1, 0], [1] * 5, [1] * 5, [1] * 5, [1] * 5]):
        for b in (ba, be):
            b["x"].upload(xs[i + 1])
            b["counts"].upload(np.int32(counts))
        cm.call("cactus_hip_graph_launch", graph, st.handle)
        e.run(be, 1, None)                 # on another stream, at the same time
        st.sync()
        cm.call("cactus_hip_stream_sync", None)
        assert a.cache.status(st.handle) == 0 and e.cache.status() == 0
        for k, kind in (("q", np.uint16), ("o", np.uint16), ("out", np.uint32), ("best", np.uint32)):
            n = ba[k].nbytes // np.dtype(kind).itemsize
            got, want = ba[k].to_numpy(kind, n), be[k].to_numpy(kind, n)
            rows = np.repeat(np.array(counts) > 0, n // B)      # (without a token: an old output's logits)
            np.testing.assert_array_equal(got[rows], want[rows], err_msg=f"replay {i}: {k}")
        for name, v in a.cache.tables().items():
            np.testing.assert_array_equal(v, e.cache.tables()[name])
        size = a.cache._buf["pages"].nbytes
        np.testing.assert_array_equal(a.cache._buf["pages"].to_numpy(np.uint8, size), e.cache._buf["pages"].to_numpy(np.uint8, size))
    cm.call("cactus_hip_graph_destroy", graph)
