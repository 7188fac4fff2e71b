"""The paged 4-bit KV cache on the GPU against its plain restatement."""
import ctypes
import math

import numpy as np
import pytest

from _kv4 import Model, attention, quantize, values

pytestmark = pytest.mark.gpu


class Cache:
    """A KV4Cache and its model side by side; fresh pages hold 0xFF bytes (NaN scales)."""

    def __init__(self, cm, layers=1, kv_heads=2, head_dim=64, page_size=16, num_pages=40, max_seqs=6, max_pages=12):
        from cactus_amd.kv4 import KV4Cache
        self.cm, self.shape = cm, (layers, kv_heads, head_dim, page_size, num_pages, max_seqs, max_pages)
        self.gpu, self.cpu = KV4Cache(*self.shape), Model(*self.shape)
        self.put_pages()

    def put_pages(self):
        self.gpu._buf["pages"].upload(self.cpu.pages)

    def pages(self):
        return self.gpu._buf["pages"].to_numpy(np.uint8, self.cpu.pages.shape)

    def check(self):
        t = self.gpu.tables()
        for name in ("table", "lens", "refs"):
            np.testing.assert_array_equal(t[name], getattr(self.cpu, name), err_msg=name)
        assert t["state"][0] == (self.cpu.refs == 0).sum()
        assert (self.cpu.refs[:t["state"][1]] > 0).all()
        np.testing.assert_array_equal(self.pages(), self.cpu.pages)

    def extend(self, seqs, counts):
        want = self.cpu.extend(seqs, counts)
        self.gpu.extend(len(seqs), seqs=seqs, counts=counts)
        assert self.gpu.status() == want
        return want

    def append(self, layer, seqs, counts, k, v, stride=None, named=True):
        """k, v [B][S][H][d]; the model and the GPU write the rows."""
        B, S, H, d = k.shape
        stride = stride or H * d
        rows = np.full((2, B * S, stride), 0x7E00, np.uint16).view(np.float16)
        rows[0, :, :H * d], rows[1, :, :H * d] = k.reshape(B * S, -1), v.reshape(B * S, -1)
        dk, dv = (self.cm.DeviceBuffer.from_numpy(r) for r in rows)
        self.gpu.append(layer, dk.ptr, dv.ptr, B, S, stride, seqs=list(seqs) if named else None, counts=list(counts))
        for b, (s, m) in enumerate(zip(seqs, counts)):
            for r in range(m):
                self.cpu.write(layer, s, self.cpu.lens[s] - m + r, k[b, r], v[b, r])

    def fill(self, rng, lens, seqs=None, layers=None, scale=1.0):
        """Random tokens for slots `seqs`, all layers."""
        seqs = list(range(len(lens))) if seqs is None else list(seqs)
        assert self.extend(seqs, lens) == 0
        S = max(max(lens), 1)
        for layer in range(self.cpu.layers):
            k = kv_rows(rng, len(lens), S, self.cpu.H, self.cpu.d, scale)
            self.append(layer, seqs, lens, k, kv_rows(rng, len(lens), S, self.cpu.H, self.cpu.d, scale))

    def attend(self, q, seqs, counts, layer=0, scale=0.0, window=0, sink=0, causal=True, stride=None, small=True):
        """Runs the kernel on q [B][S][Hq][d] and holds every row to the plain attention."""
        B, S, Hq, d = q.shape
        stride = stride or Hq * d
        rows = np.full((B * S, stride), np.float16(np.nan))
        rows[:, :Hq * d] = q.reshape(B * S, -1)
        mark = np.float16(-77.25)      # rows that are not there stay as they are
        dq, do = self.cm.DeviceBuffer.from_numpy(rows), self.cm.DeviceBuffer.from_numpy(np.full(q.shape, mark))
        self.gpu.attention(layer, dq.ptr, do.ptr, B, S, Hq, scale, window, sink, causal, stride, seqs=list(seqs),
                           counts=list(counts))
        o = do.to_numpy(np.float16, q.shape)
        for b, (s, m) in enumerate(zip(seqs, counts)):
            if not 0 <= s < self.cpu.max_seqs:
                m = 0
            assert (o[b, m:] == mark).all(), f"request {b}: rows behind the last one changed"
            if m == 0:
                continue
            (kc, ks), (vc, vs) = self.cpu.read(layer, s)
            want, tol = attention(q[b, :m], kc, ks, vc, vs, len(kc), scale or 1 / math.sqrt(d), window, sink, causal,
                                  small)
            got = o[b, :m].astype(np.float64)
            np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=f"request {b}: NaN")
            off = np.where(np.isnan(want), 0, np.abs(got - want) - tol)
            assert (off <= 0).all(), f"request {b}: off by {np.nanmax(np.abs(got - want))}, {np.max(off)} over the bound"
        return o


def kv_rows(rng, B, S, H, d, scale=1.0):
    x = rng.standard_normal((B, S, H, d)) * scale + rng.standard_normal((H, d)) * scale
    return (x * np.exp(0.7 * rng.standard_normal((H, d)))).astype(np.float16)


# ------------------------------------------------------------------ append and read
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("ps,S,lens", [(16, 1, [0, 15, 16, 17]), (16, 37, [0, 3, 29, 0]), (64, 70, [0, 63, 1, 40]),
                                       (256, 5, [250, 0, 14, 12])])
def test_append_writes_the_documented_bytes(hip_ready, d, ps, S, lens):
    rng = np.random.default_rng(d + ps + S)
    c = Cache(hip_ready, 2, 3, d, ps, 40, 6, 12)
    c.fill(rng, lens, seqs=[4, 0, 2, 1])
    counts = [S, max(1, S // 2), 0, max(1, S - 1)]
    seqs = [2, 4, 0, 1]
    assert c.extend(seqs, counts) == 0
    c.append(1, seqs, counts, kv_rows(rng, 4, S, 3, d), kv_rows(rng, 4, S, 3, d), stride=3 * d + 8)
    c.check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_of_extreme_values(hip_ready, d):
    rng = np.random.default_rng(5)
    x = kv_rows(rng, 1, 40, 1, d)
    x[0, 0] = 0
    x[0, 1] = 65504
    x[0, 2] = np.float16(2.0 ** -24) * rng.integers(-9, 10, (1, d))      # subnormals, scales that round to 0
    x[0, 3] = np.where(np.arange(d) % 32 == 5, 65504, 1)
    x[0, 4, 0, 7] = np.nan
    x[0, 5, 0, d - 1] = np.inf
    x[0, 6, 0, 40] = -np.inf
    x[0, 7] = (np.arange(d) % 15 - 7) * np.float16(0.5)                   # codes exactly on the grid
    x[0, 8] = (np.arange(d) % 14 - 6.5)                                   # ties
    x[0, 8, 0, ::32] = 7
    x[0, 9] = np.float16(2.0 ** -14) * rng.standard_normal((1, d)).astype(np.float16)
    c = Cache(hip_ready, 1, 1, d)
    assert c.extend([0], [40]) == 0
    c.append(0, [0], [40], x, -x[:, ::-1])
    c.check()
    dk, dv = (c.cm.DeviceBuffer(x.nbytes) for _ in range(2))
    c.gpu.read(0, dk.ptr, dv.ptr, 1, 40)
    for buf, src in ((dk, x), (dv, -x[:, ::-1])):
        got = buf.to_numpy(np.float16, x.shape)
        want = values(*quantize(src)).reshape(x.shape)
        np.testing.assert_array_equal(got.astype(np.float64), want)      # exact, NaN included


@pytest.mark.parametrize("d", [64, 256])
def test_read_ranges(hip_ready, d):
    rng = np.random.default_rng(9)
    c = Cache(hip_ready, 2, 2, d, 32, 20, 4, 6)
    c.fill(rng, [70, 1, 0, 33])
    S = 40
    # a window in the middle, one that begins before the first token, one that ends behind the last, an empty slot
    seqs, starts, counts = [0, 3, 0, 2, 9, 1], [21, -5, 60, 0, 0, 0], [40, 12, 40, 7, 3, 1]
    mark = np.full((6, S, 2, d), 11.0, np.float16)
    dk, dv = c.cm.DeviceBuffer.from_numpy(mark), c.cm.DeviceBuffer.from_numpy(mark)
    c.gpu.read(1, dk.ptr, dv.ptr, 6, S, seqs=seqs, starts=starts, counts=counts)
    for is_v, buf in ((0, dk), (1, dv)):
        want = mark.astype(np.float64)
        for b in range(6):
            if seqs[b] >= 4:
                continue
            x = values(*c.cpu.read(1, seqs[b])[is_v]).reshape(-1, 2, d)
            for r in range(counts[b]):
                if 0 <= starts[b] + r < len(x):
                    want[b, r] = x[starts[b] + r]
        np.testing.assert_array_equal(buf.to_numpy(np.float16, mark.shape).astype(np.float64), want)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 2, 3, 8, 17])
def test_decode_lengths(hip_ready, d, G):
    rng = np.random.default_rng(d * 100 + G)
    lens = [1, 15, 16, 17, 31, 33, 64, 150]
    c = Cache(hip_ready, 1, 2, d, 16, 40, 8, 12)
    c.fill(rng, lens)
    q = rng.standard_normal((8, 1, 2 * G, d)).astype(np.float16)
    c.attend(q, range(8), [1] * 8)


@pytest.mark.parametrize("d,ps", [(64, 16), (128, 64), (256, 32), (128, 256)])
@pytest.mark.parametrize("S", [2, 5, 16, 33, 90])
@pytest.mark.parametrize("window,sink,causal", [(0, 0, True), (0, 0, False), (20, 0, True), (31, 5, True), (1, 40, True),
                                                (17, 3, False), (1 << 40, 2, True)])
def test_rows_and_masks(hip_ready, d, ps, S, window, sink, causal):
    rng = np.random.default_rng(S * 7 + d)
    c = Cache(hip_ready, 1, 2, d, ps, 48, 5, 16)
    lens = [S, S + 1, 150, S + 47, 97 if S <= 97 else S]
    c.fill(rng, lens)
    q = rng.standard_normal((5, S, 4, d)).astype(np.float16)
    c.attend(q, [3, 1, 0, 2, 4], [S, S, 0, max(1, S - 1), max(1, S // 2)], window=window, sink=sink, causal=causal,
             stride=4 * d + 16)


@pytest.mark.parametrize("d,G,lens,counts", [(64, 4, [700, 0, 333], [300, 5, 257]), (128, 1, [900, 130], [513, 1]),
                                             (256, 3, [260, 41], [130, 41]), (128, 8, [1500], [40])])
@pytest.mark.parametrize("window,sink,causal,scale", [(0, 0, True, 0.0), (100, 70, True, 0.3), (0, 0, False, -0.2)])
def test_many_rows(hip_ready, d, G, lens, counts, window, sink, causal, scale):
    """Several blocks of query vectors, key ranges that workgroups share, scores far apart, a negative scale."""
    rng = np.random.default_rng(d + G + window)
    c = Cache(hip_ready, 1, 2, d, 32, 80, len(lens), 50)
    c.fill(rng, lens, scale=1.5)
    q = (2 * rng.standard_normal((len(lens), max(counts), 2 * G, d))).astype(np.float16)
    c.attend(q, range(len(lens)), counts, window=window, sink=sink, causal=causal, scale=scale)


@pytest.mark.parametrize("S", [3, 40])
def test_more_rows_than_tokens(hip_ready, S):
    """Rows before the first token: positions below 0, which causal rows see nothing from."""
    rng = np.random.default_rng(S)
    c = Cache(hip_ready, 1, 2, 64, 16, 20, 3, 8)
    c.fill(rng, [2, 30])
    q = rng.standard_normal((3, S, 4, 64)).astype(np.float16)
    c.attend(q, [0, 1, 2], [S, S, S])
    c.attend(q, [0, 1, 2], [S, S, S], causal=False)


def test_offsets_past_32_bits(hip_ready):
    """A pool of 4.9 GB of which only the last pages are used."""
    from cactus_amd.kv4 import CacheDesc
    cm, rng = hip_ready, np.random.default_rng(21)
    H, d, ps, N, n = 8, 256, 256, 8300, 600
    one = Cache(cm, 1, H, d, ps, 4, 1, 4)                     # the same tokens in a small pool
    assert one.extend([0], [n]) == 0
    k, v = kv_rows(rng, 1, n, H, d), kv_rows(rng, 1, n, H, d)
    page = H * ps * d * 9 // 8
    pool = cm.DeviceBuffer(N * page)
    table = np.full((1, 4), -1, np.int32)
    table[0, :3] = [N - 1, 8000, N - 7]
    bufs = [cm.DeviceBuffer.from_numpy(x) for x in (table, np.array([n], np.int32), np.zeros(N, np.int32), np.zeros(4, np.int32))]
    desc = CacheDesc(pages=pool.ptr, table=bufs[0].ptr, lens=bufs[1].ptr, refs=bufs[2].ptr, state=bufs[3].ptr, layers=1,
                     kv_heads=H, head_dim=d, page_size=ps, num_pages=N, max_seqs=1, max_pages=4)
    dk, dv = cm.DeviceBuffer.from_numpy(k), cm.DeviceBuffer.from_numpy(v)
    for c in (desc, one.gpu.desc):
        cm.call("cactus_hip_kv4_append_f16", c.ref, 0, None, None, dk.ptr, dv.ptr, 1, n, H * d, None)
    for S, Hq in ((1, 16), (5, 32), (60, 8)):
        q = rng.standard_normal((1, S, Hq, d)).astype(np.float16)
        dq, outs = cm.DeviceBuffer.from_numpy(q), []
        for c in (desc, one.gpu.desc):
            need = cm.hip().cactus_hip_attention_kv4_workspace(c.ref, 1, S, Hq)
            work, do = cm.DeviceBuffer(need), cm.DeviceBuffer(q.nbytes)
            cm.call("cactus_hip_memset", work.ptr, 0, 4096, None)
            cm.call("cactus_hip_attention_kv4_f16", c.ref, 0, None, None, dq.ptr, Hq * d, do.ptr, 1, S, Hq, 0.0, 0, 0, 1,
                    work.ptr, need, None)
            outs.append(do.to_numpy(np.uint16, q.shape))
        np.testing.assert_array_equal(*outs)                  # the same bits wherever the pages lie
    # pages far up copied far up
    lists = [cm.DeviceBuffer.from_numpy(np.array(x, np.int32)) for x in ([N - 1, 8000], [N - 3, 7999])]
    cm.call("cactus_hip_kv4_copy_pages", desc.ref, lists[0].ptr, lists[1].ptr, 2, None)
    table[0, :2] = [N - 3, 7999]
    bufs[0].upload(table)
    back = [[cm.DeviceBuffer(k.nbytes) for _ in range(2)] for _ in range(2)]
    for c, (bk, bv) in zip((desc, one.gpu.desc), back):
        cm.call("cactus_hip_kv4_read_f16", c.ref, 0, None, None, None, bk.ptr, bv.ptr, 1, n, None)
    for i in range(2):
        np.testing.assert_array_equal(*(b[i].to_numpy(np.uint16, k.shape) for b in back))


@pytest.mark.parametrize("S,Hq", [(70, 8), (60, 32)])
def test_many_rows_past_32_bits(hip_ready, S, Hq):
    """The many-row kernel over pages that begin behind 4 GB of a pool."""
    from cactus_amd.kv4 import CacheDesc
    cm, rng = hip_ready, np.random.default_rng(24)
    H, d, ps, N, n = 8, 256, 256, 8300, 600
    page = H * ps * d * 9 // 8
    ids = [N - 1, 8000, N - 7]
    assert min(ids) * page > 1 << 32
    one = Cache(cm, 1, H, d, ps, 4, 1, 4)                     # the same tokens in a small pool
    assert one.extend([0], [n]) == 0
    pool = cm.DeviceBuffer(N * page)
    bufs = [cm.DeviceBuffer.from_numpy(np.array(x, np.int32)) for x in ([ids + [-1]], [n], [0] * N, [0] * 4)]
    desc = CacheDesc(pages=pool.ptr, table=bufs[0].ptr, lens=bufs[1].ptr, refs=bufs[2].ptr, state=bufs[3].ptr, layers=1,
                     kv_heads=H, head_dim=d, page_size=ps, num_pages=N, max_seqs=1, max_pages=4)
    k, v = (cm.DeviceBuffer.from_numpy(kv_rows(rng, 1, n, H, d)) for _ in range(2))
    q = rng.standard_normal((1, S, Hq, d)).astype(np.float16)
    dq, outs = cm.DeviceBuffer.from_numpy(q), []
    need = cm.hip().cactus_hip_attention_kv4_workspace(desc.ref, 1, S, Hq)
    work = cm.DeviceBuffer(need)
    cm.call("cactus_hip_memset", work.ptr, 0, 4096, None)
    for c in (desc, one.gpu.desc):
        cm.call("cactus_hip_kv4_append_f16", c.ref, 0, None, None, k.ptr, v.ptr, 1, n, H * d, None)
        do = cm.DeviceBuffer.from_numpy(np.full(q.shape, np.float16(np.nan)))
        cm.call("cactus_hip_attention_kv4_f16", c.ref, 0, None, None, dq.ptr, Hq * d, do.ptr, 1, S, Hq, 0.0, 0, 0, 1, work.ptr,
                need, None)
        outs.append(do.to_numpy(np.float16, q.shape))
    assert np.isfinite(outs[0]).all()
    np.testing.assert_array_equal(*outs)


def test_two_streams_at_once(hip_ready):
    """Calls that overlap, with a workspace each, give what they give alone."""
    cm, rng = hip_ready, np.random.default_rng(22)
    c = Cache(cm, 1, 4, 128, 16, 700, 3, 300)
    c.fill(rng, [4000, 333, 2500])
    cases = []
    for S in (1, 7, 50):
        q = rng.standard_normal((3, S, 8, 128)).astype(np.float16)
        need = cm.hip().cactus_hip_attention_kv4_workspace(c.gpu.desc.ref, 3, S, 8)
        alone = c.attend(q, [0, 1, 2], [S] * 3)
        work = [cm.DeviceBuffer(need) for _ in range(2)]
        for w in work:
            cm.call("cactus_hip_memset", w.ptr, 0, 4096, None)
        cases.append((S, cm.DeviceBuffer.from_numpy(q), alone, need, work, [cm.DeviceBuffer(q.nbytes) for _ in range(2)]))
    cm.call("cactus_hip_stream_sync", None)
    streams = [cm.Stream(), cm.Stream()]
    for _ in range(5):
        for S, dq, _, need, work, do in cases:
            for i in range(2):
                cm.call("cactus_hip_attention_kv4_f16", c.gpu.desc.ref, 0, None, None, dq.ptr, 8 * 128, do[i].ptr, 3, S, 8, 0.0,
                        0, 0, 1, work[i].ptr, need, streams[i].handle)
    for s in streams:
        s.sync()
    for S, _, alone, _, _, do in cases:
        for b in do:
            np.testing.assert_array_equal(b.to_numpy(np.float16, alone.shape), alone)


def test_long_decode_and_sharp_softmax(hip_ready):
    rng = np.random.default_rng(3)
    c = Cache(hip_ready, 1, 1, 128, 64, 40, 3, 34)
    c.fill(rng, [2100, 3, 300], scale=2.0)
    q = (4 * rng.standard_normal((3, 1, 4, 128))).astype(np.float16)
    c.attend(q, [0, 1, 2], [1, 1, 1])
    c.attend(q, [0, 0, 2], [1, 1, 1], scale=0.004)          # the same slot twice
    c.attend(np.zeros_like(q), [0, 1, 2], [1, 1, 1])        # a mean
    c.attend(q, [2, -1, 5], [1, 1, 1])                      # slots that do not exist


@pytest.mark.parametrize("d,B,S", [(64, 64, 1), (64, 150, 1), (64, 64, 40), (128, 40, 40), (64, 130, 37), (256, 33, 70)])
def test_many_short_requests(hip_ready, d, B, S):
    """More units than workgroups, more requests than a wave has lanes, some without rows."""
    rng = np.random.default_rng(B + S)
    c = Cache(hip_ready, 1, 8, d, 16, 8 * B, B, 8)
    lens = [int(x) for x in rng.integers(0, 100, B)]
    lens[0], lens[-1] = 0, 100
    c.fill(rng, lens)
    q = rng.standard_normal((B, S, 16, d)).astype(np.float16)
    counts = [int(x) for x in rng.integers(0, S + 1, B)]
    counts[-1] = S
    order = [int(x) for x in rng.permutation(B)]
    c.attend(q, order, counts)
    c.attend(q, order, counts, window=9, sink=3)


@pytest.mark.parametrize("d,B,S,H,longest", [(64, 70, 70, 2, 600), (128, 66, 40, 3, 500), (256, 33, 70, 1, 400),
                                             (64, 150, 2, 2, 900)])
def test_many_requests_whose_units_are_shared(hip_ready, d, B, S, H, longest):
    """More requests, or blocks of query vectors, than a wave has lanes, and units that several workgroups take."""
    rng = np.random.default_rng(B + d)
    c = Cache(hip_ready, 1, H, d, 32, B * (longest // 32 + 1), B, longest // 32 + 1)
    lens = [int(x) for x in rng.integers(0, longest + 1, B)]
    lens[0], lens[1], lens[-1] = 0, 1, longest
    c.fill(rng, lens)
    q = rng.standard_normal((B, S, 2 * H, d)).astype(np.float16)
    counts = [S if b % 3 else int(rng.integers(0, S + 1)) for b in range(B)]
    c.attend(q, [int(x) for x in rng.permutation(B)], counts)
    c.attend(q, range(B), counts, window=200, sink=70)
    c.attend(q, range(B), counts, causal=False)


@pytest.mark.parametrize("d,G,lens", [(128, 2, [9000]), (64, 1, [9000, 130]), (64, 6, [5000]), (256, 1, [9000, 4000, 1])])
def test_parts_joined_in_rounds(hip_ready, d, G, lens):
    """Keys in more parts than the joining takes at a time, in stretches of one or more steps."""
    rng = np.random.default_rng(d + G)
    c = Cache(hip_ready, 1, 2, d, 64, 330, len(lens), 150)
    c.fill(rng, lens)
    q = rng.standard_normal((len(lens), 1, 2 * G, d)).astype(np.float16)
    c.attend(q, range(len(lens)), [1] * len(lens))
    c.attend(q, range(len(lens)), [1] * len(lens), window=5000, sink=200)


@pytest.mark.parametrize("d,S,G", [(64, 1, 1), (128, 1, 2), (256, 1, 2), (64, 5, 3), (128, 9, 2), (256, 4, 4), (64, 80, 1),
                                   (128, 40, 2), (256, 70, 1)])
@pytest.mark.parametrize("size", [0.02, 1e-3])
def test_many_small_weights_beside_a_large_one(hip_ready, d, S, G, size):
    """A first key that takes nearly all the weight and has no value, as attention sinks are: the others' weights,
    2^-17 of its, and their small values keep their bits (2^-17 of the products with the kernels' factors stay above
    2^-14, so that no rounding is absolute but that of the output)."""
    rng = np.random.default_rng(d + S)
    n = 3000
    c = Cache(hip_ready, 1, 1, d, 64, 50, 1, 50)
    assert c.extend([0], [n]) == 0
    k = (0.1 * rng.standard_normal((1, n, 1, d))).astype(np.float16)
    v = (size * (1 + 0.3 * rng.standard_normal((1, n, 1, d)))).astype(np.float16)
    k[..., 0], k[0, 0, 0, 0], v[0, 0] = 0, 12, 0
    c.append(0, [0], [n], k, v)
    q = rng.standard_normal((1, S, G, d)).astype(np.float16)
    q[..., 0] = 8
    c.attend(q, [0], [S], scale=1 / 8, small=False)


@pytest.mark.parametrize("d,S,G", [(64, 1, 1), (128, 1, 2), (256, 1, 2), (64, 5, 3), (128, 9, 2), (256, 4, 4), (64, 80, 1)])
@pytest.mark.parametrize("n,sink,outlier", [(3000, 3, 0), (3000, 3, 1999), (3000, 1500, 0), (3000, 1500, 1501), (200, 3, 0),
                                            (200, 150, 60), (30, 3, 0), (30, 3, 20)])
@pytest.mark.parametrize("size", [0.02, 2.0])
def test_a_large_value_without_weight_leaves_the_others_their_bits(hip_ready, d, S, G, n, sink, outlier, size):
    """As above, and one key with values of up to 60000 whose weight is 2^-100 of the largest: the products of weight and
    value scale that count lie within 2^11 of each other, whatever the scales alone do (an output then is off by the
    products' and its own rounding, 2^-11 each, and 2^-25; that key's share is below 2^-80)."""
    rng = np.random.default_rng(d + S + outlier)
    c = Cache(hip_ready, 1, 1, d, 64, 50, 1, 50)
    assert c.extend([0], [n]) == 0
    k = (0.1 * rng.standard_normal((1, n, 1, d))).astype(np.float16)
    v = (size * (1 + 0.3 * rng.standard_normal((1, n, 1, d)))).astype(np.float16)
    k[..., 0], k[0, sink, 0, 0], k[0, outlier, 0, 0] = 0, 12, -60
    v[0, sink], v[0, outlier] = 0, (60000 * rng.uniform(-1, 1, (1, d))).astype(np.float16)
    c.append(0, [0], [n], k, v)
    S = min(S, n - 4)
    q = rng.standard_normal((1, S, G, d)).astype(np.float16)
    q[..., 0] = 8
    c.attend(q, [0], [S], scale=1 / 8, small=False)


def test_a_query_that_is_not_finite_leaves_the_others(hip_ready):
    rng = np.random.default_rng(23)
    c = Cache(hip_ready, 1, 2, 128, 16, 40, 2, 20)
    c.fill(rng, [300, 40])
    for S in (1, 5, 40):
        q = rng.standard_normal((2, S, 8, 128)).astype(np.float16)
        clean = c.attend(q, [0, 1], [S, S])
        q[0, S // 2, 1, 7], q[1, 0, 6, 100] = np.nan, np.inf
        dq, do = c.cm.DeviceBuffer.from_numpy(q), c.cm.DeviceBuffer(q.nbytes)
        c.gpu.attention(0, dq.ptr, do.ptr, 2, S, 8)
        o = do.to_numpy(np.float16, q.shape)
        o[0, S // 2, 1], o[1, 0, 6] = clean[0, S // 2, 1], clean[1, 0, 6]
        np.testing.assert_array_equal(o, clean)


@pytest.mark.parametrize("ps", [512, 4096])
def test_large_pages(hip_ready, ps):
    rng = np.random.default_rng(ps)
    c = Cache(hip_ready, 2, 2, 64, ps, 6, 3, 2)
    c.fill(rng, [ps + 70, 33])
    c.cpu.fork([0], [2])
    c.gpu.fork([0], [2])
    c.check()
    for S in (1, 4, 70):
        q = rng.standard_normal((3, S, 4, 64)).astype(np.float16)
        c.attend(q, [0, 1, 2], [S, min(S, 33), S], layer=1, window=ps - 40, sink=3)


def test_rows_without_keys_are_zero(hip_ready):
    rng = np.random.default_rng(4)
    c = Cache(hip_ready, 1, 2, 64, 16, 20, 3, 8)
    c.fill(rng, [40], seqs=[1])
    q = rng.standard_normal((2, 3, 4, 64)).astype(np.float16)
    do = c.cm.DeviceBuffer.from_numpy(np.full(q.shape, np.float16(5)))
    dq = c.cm.DeviceBuffer.from_numpy(q)
    c.gpu.attention(0, dq.ptr, do.ptr, 2, 3, 4, seqs=[0, 1])
    o = do.to_numpy(np.float16, q.shape)
    assert (o[0] == 0).all() and np.isfinite(o).all() and (o[1] != 5).all()


@pytest.mark.parametrize("S", [1, 4, 70])
def test_non_finite_keys_reach_only_the_rows_that_see_them(hip_ready, S):
    rng = np.random.default_rng(6)
    c = Cache(hip_ready, 1, 1, 64, 16, 20, 2, 8)
    n = 100
    assert c.extend([0], [n]) == 0
    k, v = kv_rows(rng, 1, n, 1, 64), kv_rows(rng, 1, n, 1, 64)
    k[0, 20, 0, 3] = np.inf        # seen by every row from 20 on
    v[0, 60, 0, 40] = np.nan       # dims 32 to 63 only
    v[0, 98, 0, 2] = np.inf
    c.append(0, [0], [n], k, v)
    q = rng.standard_normal((1, S, 2, 64)).astype(np.float16)
    c.attend(q, [0], [S], window=25)
    c.attend(q, [0], [S], window=5)
    c.attend(q, [0], [S])


def test_pages_that_do_not_exist_are_not_there(hip_ready):
    rng = np.random.default_rng(8)
    c = Cache(hip_ready, 1, 1, 64, 16, 20, 2, 8)
    c.fill(rng, [60, 20])
    whole = c.cpu.table.copy()
    for bad in (-1, 20, 1 << 30, -(1 << 31)):
        c.cpu.table = whole.copy()
        c.cpu.table[:, 1] = bad
        c.gpu._buf["table"].upload(c.cpu.table)
        q = rng.standard_normal((1, 1, 2, 64)).astype(np.float16)
        dq, do = c.cm.DeviceBuffer.from_numpy(q), c.cm.DeviceBuffer(q.nbytes)
        c.gpu.attention(0, dq.ptr, do.ptr, 1, 1, 2, seqs=[0])
        # the same keys without those of the missing page
        c.cpu.table = whole.copy()
        (kc, ks), (vc, vs) = c.cpu.read(0, 0)
        at = np.r_[0:16, 32:60]
        want, tol = attention(q[0], kc[at], ks[at], vc[at], vs[at], 44, 1 / 8, causal=False)
        assert (np.abs(do.to_numpy(np.float16, q.shape)[0] - want) <= tol).all()
        c.gpu.append(0, do.ptr, do.ptr, 1, 1, 64, seqs=[1])        # slot 1's last token stands on it: nothing is written
        np.testing.assert_array_equal(c.pages(), c.cpu.pages)
        dk = c.cm.DeviceBuffer.from_numpy(np.full((60, 64), np.float16(3)))
        c.gpu.read(0, dk.ptr, None, 1, 60, seqs=[0])
        got = dk.to_numpy(np.float16, (60, 64))
        assert (got[16:32] == 3).all()


def leftovers(c, bits, rng):
    """Every page holds other data, as recycled memory does: slot 0's token takes page 0 and is never written."""
    c.cpu.pages[:] = rng.integers(0, 256, c.cpu.pages.shape, np.uint8) if bits is None else bits
    c.put_pages()
    assert c.extend([0], [1]) == 0


# 0x7B bytes: the scale 61280, with codes 3 and -1; 0x70: 8576 (with codes -8 a product of -68608), 0xF3: -15256; random bytes
@pytest.mark.parametrize("bits", [0x7B, 0x70, 0xF3, 0xFB, None])
@pytest.mark.parametrize("d,G,ps", [(64, 2, 16), (128, 4, 64), (256, 3, 256)])
def test_what_unused_page_bytes_hold_reaches_no_row(hip_ready, d, G, ps, bits):
    """Finite scales whose products with a code are beyond FP16, in the rest of a tile, behind the last one and in
    page 0, which stands in for pages that are not there."""
    rng = np.random.default_rng(d)
    c = Cache(hip_ready, 1, 2, d, ps, 90, 6, 1 + 700 // ps)
    leftovers(c, bits, rng)
    lens = [40, 75, 128, 131, 600]
    c.fill(rng, lens, seqs=range(1, 6))
    for S in (1, 9, 40, 70):
        q = rng.standard_normal((5, S, 2 * G, d)).astype(np.float16)
        for window, causal in ((0, True), (30, True), (0, False)):
            c.attend(q, range(1, 6), [min(S, n) for n in lens], window=window, sink=3, causal=causal)


@pytest.mark.parametrize("bits", [0x7B, 0x70, None])
@pytest.mark.parametrize("d,written,more", [(64, 30, 20), (64, 100, 50), (128, 70, 9), (256, 90, 70)])
def test_tokens_that_are_not_written_yet_reach_only_the_rows_that_see_them(hip_ready, d, written, more, bits):
    rng = np.random.default_rng(d + written)
    c = Cache(hip_ready, 1, 1, d, 16, 20, 2, 16)
    leftovers(c, bits, rng)
    c.fill(rng, [written], seqs=[1])
    (kc, ks), (vc, vs) = c.cpu.read(0, 1)
    assert c.extend([1], [more]) == 0
    m = written + more
    q = rng.standard_normal((1, m, 1, d)).astype(np.float16)
    dq, do = c.cm.DeviceBuffer.from_numpy(q), c.cm.DeviceBuffer(q.nbytes)
    c.gpu.attention(0, dq.ptr, do.ptr, 1, m, 1, seqs=[1])
    want, tol = attention(q[0, :written], kc, ks, vc, vs, written, 1 / math.sqrt(d))
    assert (np.abs(do.to_numpy(np.float16, q.shape)[0, :written] - want) <= tol).all()


@pytest.mark.parametrize("d,S", [(64, 1), (64, 12), (64, 80), (128, 33), (256, 70)])
def test_the_largest_values_are_not_cut(hip_ready, d, S):
    """Value groups of up to 65504 (scale 9344) beside ordinary ones; some rows see one such key alone."""
    rng = np.random.default_rng(d + S)
    c = Cache(hip_ready, 1, 1, d, 16, 20, 1, 16)
    n = 150
    assert c.extend([0], [n]) == 0
    k, v = kv_rows(rng, 1, n, 1, d), kv_rows(rng, 1, n, 1, d)
    v[0, ::5] = rng.choice([65504, -65504, 57000, 1], (30, 1, d)).astype(np.float16)
    c.append(0, [0], [n], k, v)
    q = rng.standard_normal((1, S, 2, d)).astype(np.float16)
    c.attend(q, [0], [S])
    c.attend(q, [0], [S], window=1)


# pages of less than a stage's keys and of more, in every kernel of the attention
@pytest.mark.parametrize("d,G,S", [(64, 2, 1), (64, 2, 10), (64, 2, 70), (128, 1, 40), (128, 1, 130), (256, 1, 10), (256, 2, 70)])
@pytest.mark.parametrize("ps,gone", [(16, 1), (32, 3), (64, 0), (256, 1), (256, 2)])
def test_missing_pages_in_every_kernel(hip_ready, d, G, S, ps, gone):
    rng = np.random.default_rng(S + ps + gone)
    n = 570
    c = Cache(hip_ready, 1, 2, d, ps, 60, 2, 600 // ps + 1)
    leftovers(c, 0x7B, rng)
    c.fill(rng, [n], seqs=[1])
    (kc, ks), (vc, vs) = c.cpu.read(0, 1)
    table = c.cpu.table.copy()
    table[1, gone] = (-1, 60, 1 << 30, -(1 << 31))[(S + gone) % 4]
    c.gpu._buf["table"].upload(table)
    q = rng.standard_normal((1, S, 2 * G, d)).astype(np.float16)
    dq, do = c.cm.DeviceBuffer.from_numpy(q), c.cm.DeviceBuffer(q.nbytes)
    for window in (0, 300):
        c.gpu.attention(0, dq.ptr, do.ptr, 1, S, 2 * G, window=window, seqs=[1])
        o = do.to_numpy(np.float16, q.shape)[0]
        for r in range(S):
            at = np.arange(max(0, n - S + r - window) if window else 0, n - S + r + 1)
            at = at[at // ps != gone]
            want, tol = attention(q[0, r:r + 1], kc[at], ks[at], vc[at], vs[at], len(at), 1 / math.sqrt(d), causal=False) \
                if len(at) else (0, 0)
            assert (np.abs(o[r] - want) <= tol).all(), (window, r)


# ------------------------------------------------------------------ pages
def test_extend_fork_free_compact_follow_the_model(hip_ready):
    rng = np.random.default_rng(10)
    c = Cache(hip_ready, 2, 1, 64, 16, 50, 9, 8)
    c.fill(rng, [40, 16, 1, 33, 64], seqs=[0, 2, 3, 5, 8])
    c.check()
    for step in range(40):
        op = rng.integers(0, 5)
        if op == 0:
            n = int(rng.integers(1, 6))
            c.extend([int(s) for s in rng.permutation(9)[:n]], [int(x) for x in rng.integers(0, 40, n)])
        elif op == 1:
            n = int(rng.integers(1, 10))
            src, dst = [int(s) for s in rng.integers(0, 9, n)], [int(s) for s in rng.permutation(9)[:n]]
            want = c.cpu.fork(src, dst)
            c.gpu.fork(src, dst)
            assert c.gpu.status() == want
        elif op == 2:
            seqs = [int(s) for s in rng.integers(0, 9, 2)]
            c.cpu.free(seqs)
            c.gpu.free(seqs)
        elif op == 3:
            c.cpu.compact()
            c.gpu.compact()
        else:
            a = [int(x) for x in rng.permutation(50)[:6]]
            c.cpu.pages[:, a[3:]] = c.cpu.pages[:, a[:3]]
            c.gpu.copy_pages(a[:3], a[3:])
        c.check()


def test_large_pools(hip_ready):
    """More pages than one round of the allocation takes, more than one workgroup counts, and many requests."""
    rng = np.random.default_rng(11)
    c = Cache(hip_ready, 1, 1, 64, 16, 21000, 1500, 900)
    counts = [int(x) for x in rng.integers(0, 160, 1500)]
    counts[7], counts[1400] = 16 * 900, 16 * 900
    assert c.extend(list(range(1500)), counts) == 0
    c.cpu.pages[0, :, 0, 0, :4] = np.arange(21000, dtype=np.int32).view(np.uint8).reshape(-1, 4)
    c.put_pages()
    c.check()
    gone = [int(s) for s in rng.permutation(1500)[:700]] + [7]
    c.cpu.free(gone)
    c.gpu.free(gone)
    c.check()
    dst = list(dict.fromkeys(gone))[:600]
    src = [int(s) for s in rng.integers(0, 1500, len(dst))]
    assert c.cpu.fork(src, dst) == 0
    c.gpu.fork(src, dst)
    c.check()
    c.cpu.compact()
    c.gpu.compact()
    c.check()
    assert c.extend([3, 4], [16 * 300, 100]) == 0
    c.check()


def test_refused_requests_change_nothing(hip_ready):
    rng = np.random.default_rng(12)
    c = Cache(hip_ready, 1, 1, 64, 16, 10, 4, 8)
    c.fill(rng, [40, 17])
    assert c.extend([2, 3], [64, 32]) == 1          # six pages, five free
    assert c.extend([2, 2], [1, 1]) == 2            # named twice
    assert c.extend([2, 4], [1, 1]) == 2            # no such slot
    assert c.extend([2, 3], [1, -1]) == 2
    assert c.extend([2, 0], [1, 200]) == 2          # more than a table row holds
    c.check()
    for src, dst, want in (([0, 1], [2, 2], 2), ([0, -1], [2, 3], 2), ([0, 1], [2, 4], 2)):
        assert c.cpu.fork(src, dst) == want
        c.gpu.fork(src, dst)
        assert c.gpu.status() == want
    c.check()
    assert c.extend([2, 3], [16, 64]) == 0          # the pool is full
    assert c.cpu.fork([0], [3]) == 1
    c.gpu.fork([0], [3])
    # until the status is read, appends write nothing
    k = kv_rows(rng, 1, 1, 1, 64)
    d = c.cm.DeviceBuffer.from_numpy(k)
    c.gpu.append(0, d.ptr, d.ptr, 1, 1, seqs=[0])
    c.check()
    assert c.gpu.status() == 1 and c.gpu.status() == 0
    c.gpu.free([1, 77])
    c.cpu.free([1, 77])
    assert c.gpu.status() == 2
    c.gpu.copy_pages([0, 1, -3], [1, 10, 2])
    c.cpu.pages[:, 1] = c.cpu.pages[:, 0]
    assert c.gpu.status() == 2
    c.check()


def test_nothing_grows_until_the_status_is_read(hip_ready):
    """An append that the status holds back leaves no tokens behind: extend and fork are held back with it."""
    rng = np.random.default_rng(16)
    c = Cache(hip_ready, 2, 1, 64, 16, 12, 4, 8)
    c.fill(rng, [40, 17])
    k = c.cm.DeviceBuffer.from_numpy(kv_rows(rng, 2, 20, 1, 64))
    for set_bit, bit in ((lambda: c.gpu.free([77]), 2), (lambda: c.gpu.copy_pages([0], [12]), 2),
                         (lambda: c.gpu.extend(1, 128, seqs=[3]), 1), (lambda: c.gpu.fork([0, 0], [2, 2]), 2)):
        set_bit()
        c.gpu.extend(2, seqs=[0, 1], counts=[3, 20])
        for layer in range(2):
            c.gpu.append(layer, k.ptr, k.ptr, 2, 20, seqs=[0, 1], counts=[3, 20])
        c.gpu.fork([0, 1], [2, 0])
        c.check()
        assert c.gpu.status() == bit and c.gpu.status() == 0
    # pages are given up in any case, and what follows the reading goes on from there
    c.gpu.free([1, 9])
    c.cpu.free([1])
    c.gpu.compact()
    c.cpu.compact()
    c.check()
    assert c.gpu.status() == 2
    c.fill(rng, [3, 20], seqs=[0, 1])
    assert c.cpu.fork([0, 1], [2, 0]) == 0
    c.gpu.fork([0, 1], [2, 0])
    c.check()
    assert c.gpu.status() == 0


def test_a_captured_step_in_a_full_pool(hip_ready):
    """Replays of extend and append past the last free page, then with pages free but the status not read yet."""
    cm, rng = hip_ready, np.random.default_rng(17)
    c = Cache(cm, 1, 1, 64, 16, 6, 3, 4)
    c.fill(rng, [30, 14, 20])
    stream = cm.Stream()
    st = stream.handle
    kv = [cm.DeviceBuffer(2 * 64 * 2) for _ in range(2)]
    graph = ctypes.c_void_p()
    cm.call("cactus_hip_graph_capture_begin", st)
    cm.call("cactus_hip_kv4_extend", c.gpu.desc.ref, None, None, 2, 1, st)
    cm.call("cactus_hip_kv4_append_f16", c.gpu.desc.ref, 0, None, None, kv[0].ptr, kv[1].ptr, 2, 1, 64, st)
    cm.call("cactus_hip_graph_capture_end", st, ctypes.byref(graph))

    def replay(grows):
        k, v = kv_rows(rng, 2, 1, 1, 64), kv_rows(rng, 2, 1, 1, 64)
        kv[0].upload(k, st), kv[1].upload(v, st)
        cm.call("cactus_hip_graph_launch", graph, st)
        stream.sync()
        if grows:
            assert c.cpu.extend([0, 1], [1, 1]) == 0
            for b in range(2):
                c.cpu.write(0, b, c.cpu.lens[b] - 1, k[b, 0], v[b, 0])
        c.check()

    replay(True)
    replay(True)               # both pages are full now, and one page is free
    replay(False)              # two are needed
    replay(False)
    c.gpu.free([2], stream=st)
    c.cpu.free([2])
    replay(False)              # there would be pages
    assert c.gpu.status(st) == 1
    for _ in range(3):
        replay(True)
    assert c.gpu.status(st) == 0
    cm.call("cactus_hip_graph_destroy", graph)


def test_a_fork_that_a_wrong_free_count_lets_through(hip_ready):
    """state[0] promises a page that is not there: the status says so, and no page is used twice."""
    rng = np.random.default_rng(18)
    c = Cache(hip_ready, 1, 1, 64, 16, 4, 3, 4)
    c.fill(rng, [40, 10])
    before = c.gpu.tables()
    c.gpu._buf["state"].upload(np.array([3, 0, 0, 0], np.int32))
    c.gpu.fork([0], [2])
    assert c.gpu.status() == 1
    after = c.gpu.tables()
    np.testing.assert_array_equal(after["refs"], before["refs"] + [1, 1, 0, 0])
    np.testing.assert_array_equal(after["table"], np.vstack([before["table"][:2], [0, 1, -1, -1]]))
    np.testing.assert_array_equal(c.pages(), c.cpu.pages)


# ------------------------------------------------------------------ together
def test_a_serving_run(hip_ready):
    """Prompts, beams, drafted tokens, conversations that end and a packed pool, every step's attention checked."""
    rng = np.random.default_rng(13)
    H, G, d, layers = 2, 2, 64, 2
    c = Cache(hip_ready, layers, H, d, 16, 60, 8, 20)

    def step(seqs, counts):
        assert c.extend(seqs, counts) == 0
        S = max(counts)
        for layer in range(layers):
            c.append(layer, seqs, counts, kv_rows(rng, len(seqs), S, H, d), kv_rows(rng, len(seqs), S, H, d))
            q = rng.standard_normal((len(seqs), S, H * G, d)).astype(np.float16)
            c.attend(q, seqs, counts, layer, window=int(rng.integers(0, 2)) * 40, sink=4)

    step([0, 1, 5], [75, 33, 120])
    step([0, 1, 5], [1, 1, 1])
    c.cpu.fork([0, 0, 5], [2, 3, 1])
    c.gpu.fork([0, 0, 5], [2, 3, 1])
    for _ in range(3):
        step([0, 1, 2, 3, 5], [1, 4, 1, 1, 2])
    c.cpu.fork([3, 0, 3], [0, 3, 6])
    c.gpu.fork([3, 0, 3], [0, 3, 6])
    step([0, 3, 6], [1, 1, 1])
    c.cpu.free([1, 2])
    c.gpu.free([1, 2])
    c.cpu.compact()
    c.gpu.compact()
    c.check()
    step([0, 3, 5, 6, 7], [1, 1, 1, 1, 50])
    c.check()


def test_a_captured_step(hip_ready):
    """extend, append and attention captured once and replayed, eager work in between; the lengths grow on the device."""
    cm = hip_ready
    rng = np.random.default_rng(14)
    H, G, d, B = 2, 2, 128, 3
    c = Cache(cm, 1, H, d, 16, 60, 4, 16)
    c.fill(rng, [30, 5, 64])
    stream = cm.Stream()
    st = stream.handle
    kv = [cm.DeviceBuffer(B * H * d * 2) for _ in range(2)]
    dq, do = cm.DeviceBuffer(B * H * G * d * 2), cm.DeviceBuffer(B * H * G * d * 2)
    need = cm.hip().cactus_hip_attention_kv4_workspace(c.gpu.desc.ref, B, 1, H * G)
    work = cm.DeviceBuffer(need)
    cm.call("cactus_hip_memset", work.ptr, 0, 4096, st)
    cm.call("cactus_hip_stream_sync", st)
    graph = ctypes.c_void_p()
    cm.call("cactus_hip_graph_capture_begin", st)
    cm.call("cactus_hip_kv4_extend", c.gpu.desc.ref, None, None, B, 1, st)
    cm.call("cactus_hip_kv4_append_f16", c.gpu.desc.ref, 0, None, None, kv[0].ptr, kv[1].ptr, B, 1, H * d, st)
    cm.call("cactus_hip_attention_kv4_f16", c.gpu.desc.ref, 0, None, None, dq.ptr, H * G * d, do.ptr, B, 1, H * G, 0.0, 0, 0,
            1, work.ptr, need, st)
    cm.call("cactus_hip_graph_capture_end", st, ctypes.byref(graph))
    for i in range(20):
        k, v = kv_rows(rng, B, 1, H, d), kv_rows(rng, B, 1, H, d)
        q = rng.standard_normal((B, 1, H * G, d)).astype(np.float16)
        kv[0].upload(k, st), kv[1].upload(v, st), dq.upload(q, st)
        cm.call("cactus_hip_graph_launch", graph, st)
        o = do.to_numpy(np.float16, q.shape, st)
        assert c.cpu.extend([0, 1, 2], [1, 1, 1]) == 0
        for b in range(B):
            c.cpu.write(0, b, c.cpu.lens[b] - 1, k[b, 0], v[b, 0])
            (kc, ks), (vc, vs) = c.cpu.read(0, b)
            want, tol = attention(q[b], kc, ks, vc, vs, len(kc), 1 / math.sqrt(d))
            assert (np.abs(o[b] - want) <= tol).all(), (i, b)
        eager = c.attend(q, [0, 1, 2], [1, 1, 1])          # on the default stream, with a workspace of its own
        np.testing.assert_array_equal(o, eager)
    cm.call("cactus_hip_graph_destroy", graph)
    c.check()


def test_captured_prompts_and_pages(hip_ready):
    """Prompts of 40 rows (the many-row kernel), a fork, an end and a compaction in one graph, replayed with eager calls
    between; graph and eager calls have a workspace each."""
    cm = hip_ready
    rng = np.random.default_rng(15)
    H, G, d, B, S = 2, 2, 64, 2, 40
    c = Cache(cm, 2, H, d, 16, 90, 5, 20)
    c.fill(rng, [30, 130, 20])
    stream = cm.Stream()
    st = stream.handle
    ref = c.gpu.desc.ref
    kv = [cm.DeviceBuffer(B * S * H * d * 2) for _ in range(2)]
    dq, do = cm.DeviceBuffer(B * S * H * G * d * 2), cm.DeviceBuffer(B * S * H * G * d * 2)
    lists = {n: cm.DeviceBuffer.from_numpy(np.array(v, np.int32)) for n, v in
             (("seqs", [1, 3]), ("counts", [40, 33]), ("src", [1, 3]), ("dst", [4, 1]), ("gone", [3, 4]))}
    p = {n: b.ptr for n, b in lists.items()}
    hip = cm.hip()
    need = max(hip.cactus_hip_attention_kv4_workspace(ref, B, S, H * G), hip.cactus_hip_kv4_pages_workspace(ref, 2))
    work = cm.DeviceBuffer(need)
    cm.call("cactus_hip_memset", work.ptr, 0, 4096, st)
    cm.call("cactus_hip_stream_sync", st)
    cm.call("cactus_hip_stream_sync", None)
    graph = ctypes.c_void_p()
    cm.call("cactus_hip_graph_capture_begin", st)
    cm.call("cactus_hip_kv4_extend", ref, p["seqs"], p["counts"], B, 0, st)
    for layer in range(2):
        cm.call("cactus_hip_kv4_append_f16", ref, layer, p["seqs"], p["counts"], kv[0].ptr, kv[1].ptr, B, S, H * d, st)
    cm.call("cactus_hip_attention_kv4_f16", ref, 1, p["seqs"], p["counts"], dq.ptr, H * G * d, do.ptr, B, S, H * G, 0.0, 0, 0, 1,
            work.ptr, need, st)
    cm.call("cactus_hip_kv4_fork", ref, p["src"], p["dst"], 2, work.ptr, need, st)
    cm.call("cactus_hip_kv4_free", ref, p["gone"], 2, st)
    cm.call("cactus_hip_kv4_compact", ref, work.ptr, need, st)
    cm.call("cactus_hip_graph_capture_end", st, ctypes.byref(graph))
    for i in range(4):
        k, v = kv_rows(rng, B, S, H, d), kv_rows(rng, B, S, H, d)
        q = rng.standard_normal((B, S, H * G, d)).astype(np.float16)
        kv[0].upload(k, st), kv[1].upload(v, st), dq.upload(q, st)
        cm.call("cactus_hip_graph_launch", graph, st)
        o = do.to_numpy(np.float16, q.shape, st)
        assert c.cpu.extend([1, 3], [40, 33]) == 0
        for b, (slot, m) in enumerate(((1, 40), (3, 33))):
            for layer in range(2):
                for r in range(m):
                    c.cpu.write(layer, slot, c.cpu.lens[slot] - m + r, k[b, r], v[b, r])
            (kc, ks), (vc, vs) = c.cpu.read(1, slot)
            want, tol = attention(q[b, :m], kc, ks, vc, vs, len(kc), 1 / math.sqrt(d))
            assert (np.abs(o[b, :m] - want) <= tol).all(), (i, b)
        assert c.cpu.fork([1, 3], [4, 1]) == 0
        c.cpu.free([3, 4])
        c.cpu.compact()
        assert c.gpu.status(st) == 0
        c.check()
        c.attend(q, [0, 1], [30, 33], layer=0)          # eager, on the default stream
        cm.call("cactus_hip_stream_sync", None)
    cm.call("cactus_hip_graph_destroy", graph)
