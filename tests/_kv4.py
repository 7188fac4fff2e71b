"""Plain restatement of the paged 4-bit KV cache in numpy, 64 bits: the
quantization, the page layout byte by byte, the page bookkeeping and the
attention, with the error that the kernels' roundings may make."""
import functools
import math

import numpy as np

GROUP, TILE = 32, 16


def bf16(x):
    """fp32 values rounded to bf16 (nearest, ties to even), as fp32."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    b = (b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000
    return b.astype(np.uint32).view(np.float32)


def quantize(x):
    """x [..., d] fp16 -> codes (int) [..., d], scales fp16 [..., d / 32]."""
    g = x.astype(np.float32).reshape(*x.shape[:-1], -1, GROUP)
    bad = ~np.isfinite(g).all(-1)
    amax = np.abs(np.where(bad[..., None], 0, g)).max(-1)
    s = bf16((amax / np.float32(7)).astype(np.float32)).astype(np.float16)
    sf = s.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.rint((np.where(bad[..., None], 0, g) / sf).astype(np.float32))
    c = np.where(sf > 0, np.clip(c, -7, 7), 0).astype(np.int64)
    s = np.where(bad, np.float16(np.nan), s)
    return c.reshape(x.shape), s.astype(np.float16)


def values(codes, scales):
    return codes.reshape(*codes.shape[:-1], codes.shape[-1] // GROUP, GROUP).astype(np.float64) * scales.astype(np.float64)[..., None]


def code_at(d, key, dim, value):
    """(byte, shift) within an 18 d tile of a key's or value's code."""
    if not value:
        p, a, h, t = dim // 64, dim // 32 % 2, dim % 32 // 8, dim % 8
        return h * 2 * d + key * (d // 8) + p * 8 + t, 4 * a
    g, a, x = dim // 32, dim // 16 % 2, dim % 16
    return 9 * d + key // 4 * 2 * d + x * (d // 8) + g * 4 + key % 4, 4 * a


def scale_at(d, key, g, value):
    return (17 if value else 8) * d + 2 * ((key // 4 * (d // 32) + g) * 4 + key % 4)


@functools.lru_cache(None)
def places(d, key, value):
    """Bytes and shifts of a token's codes, and bytes of its scales."""
    at = np.array([code_at(d, key, i, value) for i in range(d)])
    return at[:, 0], at[:, 1], np.array([scale_at(d, key, g, value) for g in range(d // GROUP)])


class Model:
    """A cache on the host: pages as bytes, tables as the header defines them."""

    def __init__(self, layers, kv_heads, head_dim, page_size, num_pages, max_seqs, max_pages, fill=0xFF):
        self.layers, self.H, self.d, self.ps = layers, kv_heads, head_dim, page_size
        self.N, self.max_seqs, self.max_pages = num_pages, max_seqs, max_pages
        self.pages = np.full((layers, num_pages, kv_heads, page_size // TILE, 18 * head_dim), fill, np.uint8)
        self.table = np.full((max_seqs, max_pages), -1, np.int32)
        self.lens = np.zeros(max_seqs, np.int32)
        self.refs = np.zeros(num_pages, np.int32)

    def npages(self, n):
        return -(-n // self.ps)

    def free_pages(self):
        return [int(i) for i in np.flatnonzero(self.refs == 0)]

    def extend(self, seqs, counts):
        free, at = self.free_pages(), 0
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < self.max_seqs for s in seqs) or min(counts, default=0) < 0:
            return 2
        if any(self.lens[s] + c > self.max_pages * self.ps for s, c in zip(seqs, counts)):
            return 2
        if sum(self.npages(self.lens[s] + c) - self.npages(self.lens[s]) for s, c in zip(seqs, counts)) > len(free):
            return 1
        for s, c in zip(seqs, counts):
            for j in range(self.npages(self.lens[s]), self.npages(self.lens[s] + c)):
                self.table[s, j] = free[at]
                self.refs[free[at]] = 1
                at += 1
            self.lens[s] += c
        return 0

    def release(self, s):
        for j in range(self.npages(self.lens[s])):
            self.refs[self.table[s, j]] -= 1
        self.table[s] = -1
        self.lens[s] = 0

    def fork(self, src, dst):
        if len(set(dst)) < len(dst) or any(not 0 <= s < self.max_seqs for s in list(src) + list(dst)):
            return 2
        pairs = [(s, d) for s, d in zip(src, dst) if s != d]
        free = self.free_pages()
        if sum(self.lens[s] % self.ps > 0 for s, _ in pairs) > len(free):
            return 1
        was = [(self.table[s].copy(), int(self.lens[s])) for s, _ in pairs]
        for (row, n), (_, d) in zip(was, pairs):
            for j in range(n // self.ps):
                self.refs[row[j]] += 1
            if n % self.ps:
                new = free.pop(0)
                self.refs[new] = 1
                self.pages[:, new] = self.pages[:, row[n // self.ps]]
                row[n // self.ps] = new
        for (row, n), (_, d) in zip(was, pairs):
            self.release(d)
            self.table[d] = row
            self.lens[d] = n
        return 0

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < self.max_seqs:
                self.release(s)
        return 0 if all(0 <= s < self.max_seqs for s in seqs) else 2

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [i for i in range(live) if self.refs[i] == 0]
        movers = [i for i in range(live, self.N) if self.refs[i] > 0]
        to = {a: b for a, b in zip(movers, holes)}
        for a, b in to.items():
            self.pages[:, b] = self.pages[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(self.max_seqs):
            for j in range(self.npages(self.lens[s])):
                self.table[s, j] = to.get(int(self.table[s, j]), self.table[s, j])

    def write(self, layer, slot, pos, k, v):
        """k, v [H][d] fp16 as the token at `pos`."""
        page = self.pages[layer, self.table[slot, pos // self.ps]]
        tile, key = page[:, pos % self.ps // TILE], pos % TILE
        for x, is_v in ((k, False), (v, True)):
            c, s = quantize(x)
            at, up, sat = places(self.d, key, is_v)
            for shift in (0, 4):                  # the two nibbles of the token's bytes
                mine = up == shift
                keep = tile[:, at[mine]] & (0xF0 if shift == 0 else 0x0F)
                tile[:, at[mine]] = keep | ((c[:, mine] + 8) << shift).astype(np.uint8)
            b = np.ascontiguousarray(s).view(np.uint8).reshape(self.H, -1, 2)
            tile[:, sat], tile[:, sat + 1] = b[..., 0], b[..., 1]

    def read(self, layer, slot, n=None):
        """Codes [n][H][d] and scales [n][H][d / 32] of a slot's keys and values, from the page bytes."""
        n = int(self.lens[slot]) if n is None else n
        if n == 0:
            z, s = np.zeros((0, self.H, self.d)), np.zeros((0, self.H, self.d // GROUP), np.float16)
            return (z, s), (z, s)
        ids = self.table[slot, :self.npages(n)]
        tiles = self.pages[layer, ids].transpose(0, 2, 1, 3).reshape(-1, self.H, 18 * self.d)
        out = []
        for is_v in (False, True):
            at, up, sa = (np.stack(x) for x in zip(*(places(self.d, k, is_v) for k in range(TILE))))
            c = (tiles[:, :, at].astype(np.int64) >> up) % 16 - 8          # [tile][H][key][d]
            raw = np.stack([tiles[:, :, sa], tiles[:, :, sa + 1]], -1)
            s = np.ascontiguousarray(raw).view(np.float16)[..., 0]
            c = c.transpose(0, 2, 1, 3).reshape(-1, self.H, self.d)[:n]
            s = s.transpose(0, 2, 1, 3).reshape(-1, self.H, self.d // GROUP)[:n]
            out.append((c, s))
        return out


def attention(q, kc, ks, vc, vs, n, scale, window=0, sink=0, causal=True, small=True):
    """q [m][Hq][d] of the rows at positions n - m to n - 1 over n tokens' codes and scales.
    -> (o [m][Hq][d] in 64 bits, the largest error that the kernel may make in each output).

    The error, with e = 2^-24 for FP32 and 2^-11 for FP16 (half a step relative
    to the value; 2^-25 absolute below FP16's normal range):
      * the output is rounded to FP16: 2^-11 |o| + 2^-25;
      * the weight p s of a key and group is rounded to FP16: 2^-11 sum p |v| / L,
        and 2^-25 |code| / L where p s < 2^-14 (p <= 1 is relative to the maximum;
        not with small = False, for weights that the kernels lift above that);
      * a score is a sum of d products of |q| and at most 16 s (code + 8, and the
        8 that comes off): (d + 16) e scale sum |q| 16 s, its product with the
        scale and the difference from the maximum 4 e (|x| + |max|), the power of two 4 e
        relative; a weight that is off by w moves the output by at most
        p w (|v| + |o|) / L;
      * the FP32 sums of n weights and of n products of at most 16 p s:
        (n + 64) e (|o| + sum p 16 s / L), and twice more for the joining of
        partial sums.
    """
    m, Hq, d = q.shape
    H = kc.shape[1]
    G = Hq // H
    k, v = values(kc, ks).reshape(n, H, d), values(vc, vs).reshape(n, H, d)
    k16 = np.repeat(16 * ks.astype(np.float64), GROUP, -1)
    v16 = np.repeat(16 * vs.astype(np.float64), GROUP, -1)
    o, tol = np.zeros((m, Hq, d)), np.full((m, Hq, d), 2.0 ** -25)
    pos, j = np.arange(n - m, n)[:, None], np.arange(n)[None]
    seen = np.broadcast_to((j <= pos) if causal else np.ones_like(j, bool), (m, n))
    if window:
        seen = seen & ((pos - j <= window) | (j < sink))
    seen = seen & (pos >= -(1 << 40))
    e = 2.0 ** -24
    for h in range(Hq):
        kh, vh, vch = k[:, h // G], v[:, h // G], np.abs(vc[:, h // G])
        qh = q[:, h].astype(np.float64)
        x = np.where(seen, qh @ kh.T * scale, -np.inf)
        err = np.where(seen, (d + 16) * e * abs(scale) * (np.abs(qh) @ k16[:, h // G].T), 0)
        bad = np.isnan(x).any(1)                       # rows that see a key that reads as NaN
        mx = np.where(np.isfinite(x), x, -np.inf).max(1, initial=-np.inf)
        some = (mx > -np.inf) & ~bad
        base = np.where(some, mx, 0)[:, None]
        p = np.where(seen & some[:, None], np.exp(np.where(seen, x, -np.inf) - base), 0)
        L = np.where(some, p.sum(1), 1)[:, None]
        # a value that reads as NaN does so in its own dims, for the rows that see its key
        nan = np.isnan(vh)
        hit = seen.astype(np.float64) @ nan > 0
        vz, v16z = np.where(nan, 0, vh), np.where(np.isnan(v16[:, h // G]), 0, v16[:, h // G])
        av = np.abs(vz)
        oh = p @ vz / L
        ao = np.abs(oh)
        w = err + err.max(1, initial=0)[:, None] + 4 * e * (np.abs(np.where(seen, x, 0)) + np.abs(base)) + 4 * e
        t = 2.0 ** -25 + 2.0 ** -11 * ao + 2.0 ** -11 * (p @ av) / L
        for g in range(d // GROUP if small else 0):
            s = slice(g * GROUP, (g + 1) * GROUP)
            tiny = seen & (p * v16z[:, g * GROUP] / 16 < 2.0 ** -14)
            t[:, s] += 2.0 ** -25 * (tiny @ vch[:, s]) / L
        pw = p * np.where(np.isnan(w), 0, w)
        t += (pw @ av + pw.sum(1)[:, None] * ao) / L
        t += 3 * (seen.sum(1)[:, None] + 64) * e * (ao + p @ v16z / L)
        o[:, h] = np.where(bad[:, None] | (hit & (seen.any(1)[:, None])), np.nan, np.where(some[:, None], oh, 0))
        tol[:, h] = t
    return o, tol
