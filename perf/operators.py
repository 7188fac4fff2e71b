"""Workloads of the paged 4-bit KV cache (include/cactus_hip.h, the
cactus_hip_kv4_* and cactus_hip_attention_kv4_* entry points).

Each case is a dict of plain values with a "kind":

  append     new FP16 key and value rows quantized into the pages of their
             sequences, and read back as the values the pages now hold
  attention  one layer's attention of each sequence's newest rows over its
             pages: one row (decode), a few (verified drafts), many (prefill)
  fork       sequences take over other sequences' tokens: full pages shared,
             the partly filled last page copied in every layer
  compact    some sequences freed, then the live pages moved to the front
  copy       whole pages copied in every layer

The plain forms are torch operations in 32 bits on the same pages; page
bookkeeping and page bytes are whole numbers and have to be equal.
"""
import math

import torch

own = False

DEV = "cuda"
GROUP = 32   # dims that share a scale
TILE = 16    # keys of a tile


def listed():
    return [
        # a decode step of 64 conversations: one new row each, Qwen3-0.6B's KV heads
        {"name": "append_step", "kind": "append", "B": 64, "S": 1, "len": 4096, "ragged": True, "Hkv": 8, "d": 128, "ps": 64},
        # one layer of four prompts of different lengths, right-padded to the longest
        {"name": "append_prompts", "kind": "append", "B": 4, "S": 2048, "len": 2500, "ragged": True, "Hkv": 8, "d": 128,
         "ps": 64},
        # the first tokens of an answer from a small model (one KV head of 256 dims): all latency
        {"name": "attn_57", "kind": "attention", "B": 1, "S": 1, "len": 57, "ragged": False, "Hq": 4, "Hkv": 1, "d": 256,
         "ps": 16, "window": 0, "sink": 0, "causal": True},
        # one decode step late in a long conversation, Qwen3-0.6B's heads
        {"name": "attn_4096", "kind": "attention", "B": 1, "S": 1, "len": 4096, "ragged": False, "Hq": 16, "Hkv": 8, "d": 128,
         "ps": 64, "window": 0, "sink": 0, "causal": True},
        # a decode step of 32 conversations of very different lengths
        {"name": "attn_batch_32", "kind": "attention", "B": 32, "S": 1, "len": 24000, "ragged": True, "Hq": 32, "Hkv": 8,
         "d": 128, "ps": 64, "window": 0, "sink": 0, "causal": True},
        # eight sequences verify up to five drafted tokens each, under a sliding window with sinks, 64-dim heads
        {"name": "attn_verify_5", "kind": "attention", "B": 8, "S": 5, "len": 9001, "ragged": True, "Hq": 32, "Hkv": 8, "d": 64,
         "ps": 32, "window": 4095, "sink": 4, "causal": True},
        # a prefill chunk of odd length behind 3000 tokens
        {"name": "prefill_333", "kind": "attention", "B": 1, "S": 333, "len": 3333, "ragged": False, "Hq": 16, "Hkv": 8,
         "d": 128, "ps": 64, "window": 0, "sink": 0, "causal": True},
        # a large prefill chunk of a long document
        {"name": "prefill_2048", "kind": "attention", "B": 1, "S": 2048, "len": 16384, "ragged": False, "Hq": 32, "Hkv": 8,
         "d": 128, "ps": 128, "window": 0, "sink": 0, "causal": True},
        # a beam search step: 16 beams re-ordered among themselves, 28 layers
        {"name": "fork_beams", "kind": "fork", "seqs": 16, "pairs": 16, "len": 900, "layers": 28, "Hkv": 8, "d": 128, "ps": 64},
        # one system prompt handed to 48 new conversations, short pages
        {"name": "fork_prompt", "kind": "fork", "seqs": 50, "pairs": 48, "len": 2000, "layers": 12, "Hkv": 8, "d": 64, "ps": 32},
        # a third of the conversations end and the pool is packed
        {"name": "compact_pool", "kind": "compact", "seqs": 48, "gone": 16, "len": 1500, "layers": 28, "Hkv": 8, "d": 128,
         "ps": 64},
        # pages moved by a caller that keeps its own tables
        {"name": "copy_pages", "kind": "copy", "pages": 75, "moved": 31, "layers": 18, "Hkv": 1, "d": 256, "ps": 64},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, round(v / step) * step)))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "fork", "compact", "copy"])
    d, ps = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 64, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    if kind == "append":
        S = rng.choice([1, _log(rng, 2, 2048)])
        B = _log(rng, 1, 64 if S == 1 else max(1, min(16, 8192 // S)))
        return {"kind": kind, "B": B, "S": S, "len": S + _log(rng, 1, 4000), "ragged": rng.random() < 0.7, "Hkv": Hkv, "d": d,
                "ps": ps}
    if kind == "attention":
        S = rng.choice([1, 1, 1, _log(rng, 2, 12), _log(rng, 13, 1024)])
        n = _log(rng, 16, 24000)
        B = _log(rng, 1, max(1, min(48, 200000 // n, 4096 // S)))
        w = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        Hq = Hkv * rng.choice([1, 2, 3, 4, 8])
        n = min(n, 10 ** 11 // (B * S * Hq * d))
        return {"kind": kind, "B": B, "S": S, "len": S + n, "ragged": rng.random() < 0.7, "Hq": Hq, "Hkv": Hkv, "d": d,
                "ps": ps, "window": w, "sink": rng.choice([0, 4, 19]) if w else 0, "causal": rng.random() < 0.85}
    layers = rng.randint(1, 24)
    if kind == "fork":
        seqs = rng.randint(2, 40)
        return {"kind": kind, "seqs": seqs, "pairs": rng.randint(1, seqs), "len": _log(rng, 20, 1000), "layers": layers,
                "Hkv": Hkv, "d": d, "ps": min(ps, 64)}
    if kind == "compact":
        seqs = rng.randint(3, 40)
        return {"kind": kind, "seqs": seqs, "gone": rng.randint(1, seqs - 1), "len": _log(rng, 20, 1000), "layers": layers,
                "Hkv": Hkv, "d": d, "ps": min(ps, 64)}
    pages = rng.randint(4, 150)
    return {"kind": kind, "pages": pages, "moved": rng.randint(1, pages // 2), "layers": layers, "Hkv": Hkv, "d": d,
            "ps": min(ps, 64)}


# ------------------------------------------------------------------ shapes
def _spread(n, lo, hi):
    """n lengths between lo and hi, the same ones for a case, the last one hi."""
    return [lo + round((hi - lo) * math.modf((i + 1) * 0.6180339887)[0]) for i in range(n - 1)] + [hi]


def _rows(c):
    """New rows and length of each sequence of an append or attention case."""
    counts = [c["S"]] * c["B"]
    lens = [c["len"]] * c["B"]
    if c["ragged"]:
        counts = _spread(c["B"], max(1, c["S"] // 3), c["S"])
        lens = _spread(c["B"], max(c["S"], c["len"] // 16), c["len"])
    return counts, lens


def _visible(c, p, n):
    """Keys that a row at position p of a sequence of n tokens sees."""
    top = min(p + 1, n) if c["causal"] else n
    if not c["window"]:
        return top
    lo = max(0, p - c["window"])
    return top - lo + min(c["sink"], lo) if top > lo else min(c["sink"], top)


def _page_bytes(c):
    return c["Hkv"] * c["ps"] * 9 * c["d"] // 8


def work(case):
    c = case
    if c["kind"] == "append":
        values = sum(_rows(c)[0]) * c["Hkv"] * c["d"] * 2
        # FP16 rows in, codes and scales out, and back: codes and scales in, FP16 rows out
        return {"bytes": 2 * (2 * values + values * 9 // 16), "flops": 4 * values}
    if c["kind"] == "attention":
        keys = pairs = rows = 0
        for m, n in zip(*_rows(c)):
            rows += m
            seen = [_visible(c, n - m + r, n) for r in range(m)]
            pairs += sum(seen)
            # the union of the rows' keys: the last row's, and what the first row's window reaches further back
            keys += min(n, max(seen[-1], seen[0] if c["window"] else 0) + (m - 1 if c["window"] else 0))
        return {"bytes": keys * c["Hkv"] * 9 * c["d"] // 8 + 4 * rows * c["Hq"] * c["d"], "flops": 4 * pairs * c["Hq"] * c["d"]}
    if c["kind"] == "copy":
        moved = c["moved"]
    else:
        moved = _bookkeeping(c)["moved"]
    return {"bytes": 2 * moved * c["layers"] * _page_bytes(c), "flops": 0}


# ------------------------------------------------------------------ inputs
def _bookkeeping(c):
    """Tables of a fork or compact case as lists, before the call, and how many pages the call has to copy."""
    ps, n = c["ps"], c["seqs"]
    lens = _spread(n, max(1, c["len"] // 2), c["len"])
    if c["kind"] == "fork" and c["pairs"] < c["seqs"]:
        # the slots behind the sources hold nothing yet, or a short stale sequence
        for i in range(n - c["pairs"], n):
            lens[i] = 0 if i % 3 else min(lens[i], ps + 1)
    need = [-(-v // ps) for v in lens]
    total = sum(need)
    pages = total + c.get("pairs", 0) + 7
    # a pool in use: the sequences' pages interleaved, a few pages free in between
    step = next(k for k in (17, 19, 23, 29, 31, 37, 41) if math.gcd(k, pages) == 1)
    order = [(i * step) % pages for i in range(pages)]
    table, at = [], 0
    for m in need:
        table.append(order[at:at + m])
        at += m
    out = {"lens": lens, "table": table, "pages": pages, "max_pages": max(max(need), -(-c["len"] // ps)) + 1}
    if c["kind"] == "fork":
        dst = list(range(n - c["pairs"], n))
        if c["pairs"] == n:      # beams: every slot takes another's tokens, some stay
            src = [(i * 5 + 2) // 2 % n for i in range(n)]
        else:
            src = [i % (n - c["pairs"]) for i in range(c["pairs"])]
        out.update(src=src, dst=dst, moved=sum(1 for a, b in zip(src, dst) if a != b and lens[a] % ps))
    else:
        gone = [(i * 7 + 3) % n for i in range(n)]
        gone = list(dict.fromkeys(gone + list(range(n))))[:c["gone"]]
        left = [p for i, t in enumerate(table) if i not in gone for p in t]
        out.update(gone=gone, moved=sum(p >= len(left) for p in left))
    return out


def _quantize(x):
    """Codes + 8 and scales of the last dimension's groups of 32: the scale is max|x| / 7 rounded to 8 significant
    bits, so that code * scale is an exact FP16 value."""
    x = x.float().view(*x.shape[:-1], -1, GROUP)
    s = (x.abs().amax(-1, keepdim=True) / 7).bfloat16().half()
    c = torch.where(s > 0, torch.round(x / s.float()), torch.zeros_like(x)).clamp(-7, 7)
    return (c + 8).to(torch.uint8).flatten(-2), s.squeeze(-1)


def _tiles(k, v):
    """Tiles of keys and values [T][Hkv][d] (T a multiple of 16): uint8 [T / 16][Hkv][18 d], the layout of the pages."""
    T, H, d = k.shape
    n, parts = T // TILE, []
    for x, key in ((k, True), (v, False)):
        u, s = _quantize(x)
        if key:    # [n][key][H][slab][half][h][t] -> [n][H][h][key][slab][t], the halves in one byte
            u = u.view(n, TILE, H, d // 64, 2, 4, 8)
            b = (u[:, :, :, :, 0] | (u[:, :, :, :, 1] << 4)).permute(0, 2, 4, 1, 3, 5)
        else:      # [n][h][i][H][group][half][x] -> [n][H][h][x][group][i]
            u = u.view(n, 4, 4, H, d // 32, 2, 16)
            b = (u[:, :, :, :, :, 0] | (u[:, :, :, :, :, 1] << 4)).permute(0, 3, 1, 5, 4, 2)
        # scales [n][h][i][H][group] -> [n][H][h][group][i]
        s = s.view(n, 4, 4, H, d // GROUP).permute(0, 3, 1, 4, 2).contiguous()
        parts += [b.reshape(n, H, 8 * d), s.view(torch.uint8).reshape(n, H, d)]
    return torch.cat(parts, -1)


def _untile(t, d):
    """The values that tiles [n][Hkv][18 d] stand for, in float: keys and values [n * 16][Hkv][d]."""
    n, H = t.shape[:2]
    out = []
    for at, key in ((0, True), (9 * d, False)):
        b = t[..., at:at + 8 * d]
        s = t[..., at + 8 * d:at + 9 * d].contiguous().view(torch.float16).float().view(n, H, 4, d // GROUP, 4)
        s = s.permute(0, 2, 4, 1, 3).reshape(n, TILE, H, d // GROUP, 1)
        u = torch.stack((b & 15, b >> 4))
        if key:
            u = u.view(2, n, H, 4, TILE, d // 64, 8).permute(1, 4, 2, 5, 0, 3, 6)
        else:
            u = u.view(2, n, H, 4, 16, d // 32, 4).permute(1, 3, 6, 2, 5, 0, 4)
        out.append(((u.reshape(n, TILE, H, d // GROUP, GROUP).float() - 8) * s).view(n * TILE, H, d))
    return out


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _kv(g, T, H, d):
    """Keys with a few channels larger than the rest and offset, as after rotary positions; values around zero."""
    k = torch.randn(T, H, d, generator=g, device=DEV)
    k *= 1 + 3 * (torch.rand(H, d, generator=g, device=DEV) > 0.95)
    k += 0.5 * torch.randn(H, d, generator=g, device=DEV)
    return k.half(), torch.randn(T, H, d, generator=g, device=DEV).half()


def _inputs(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    ps = c["ps"]
    shape = {"kv_heads": c["Hkv"], "head_dim": c["d"], "page_size": ps}
    if c["kind"] in ("append", "attention"):
        counts, lens = _rows(c)
        need = [-(-n // ps) for n in lens]
        most, pages = max(need) + 1, sum(need) + 5
        order = torch.randperm(pages, generator=g, device=DEV).int()
        table = torch.full((c["B"], most), -1, dtype=torch.int32, device=DEV)
        refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = order[at:at + m]
            at += m
        refs[order[:at].long()] = 1
        # each sequence's tokens, padded to whole pages
        if c["kind"] == "attention":
            k, v = _kv(g, at * ps, c["Hkv"], c["d"])
            tiles = _tiles(k, v).view(at, ps // TILE, c["Hkv"], 18 * c["d"]).transpose(1, 2)
            data = torch.zeros(1, pages, c["Hkv"], ps // TILE, 18 * c["d"], dtype=torch.uint8, device=DEV)
            data[0, order[:at].long()] = tiles
            s = {"q": (1.5 * torch.randn(c["B"], c["S"], c["Hq"], c["d"], generator=g, device=DEV)).half()}
            s["o"] = torch.zeros_like(s["q"])
        else:
            # a pool in use holds older tokens
            data = torch.randint(0, 256, (1, pages, c["Hkv"], ps // TILE, 18 * c["d"]), generator=g, device=DEV, dtype=torch.uint8)
            k, v = _kv(g, c["B"] * c["S"], c["Hkv"], c["d"])
            s = {"k": k.view(c["B"], c["S"], c["Hkv"], c["d"]), "v": v.view(c["B"], c["S"], c["Hkv"], c["d"])}
            s["k_out"], s["v_out"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        s.update(pages=data, table=table, lens=_ints(lens), refs=refs, counts=_ints(counts), state=_ints([5, 0, 0, 0]))
        shape.update(layers=1, num_pages=pages, max_seqs=c["B"], max_pages=most)
        return s, shape
    if c["kind"] == "copy":
        pages = c["pages"]
        order = torch.randperm(pages, generator=g, device=DEV).int()
        s = {"src": order[:c["moved"]].contiguous(), "dst": order[c["moved"]:2 * c["moved"]].contiguous(),
             "table": _ints([[-1]]), "lens": _ints([0]), "refs": torch.zeros(pages, dtype=torch.int32, device=DEV),
             "state": _ints([pages, 0, 0, 0])}
        shape.update(layers=c["layers"], num_pages=pages, max_seqs=1, max_pages=1)
    else:
        k = _bookkeeping(c)
        pages, n, most = k["pages"], c["seqs"], k["max_pages"]
        # which page stands where goes by the seed
        name = torch.randperm(pages, generator=g, device=DEV).int()
        if c["kind"] == "compact":      # the pages to move are the same number for every seed
            name = torch.arange(pages, device=DEV, dtype=torch.int32)
        flat = [p for t in k["table"] for p in t]
        rows = [i for i, t in enumerate(k["table"]) for _ in t]
        cols = [j for t in k["table"] for j in range(len(t))]
        table = torch.full((n, most), -1, dtype=torch.int32, device=DEV)
        ids = name[_ints(flat).long()]
        table[_ints(rows).long(), _ints(cols).long()] = ids
        refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        refs[ids.long()] = 1
        # tables, lengths and reference counts in one buffer, and a copy of it that each pass starts from
        saved = torch.cat([table.view(-1), _ints(k["lens"]), refs, _ints([pages - len(flat), 0, 0, 0])])
        book = saved.clone()
        a, b = n * most, n * most + n
        s = {"saved": saved, "book": book, "table": book[:a].view(n, most), "lens": book[a:b], "refs": book[b:b + pages],
             "state": book[b + pages:]}
        if c["kind"] == "fork":
            s.update(src=_ints(k["src"]), dst=_ints(k["dst"]))
        else:
            s.update(gone=_ints(k["gone"]))
        shape.update(layers=c["layers"], num_pages=pages, max_seqs=n, max_pages=most)
    s["pages"] = torch.randint(0, 256, (c["layers"], pages, c["Hkv"], ps // TILE, 18 * c["d"]), generator=g, device=DEV,
                               dtype=torch.uint8)
    return s, shape


def prepare(case, seed):
    """The cache with its tables, the inputs and the output buffers, as a serving program holds them."""
    s, shape = _inputs(case, seed)
    s.update(case=case, shape=shape)
    # scratch memory of the calls: counters and partial sums (zero before the first call), page lists
    s["workspace"] = torch.zeros(128 << 20, dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------ plain forms
def _positions(s):
    """Position of each batch row's rows in its sequence, and which rows are there: [B][S]."""
    r = torch.arange(s["case"]["S"], device=DEV)
    m = s["counts"].long()[:, None]
    return s["lens"].long()[:, None] - m + r, r < m


def _plain_append(s):
    c = s["case"]
    B, S, H, d, ps = c["B"], c["S"], c["Hkv"], c["d"], c["ps"]
    pos, there = _positions(s)
    b, r = there.nonzero(as_tuple=True)
    p = pos[b, r]
    page = s["table"].long()[b, p // ps]
    tile, key = p % ps // TILE, p % TILE
    flat = s["pages"][0].view(-1, 18 * d)                               # [page, head, tile] rows
    row = (page[:, None] * H + torch.arange(H, device=DEV)) * (ps // TILE) + tile[:, None]      # [n][H]
    for at, x, out, is_key in ((0, s["k"], s["k_out"], True), (9 * d, s["v"], s["v_out"], False)):
        u, sc = _quantize(x[b, r])                                      # [n][H][d], [n][H][d / 32]
        if is_key:
            u = u.view(-1, H, d // 64, 2, 4, 8)
            by = (u[:, :, :, 0] | (u[:, :, :, 1] << 4)).permute(0, 1, 3, 2, 4).reshape(-1, H, d // 2)   # [h][slab][t]
            i = torch.arange(d // 2, device=DEV)
            col = i // (d // 8) * (2 * d) + i % (d // 8) + key[:, None] * (d // 8)
        else:
            u = u.view(-1, H, d // 32, 2, 16)
            by = (u[:, :, :, 0] | (u[:, :, :, 1] << 4)).transpose(2, 3).reshape(-1, H, d // 2)          # [x][group]
            col = (key // 4 * (2 * d) + key % 4)[:, None] + torch.arange(d // 2, device=DEV) * 4
        flat[row[:, :, None], at + col[:, None]] = by
        g = torch.arange(d // GROUP, device=DEV)
        half = (key // 4 * (d // 8) + key % 4)[:, None] + g * 4         # [n][groups], in FP16 values
        flat.view(torch.float16)[row[:, :, None], (at + 8 * d) // 2 + half[:, None]] = sc
        # and back
        by = flat[row[:, :, None], at + col[:, None]]
        sc = flat.view(torch.float16)[row[:, :, None], (at + 8 * d) // 2 + half[:, None]].float()
        u = torch.stack((by & 15, by >> 4))
        if is_key:
            u = u.view(2, -1, H, 4, d // 64, 8).permute(1, 2, 4, 0, 3, 5)
        else:
            u = u.view(2, -1, H, 16, d // 32).permute(1, 2, 4, 0, 3)
        val = (u.reshape(-1, H, d // GROUP, GROUP).float() - 8) * sc[..., None]
        out[b, r] = val.reshape(-1, H, d).half()
    return {"k": s["k_out"], "v": s["v_out"]}


def _plain_attention(s):
    c = s["case"]
    B, S, H, d, ps, G = c["B"], c["S"], c["Hkv"], c["d"], c["ps"], c["Hq"] // c["Hkv"]
    n = s["table"].shape[1] - 1
    ids = s["table"][:, :n].long().clamp_min(0)
    t = s["pages"][0][ids.view(-1)].transpose(1, 2).reshape(B * n * ps // TILE, H, 18 * d)
    k, v = (x.view(B, n * ps, H, d).transpose(1, 2) for x in _untile(t, d))                         # [B][H][T][d]
    q = s["q"].float().view(B, S, H, G, d).transpose(1, 2).reshape(B, H, S * G, d)
    pos, there = _positions(s)
    j = torch.arange(n * ps, device=DEV)
    p = pos[:, :, None]
    seen = (j < s["lens"].long()[:, None, None]) & (p >= 0)
    if c["causal"]:
        seen = seen & (j <= p)
    if c["window"]:
        seen = seen & ((p - j <= c["window"]) | (j < c["sink"]))
    seen = seen.repeat_interleave(G, 1)[:, None]                                                    # [B][1][S * G][T]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1 / math.sqrt(d))
    x = torch.where(seen, x, torch.full_like(x[:1, :1, :1, :1], -math.inf))
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    o = torch.matmul(x, v.contiguous()) / x.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.view(B, H, S, G, d).transpose(1, 2).reshape(B, S, c["Hq"], d).half()
    s["o"][there] = o[there]
    return s["o"]


def _result(s):
    return {"pages": s["pages"], "table": s["table"], "lens": s["lens"], "refs": s["refs"], "free": s["state"][:1]}


def _plain_fork(s):
    ps = s["case"]["ps"]
    s["book"].copy_(s["saved"])
    table, lens, refs, pages = s["table"], s["lens"], s["refs"], s["pages"]
    src, dst = s["src"].long(), s["dst"].long()
    other = src != dst
    src, dst = src[other], dst[other]
    j = torch.arange(table.shape[1], device=DEV)
    rows, n = table[src].long(), lens[src].long()
    old, m = table[dst].long(), lens[dst].long()
    b = (n % ps > 0).nonzero()[:, 0]
    new = (refs == 0).nonzero()[:b.numel(), 0]
    tail = rows[b, n[b] // ps]
    whole = rows[j < (n // ps)[:, None]]
    gone = old[j < (-(-m // ps))[:, None]]
    refs.index_add_(0, whole, torch.ones_like(whole, dtype=torch.int32))
    refs.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    refs[new] = 1
    rows = torch.where(j < (n // ps)[:, None], rows, torch.full_like(rows, -1))
    rows[b, n[b] // ps] = new
    table[dst] = rows.int()
    lens[dst] = n.int()
    pages[:, new] = pages[:, tail]
    s["state"][0] = (refs == 0).sum()
    return _result(s)


def _plain_compact(s):
    ps = s["case"]["ps"]
    s["book"].copy_(s["saved"])
    table, lens, refs, pages = s["table"], s["lens"], s["refs"], s["pages"]
    gone = s["gone"].long()
    j = torch.arange(table.shape[1], device=DEV)
    old = table[gone].long()[j < (-(-lens[gone].long() // ps))[:, None]]
    refs.index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    table[gone] = -1
    lens[gone] = 0
    live = (refs > 0).sum()
    at = torch.arange(refs.numel(), device=DEV)
    hole = ((refs == 0) & (at < live)).nonzero()[:, 0]
    mover = ((refs > 0) & (at >= live)).nonzero()[:, 0]
    to = at.clone()
    to[mover] = hole
    pages[:, hole] = pages[:, mover]
    refs[hole] = refs[mover]
    refs[mover] = 0
    table.copy_(torch.where(table >= 0, to[table.long().clamp_min(0)].int(), table))
    s["state"][0] = refs.numel() - live
    return _result(s)


def _plain_copy(s):
    s["pages"][:, s["dst"].long()] = s["pages"][:, s["src"].long()]
    return s["pages"]


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    import cactus_amd as cm
    from cactus_amd.kv4 import CacheDesc
    c = s["case"]
    if "cache" not in s:      # the handle that a program keeps
        s["cache"] = CacheDesc(pages=s["pages"].data_ptr(), table=s["table"].data_ptr(), lens=s["lens"].data_ptr(),
                               refs=s["refs"].data_ptr(), state=s["state"].data_ptr(), **s["shape"])
    cache, work_at, work_size = s["cache"].ref, s["workspace"].data_ptr(), s["workspace"].numel()
    if c["kind"] == "append":
        cm.call("cactus_hip_kv4_append_f16", cache, 0, None, s["counts"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                c["B"], c["S"], c["Hkv"] * c["d"], None)
        cm.call("cactus_hip_kv4_read_f16", cache, 0, None, None, s["counts"].data_ptr(), s["k_out"].data_ptr(),
                s["v_out"].data_ptr(), c["B"], c["S"], None)
        return {"k": s["k_out"], "v": s["v_out"]}
    if c["kind"] == "attention":
        cm.call("cactus_hip_attention_kv4_f16", cache, 0, None, s["counts"].data_ptr(), s["q"].data_ptr(), c["Hq"] * c["d"],
                s["o"].data_ptr(), c["B"], c["S"], c["Hq"], 1 / math.sqrt(c["d"]), c["window"], c["sink"], int(c["causal"]),
                work_at, work_size, None)
        return s["o"]
    if c["kind"] == "copy":
        cm.call("cactus_hip_kv4_copy_pages", cache, s["src"].data_ptr(), s["dst"].data_ptr(), c["moved"], None)
        return s["pages"]
    s["book"].copy_(s["saved"])
    if c["kind"] == "fork":
        cm.call("cactus_hip_kv4_fork", cache, s["src"].data_ptr(), s["dst"].data_ptr(), c["pairs"], work_at, work_size, None)
    else:
        cm.call("cactus_hip_kv4_free", cache, s["gone"].data_ptr(), c["gone"], None)
        cm.call("cactus_hip_kv4_compact", cache, work_at, work_size, None)
    return _result(s)


def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "attention": _plain_attention, "fork": _plain_fork, "compact": _plain_compact,
            "copy": _plain_copy}[s["case"]["kind"]](s)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    c = case
    if c["kind"] not in ("append", "attention"):
        return None      # whole numbers: page ids, counts and bytes
    s, _ = _inputs(c, seed)
    counts, lens = _rows(c)
    if c["kind"] == "append":
        out = {}
        for name in ("k", "v"):
            x = s[name].double().unflatten(-1, (-1, 32))
            a = x.abs().max(-1, keepdim=True).values / 7
            e = torch.floor(torch.log2(a))
            step = torch.exp2(torch.clamp(e - 7, min=-24.0))            # 8 significant bits, FP16's smallest step
            scale = torch.round(a / step) * step
            y = torch.clamp(torch.round(x / scale), -7, 7) * scale
            y = torch.where(scale > 0, y, torch.zeros_like(y)).flatten(-2)
            for b in range(c["B"]):
                y[b, counts[b]:] = 0
            out[name] = y
        return out
    H, d, ps, G = c["Hkv"], c["d"], c["ps"], c["Hq"] // c["Hkv"]
    out = torch.zeros(c["B"], c["S"], c["Hq"], d, dtype=torch.float64, device=DEV)
    i16, half = torch.arange(16, device=DEV), torch.arange(d, device=DEV)
    # byte and nibble of each (key, dim) of a tile, and its scale
    k_at = (half % 32 // 8)[None] * 2 * d + i16[:, None] * (d // 8) + half // 64 * 8 + half % 8
    k_up = (half // 32 % 2).expand(16, d)
    v_at = (i16 // 4)[:, None] * 2 * d + half % 16 * (d // 8) + half // 32 * 4 + (i16 % 4)[:, None]
    v_up = (half // 16 % 2).expand(16, d)
    s_at = ((i16 // 4)[:, None] * (d // 32) + half // 32) * 4 + (i16 % 4)[:, None]
    for b in range(c["B"]):
        n, m = lens[b], counts[b]
        ids = s["table"][b, :-(-n // ps)].long()
        p = torch.arange(n - m, n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)
        seen = (j <= p) if c["causal"] else torch.ones(m, n, dtype=torch.bool, device=DEV)
        if c["window"]:
            seen = seen & ((p - j <= c["window"]) | (j < c["sink"]))
        for h in range(H):
            t = s["pages"][0, ids, h].reshape(-1, 18 * d)
            kv = []
            for at, up, base in ((k_at, k_up, 0), (v_at, v_up, 9 * d)):
                code = (t[:, base + at].long() >> (4 * up)) % 16 - 8
                scale = t[:, base + 8 * d:base + 9 * d].contiguous().view(torch.float16)[:, s_at]
                kv.append((code.double() * scale.double()).reshape(-1, d)[:n].contiguous())
            q = s["q"][b, :m, h * G:(h + 1) * G].double()
            for g in range(G):
                x = q[:, g].contiguous() @ kv[0].t().contiguous() / math.sqrt(d)
                x = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                out[b, :m, h * G + g] = x @ kv[1]
    return out
