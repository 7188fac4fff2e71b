"""Workloads of a serving step of many sequences around the paged 4-bit KV
cache (include/cactus_hip.h):

  append   cactus_hip_kv4_append_rope_f16: the head norms and the position
           rotation of new query and key rows, each at its sequence's own
           positions, with keys and values quantized into the pages; read
           back as the values that the pages hold
  lora     cactus_hip_lora_add_f16: low-rank adapters, one per request, added
           to the output of a projection that the requests share
  logits   cactus_hip_logits_rules_f16 / _f32: penalties for repeated tokens,
           biases and grammar masks of each sequence, and the best token

The plain forms are torch operations in 32 bits; keys in 64, because a key next
to the border of two 4-bit codes has to fall on the right side of it.
"""
import math

import torch

own = False

DEV = "cuda"
GROUP = 32        # dims that share a scale in the cache
THETA, EPS = 1e6, 1e-6


def listed():
    return [
        # the first tokens of an answer from a small model (Gemma-3-270m's heads): all latency
        {"name": "append_first", "kind": "append", "B": 1, "S": 1, "len": 57, "ragged": False, "Hq": 4, "Hkv": 1, "d": 256,
         "ps": 16, "norm": True},
        # a decode step of 64 conversations, Qwen3-0.6B's heads and head norms
        {"name": "append_step_64", "kind": "append", "B": 64, "S": 1, "len": 4096, "ragged": True, "Hq": 16, "Hkv": 8, "d": 128,
         "ps": 64, "norm": True},
        # eight sequences verify up to five drafted tokens, 64-dim heads without norms, far into long documents
        {"name": "append_verify_5", "kind": "append", "B": 8, "S": 5, "len": 90001, "ragged": True, "Hq": 32, "Hkv": 8, "d": 64,
         "ps": 256, "norm": False},
        # one layer of four prompts of different lengths, right-padded to the longest
        {"name": "append_prompts", "kind": "append", "B": 4, "S": 2048, "len": 2500, "ragged": True, "Hq": 16, "Hkv": 8,
         "d": 128, "ps": 64, "norm": True},
        # one conversation's token through Qwen3-0.6B's query projection: all latency
        {"name": "lora_one", "kind": "lora", "B": 1, "S": 1, "ragged": False, "K": 1024, "N": 2048, "r": 16, "adapters": 4,
         "bare": 0},
        # a decode step of 64 requests with 24 adapters, every fifth request without one, output projection
        {"name": "lora_step_64", "kind": "lora", "B": 64, "S": 1, "ragged": False, "K": 2048, "N": 1024, "r": 16, "adapters": 24,
         "bare": 5},
        # prompts of very different lengths, each with its own adapter
        {"name": "lora_prompts", "kind": "lora", "B": 5, "S": 701, "ragged": True, "K": 1024, "N": 2048, "r": 32, "adapters": 8,
         "bare": 0},
        # long prompts in a wide model with adapters of high rank
        {"name": "lora_wide", "kind": "lora", "B": 8, "S": 1024, "ragged": False, "K": 4096, "N": 4096, "r": 64, "adapters": 8,
         "bare": 0},
        # one sampled answer, the repetitions of its last 300 tokens held down
        {"name": "logits_one", "kind": "logits", "B": 1, "V": 151936, "wide": False, "H": 300, "bias": 0, "masked": 0,
         "penalties": True},
        # the largest FP32 logits of a small odd vocabulary with many biases and no penalties
        {"name": "logits_biased", "kind": "logits", "B": 6, "V": 32003, "wide": True, "H": 0, "bias": 300, "masked": 0,
         "penalties": False},
        # a step of 32 requests, three of four with a grammar
        {"name": "logits_grammar_32", "kind": "logits", "B": 32, "V": 151936, "wide": False, "H": 2000, "bias": 40, "masked": 75,
         "penalties": True},
        # a step of a full server: 256 sequences with long histories
        {"name": "logits_256", "kind": "logits", "B": 256, "V": 151936, "wide": False, "H": 8192, "bias": 16, "masked": 25,
         "penalties": True},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, round(v / step) * step)))


def draw(rng):
    kind = rng.choice(["append", "lora", "logits"])
    if kind == "append":
        S = rng.choice([1, 1, _log(rng, 2, 12), _log(rng, 13, 2048)])
        B = _log(rng, 1, 96 if S == 1 else max(1, min(32, 6000 // S)))
        Hkv = rng.choice([1, 2, 4, 8])
        return {"kind": kind, "B": B, "S": S, "len": S + _log(rng, 1, max(2, min(60000, 400000 // B))),
                "ragged": rng.random() < 0.7, "Hq": Hkv * rng.choice([1, 2, 3, 4]), "Hkv": Hkv,
                "d": rng.choice([64, 128, 128]) if S > 12 else rng.choice([64, 128, 256]), "ps": rng.choice([16, 32, 64, 128, 256]),
                "norm": rng.random() < 0.6}
    if kind == "lora":
        S = rng.choice([1, 1, _log(rng, 2, 20), _log(rng, 21, 1024)])
        B = _log(rng, 1, 128 if S == 1 else max(1, min(32, 6000 // S)))
        return {"kind": kind, "B": B, "S": S, "ragged": S > 1 and rng.random() < 0.6, "K": _log(rng, 256, 4096, 8),
                "N": _log(rng, 64, 4096, 8), "r": rng.choice([8, 8, 16, 16, 24, 32, 64]), "adapters": rng.randint(1, 32),
                "bare": rng.choice([0, 0, 2, 5])}
    B = _log(rng, 1, 180)
    return {"kind": kind, "B": B, "V": rng.choice([_log(rng, 1000, 151936), _log(rng, 1000, 151936, 8)]), "wide": rng.random() < 0.3,
            "H": rng.choice([0, _log(rng, 4, 8192), _log(rng, 4, 8192)]), "bias": rng.choice([0, 0, _log(rng, 1, 300)]),
            "masked": rng.choice([0, 25, 100]), "penalties": rng.random() < 0.8}


# ------------------------------------------------------------------ shapes
def _spread(n, lo, hi):
    """n lengths between lo and hi, the same ones for a case, the last one hi."""
    return [lo + round((hi - lo) * math.modf((i + 1) * 0.6180339887)[0]) for i in range(n - 1)] + [hi]


def _rows(c):
    """New rows and length of each sequence of an append case."""
    if not c["ragged"]:
        return [c["S"]] * c["B"], [c["len"]] * c["B"]
    return _spread(c["B"], max(1, c["S"] // 3), c["S"]), _spread(c["B"], max(c["S"], c["len"] // 16), c["len"])


def _requests(c):
    """Rows of each request of a lora case, and which adapter it has (-1: none), as numbers of a list."""
    counts = _spread(c["B"], max(1, c["S"] // 6), c["S"]) if c["ragged"] else [c["S"]] * c["B"]
    return counts, [-1 if c["bare"] and i % c["bare"] == 1 else i * 7 % c["adapters"] for i in range(c["B"])]


def _lists(c):
    """Tokens in each sequence's history, entries of its bias list, and its mask (-1: none)."""
    hist = _spread(c["B"], c["H"] // 8, c["H"])
    bias = _spread(c["B"], c["bias"] // 4, c["bias"])
    # four grammars' states; the sequences with one are spread over the batch
    mask = [i % 4 if (i * 61) % 100 < c["masked"] else -1 for i in range(c["B"])]
    return hist, bias, mask


def work(case):
    c = case
    if c["kind"] == "append":
        rows, lens = _rows(c)
        n, kv = sum(rows), sum(rows) * c["Hkv"] * c["d"] * 2
        # q in and out, k and v in, codes and scales out; read back: codes and scales in, rows out; the rotations' table
        table = sum(rows) if c["S"] > 1 else len(set(lens))
        return {"bytes": 4 * n * c["Hq"] * c["d"] + 2 * (2 * kv + kv * 9 // 16) + 4 * table * c["d"],
                "flops": n * c["d"] * (7 * c["Hq"] + 11 * c["Hkv"])}
    if c["kind"] == "lora":
        counts, ids = _requests(c)
        n, used = sum(counts), len({a for a in ids if a >= 0})
        m = sum(k for k, a in zip(counts, ids) if a >= 0)
        return {"bytes": 2 * (m * c["K"] + 2 * n * c["N"] + used * c["r"] * (c["K"] + c["N"])),
                "flops": 2 * m * c["r"] * (c["K"] + c["N"])}
    hist, bias, mask = _lists(c)
    words = -(-c["V"] // 32)
    return {"bytes": c["B"] * c["V"] * (8 if c["wide"] else 6) + 4 * sum(hist) + 8 * sum(bias) + 4 * words * len(set(mask) - {-1}),
            "flops": c["B"] * c["V"]}


# ------------------------------------------------------------------ inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _append_inputs(c, g):
    B, S, Hq, Hkv, d, ps = (c[n] for n in ("B", "S", "Hq", "Hkv", "d", "ps"))
    counts, lens = _rows(c)
    need = [-(-n // ps) for n in lens]
    most, pages = max(need), sum(need) + 5
    order = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((B, most), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    refs[order[:at].long()] = 1
    # queries, keys and values of a row side by side, as one projection leaves them; a few channels larger than the rest
    heads = Hq + 2 * Hkv
    qkv = torch.randn(B, S, heads, d, generator=g, device=DEV)
    qkv *= 1 + 3 * (torch.rand(heads, d, generator=g, device=DEV) > 0.95)
    s = {"qkv": qkv.half(), "counts": _ints(counts), "lens": _ints(lens), "table": table, "refs": refs, "state": _ints([5, 0, 0, 0])}
    s["q_norm"] = (1 + 0.3 * torch.randn(d, generator=g, device=DEV)).half() if c["norm"] else None
    s["k_norm"] = (1 + 0.3 * torch.randn(d, generator=g, device=DEV)).half() if c["norm"] else None
    # cosines and sines of the angles, from 64 bits
    i = torch.arange(d // 2, device=DEV, dtype=torch.float64)
    angle = torch.arange(most * ps, device=DEV, dtype=torch.float64)[:, None] * THETA ** (-2 * i / d)
    s["rope"] = torch.stack((angle.cos(), angle.sin()), 1).float()                # [position][cos, sin][d / 2]
    s["shape"] = {"layers": 1, "kv_heads": Hkv, "head_dim": d, "page_size": ps, "num_pages": pages, "max_seqs": B, "max_pages": most}
    return s


def _lora_inputs(c, g):
    B, S, K, N, r, n = (c[k] for k in ("B", "S", "K", "N", "r", "adapters"))
    counts, ids = _requests(c)
    name = torch.randperm(n, generator=g, device=DEV).int()
    ids = _ints(ids)
    s = {"x": torch.randn(B, S, K, generator=g, device=DEV).half(), "base": torch.randn(B, S, N, generator=g, device=DEV).half(),
         "A": (torch.randn(n, r, K, generator=g, device=DEV) / math.sqrt(K)).half(),
         "Bt": (torch.randn(n, N, r, generator=g, device=DEV) / math.sqrt(r)).half(),
         "scales": 0.25 + torch.rand(n, generator=g, device=DEV), "counts": _ints(counts),
         "ids": torch.where(ids >= 0, name[ids.long().clamp_min(0)], ids)}
    s["y"] = torch.zeros_like(s["base"])
    return s


def _logits_inputs(c, g):
    B, V = c["B"], c["V"]
    hist, bias, mask = _lists(c)
    x = 2.5 * torch.randn(B, V, generator=g, device=DEV) - 3
    x += 9 * (torch.rand(B, V, generator=g, device=DEV) > 0.9997)
    s = {"logits": x if c["wide"] else x.half()}
    # texts repeat themselves: a few tokens are most of a history
    u = torch.rand(B, max(1, c["H"]), generator=g, device=DEV, dtype=torch.float64)
    shuffled = torch.randperm(V, generator=g, device=DEV).int()
    s["history"] = shuffled[(V ** u - 1).long().clamp(0, V - 1)]
    s["hist_lens"] = _ints(hist)
    s["repetition"] = 1 + 0.3 * torch.rand(B, generator=g, device=DEV)
    s["frequency"] = torch.rand(B, generator=g, device=DEV)
    s["presence"] = torch.rand(B, generator=g, device=DEV)
    if c["bias"]:
        first = torch.randint(0, V, (B, 1), generator=g, device=DEV)
        step = V // c["bias"]
        s["bias_tokens"] = ((first + torch.arange(c["bias"], device=DEV) * step) % V).int()
        s["bias_values"] = 4 * torch.randn(B, c["bias"], generator=g, device=DEV)
        s["bias_counts"] = _ints(bias)
    # grammar states that allow from a few tokens to most of them, a bit per token
    share = torch.tensor([0.9, 0.3, 0.02, 0.0004], device=DEV)[:, None]
    words = -(-V // 32)
    bits = torch.rand(4, words * 32, generator=g, device=DEV) < share
    s["masks"] = (bits.view(4, words, 32).long() << torch.arange(32, device=DEV)).sum(-1).to(torch.int32)
    s["mask_ids"] = _ints(mask)
    s["out"] = torch.zeros(B, V, dtype=torch.float32, device=DEV)
    s["best"] = torch.zeros(B, dtype=torch.int32, device=DEV)
    return s


def _inputs(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"append": _append_inputs, "lora": _lora_inputs, "logits": _logits_inputs}[c["kind"]](c, g)


def prepare(case, seed):
    """The inputs, the cache with its tables and the output buffers, as a serving program holds them."""
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "append":
        c, n = case, s["shape"]["num_pages"]
        B, S, H, d, ps = (c[k] for k in ("B", "S", "Hkv", "d", "ps"))
        s["q_out"] = torch.zeros(B, S, c["Hq"], d, dtype=torch.float16, device=DEV)
        s["k_out"], s["v_out"] = (torch.zeros(B, S, H, d, dtype=torch.float16, device=DEV) for _ in range(2))
        s["pages"] = torch.zeros(n * H * ps * d * 9 // 8, dtype=torch.uint8, device=DEV)
        # the plain form's cache: a byte per code, keys and values
        s["codes"] = torch.zeros(2, n * ps, H, d, dtype=torch.int8, device=DEV)
        s["steps"] = torch.zeros(2, n * ps, H, d // GROUP, dtype=torch.float16, device=DEV)
    if case["kind"] == "logits":
        # scratch memory of the best token's search, zero before the first call
        s["workspace"] = torch.zeros(16 * case["B"], dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------ plain forms
def _half(x):
    """64 bits to FP16 with one rounding: the bits that FP32 would round away stay as a sticky bit."""
    b = x.view(torch.int64)
    rest = (b & 0xFFFFFFFF) != 0
    return (((b >> 32) | rest) << 32).view(torch.float64).float().half()


def _rotated(x, w, cos, sin):
    """Rows [n][heads][d] in 64 bits: normed by w (None: not), rotated by the rows' angles, rounded to FP16."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    a, b = x.chunk(2, -1)
    return _half(torch.cat((a * cos - b * sin, b * cos + a * sin), -1))


def _plain_append(s):
    c = s["case"]
    S, Hq, Hkv, d, ps = (c[n] for n in ("S", "Hq", "Hkv", "d", "ps"))
    r = torch.arange(S, device=DEV)
    m, n = s["counts"].long()[:, None], s["lens"].long()[:, None]
    b, r = (r < m).nonzero(as_tuple=True)
    pos = (n - m)[b, 0] + r
    rows = s["qkv"][b, r]                                                          # [n][heads][d]
    cos, sin = s["rope"][pos].double()[:, None].unbind(2)
    s["q_out"][b, r] = _rotated(rows[:, :Hq], s["q_norm"], cos, sin)
    new = torch.stack((_rotated(rows[:, Hq:Hq + Hkv], s["k_norm"], cos, sin), rows[:, Hq + Hkv:]))
    x = new.float().unflatten(-1, (-1, GROUP))
    step = (x.abs().amax(-1, keepdim=True) / 7).bfloat16().half()
    code = torch.where(step > 0, torch.round(x / step.float()), torch.zeros_like(x)).clamp(-7, 7)
    at = s["table"].long()[b, pos // ps] * ps + pos % ps
    s["codes"][:, at] = code.flatten(-2).to(torch.int8)
    s["steps"][:, at] = step.squeeze(-1)
    back = s["codes"][:, at].float().unflatten(-1, (-1, GROUP)) * s["steps"][:, at].float()[..., None]
    s["k_out"][b, r], s["v_out"][b, r] = back.flatten(-2).half()
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _plain_lora(s):
    a = s["ids"].long()
    scale = torch.where(a >= 0, s["scales"][a.clamp_min(0)], torch.zeros_like(s["scales"][:1]))[:, None, None]
    h = torch.bmm(s["x"].float(), s["A"][a.clamp_min(0)].float().transpose(1, 2).contiguous())
    y = s["base"].float() + scale * torch.bmm(h, s["Bt"][a.clamp_min(0)].float().transpose(1, 2).contiguous())
    there = torch.arange(y.shape[1], device=DEV)[None, :, None] < s["counts"].long()[:, None, None]
    s["y"].copy_(torch.where(there, y, s["y"].float()))
    return s["y"]


def _plain_logits(s):
    c = s["case"]
    V = c["V"]
    x = s["logits"].float()
    if c["penalties"]:
        t = s["history"].long()
        there = torch.arange(t.shape[1], device=DEV) < s["hist_lens"].long()[:, None]
        n = torch.zeros_like(x).scatter_add_(1, t, there.float())
        p, f, q = (s[k][:, None] for k in ("repetition", "frequency", "presence"))
        x = torch.where(n > 0, torch.where(x > 0, x / p, x * p) - f * n - q, x)
    if c["bias"]:
        there = torch.arange(c["bias"], device=DEV) < s["bias_counts"].long()[:, None]
        x = x.scatter_add(1, s["bias_tokens"].long(), s["bias_values"] * there)
    if c["masked"]:
        i = torch.arange(V, device=DEV)
        bits = (s["masks"][:, i // 32] >> (i % 32).int()) & 1                      # [mask][V]
        ids = s["mask_ids"].long()[:, None]
        x = torch.where((ids < 0) | (bits[ids[:, 0].clamp_min(0)] > 0), x, torch.full_like(x[:1, :1], -math.inf))
    s["out"].copy_(x)
    most = x.amax(1, keepdim=True)
    i = torch.arange(V, device=DEV)
    s["best"].copy_(torch.where(x == most, i, V).amin(1))
    return {"logits": s["out"], "best": s["best"]}


# ------------------------------------------------------------------ the framework's calls
def _own_append(s):
    import cactus_amd as cm
    from cactus_amd.kv4 import CacheDesc
    c = s["case"]
    Hq, Hkv, d = c["Hq"], c["Hkv"], c["d"]
    if "cache" not in s:      # the handle that a program keeps
        s["cache"] = CacheDesc(pages=s["pages"].data_ptr(), table=s["table"].data_ptr(), lens=s["lens"].data_ptr(),
                               refs=s["refs"].data_ptr(), state=s["state"].data_ptr(), **s["shape"])
    row, q = (Hq + 2 * Hkv) * d, s["qkv"].data_ptr()
    q_norm, k_norm = (s[n].data_ptr() if s[n] is not None else None for n in ("q_norm", "k_norm"))
    cm.call("cactus_hip_kv4_append_rope_f16", s["cache"].ref, 0, None, s["counts"].data_ptr(), q, row, s["q_out"].data_ptr(), Hq,
            q + 2 * Hq * d, q + 2 * (Hq + Hkv) * d, row, q_norm, k_norm, EPS, s["rope"].data_ptr(), s["rope"].shape[0],
            c["B"], c["S"], None)
    cm.call("cactus_hip_kv4_read_f16", s["cache"].ref, 0, None, None, s["counts"].data_ptr(), s["k_out"].data_ptr(),
            s["v_out"].data_ptr(), c["B"], c["S"], None)
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _own_lora(s):
    import cactus_amd as cm
    c = s["case"]
    cm.call("cactus_hip_lora_add_f16", s["x"].data_ptr(), c["K"], s["A"].data_ptr(), s["Bt"].data_ptr(), s["scales"].data_ptr(),
            c["adapters"], c["r"], s["ids"].data_ptr(), s["counts"].data_ptr(), s["base"].data_ptr(), c["N"], s["y"].data_ptr(),
            c["N"], c["B"], c["S"], c["K"], c["N"], None)
    return s["y"]


def _own_logits(s):
    import cactus_amd as cm
    from cactus_amd.logits import RulesDesc
    c = s["case"]
    if "rules" not in s:      # the handle that a program keeps
        r = {"max_seqs": c["B"]}
        if c["penalties"]:
            r.update(history=s["history"].data_ptr(), history_lens=s["hist_lens"].data_ptr(), history_stride=s["history"].shape[1],
                     repetition=s["repetition"].data_ptr(), frequency=s["frequency"].data_ptr(), presence=s["presence"].data_ptr())
        if c["bias"]:
            r.update(bias_tokens=s["bias_tokens"].data_ptr(), bias_values=s["bias_values"].data_ptr(),
                     bias_counts=s["bias_counts"].data_ptr(), bias_stride=c["bias"])
        if c["masked"]:
            r.update(masks=s["masks"].data_ptr(), mask_ids=s["mask_ids"].data_ptr(), num_masks=4, mask_stride=s["masks"].shape[1])
        s["rules"] = RulesDesc(**r)
    cm.call("cactus_hip_logits_rules_f32" if c["wide"] else "cactus_hip_logits_rules_f16", s["rules"].ref, None,
            s["logits"].data_ptr(), c["V"], s["out"].data_ptr(), c["V"], s["best"].data_ptr(), c["B"], c["V"],
            s["workspace"].data_ptr(), s["workspace"].numel(), None)
    return {"logits": s["out"], "best": s["best"]}


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"append": _own_append, "lora": _own_lora, "logits": _own_logits}[kind](s)
    return {"append": _plain_append, "lora": _plain_lora, "logits": _plain_logits}[kind](s)


# ------------------------------------------------------------------ in 64 bits
def _round16(x):
    """Nearest FP16 value (ties to even) of numbers within FP16's range, from its spacing."""
    step = torch.exp2((torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -30))) - 10).clamp_min(-24))
    return torch.round(x / step) * step


def _exact_append(c, s):
    Hq, Hkv, d = c["Hq"], c["Hkv"], c["d"]
    counts, lens = _rows(c)
    q = torch.zeros(c["B"], c["S"], Hq, d, dtype=torch.float64, device=DEV)
    k, v = (torch.zeros(c["B"], c["S"], Hkv, d, dtype=torch.float64, device=DEV) for _ in range(2))
    for b, (m, n) in enumerate(zip(counts, lens)):
        x = s["qkv"][b, :m].double()
        turn = torch.complex(s["rope"][n - m:n, 0].double(), s["rope"][n - m:n, 1].double())[:, None]
        for out, lo, hi, w in ((q, 0, Hq, s["q_norm"]), (k, Hq, Hq + Hkv, s["k_norm"])):
            y = x[:, lo:hi]
            if w is not None:
                y = y * w.double() * torch.rsqrt(y.square().sum(-1, keepdim=True) / d + EPS)
            z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * turn
            out[b, :m] = torch.cat((z.real, z.imag), -1)
        v[b, :m] = x[:, Hq + Hkv:]
    out = [q]
    for x in (_round16(k), v):
        x = x.view(*x.shape[:-1], d // 32, 32)
        a = x.abs().max(-1, keepdim=True).values / 7
        step = torch.exp2((torch.floor(torch.log2(a.clamp_min(2.0 ** -40))) - 7).clamp_min(-24))      # 8 significant bits
        scale = torch.round(a / step) * step
        y = torch.clamp(torch.round(x / scale), -7, 7) * scale
        out.append(torch.where(scale > 0, y, torch.zeros_like(y)).flatten(-2))
    return dict(zip("qkv", out))


def _exact_lora(c, s):
    counts, _ = _requests(c)
    y = torch.zeros(s["base"].shape, dtype=torch.float64, device=DEV)
    for b, (m, a) in enumerate(zip(counts, s["ids"].tolist())):
        y[b, :m] = s["base"][b, :m].double()
        if a >= 0:
            down, up = s["A"][a].double(), s["Bt"][a].double()
            y[b, :m] += (up @ (down @ s["x"][b, :m].double().t().contiguous())).t() * s["scales"][a].double()
    return y


def _exact_logits(c, s):
    hist, bias, mask = _lists(c)
    out = torch.empty(c["B"], c["V"], dtype=torch.float64, device=DEV)
    for b in range(c["B"]):
        x = s["logits"][b].double()
        if c["penalties"]:
            t, n = torch.unique(s["history"][b, :hist[b]].long(), return_counts=True)
            l, p = x[t], s["repetition"][b].double()
            x[t] = torch.where(l > 0, l / p, l * p) - n * s["frequency"][b].double() - s["presence"][b].double()
        if c["bias"]:
            x[s["bias_tokens"][b, :bias[b]].long()] += s["bias_values"][b, :bias[b]].double()
        if c["masked"] and mask[b] >= 0:
            allowed = (s["masks"][mask[b]][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
            x[allowed.view(-1)[:c["V"]] == 0] = -math.inf
        out[b] = x
    return {"logits": out, "best": None}


def exact(case, seed):
    s = _inputs(case, seed)
    return {"append": _exact_append, "lora": _exact_lora, "logits": _exact_logits}[case["kind"]](case, s)
