"""The operators around an fp8 cache of keys and values, as timed cases.

The cache holds, per row (one position of one sequence) and key/value head, 128 codes in e4m3 and one fp32 scale: the least
power of two 2^e (e >= -60) with amax <= 448 * 2^e.  A value is code * scale, which bf16 holds exactly.  Four operators:

* *write*: the packed rows of a dense step (or the last rows of every sequence) are quantised into the cache;
* *update*: the salient rows of a sparse step: rotary embedding of the new keys, both quantised into their caches, and the
  difference between the new and the old cached values (delta-V).  A pass is two steps that write two sets of rows in turn, so
  that every pass starts from the cache that the one before has left and meets values that changed;
* *read*: cache rows back as packed bf16;
* *attend*: exact attention of listed query rows over the cached keys and values of their sequence, optionally with scores
  capped by a tanh, with a bias that falls with the distance, and with a range of visible keys per query row (sliding window,
  block-causal prefix, documents; padding rows see nothing and give zeros).

``run`` computes them in their plain form, or, where ``own`` is set, makes the package's calls.  ``exact`` is the same from
the definitions in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
D = 128
MIN_EXP = -60
BLOCK = 32          # positions of a response block (block-causal prefixes)
FREE_ROWS = 5       # cache rows in front of the sequences that belong to nobody


def listed():
    return [
        # the dense step of one short request, grouped-query model: latency
        {"name": "write_b1_301", "kind": "write", "batch": 1, "length": 301, "gen": 301, "ragged": False, "heads": 4},
        # the dense step of the headline batch (16 x (256 + 256)); the keys are one half of a fused K/V product
        {"name": "write_b16_512", "kind": "write", "batch": 16, "length": 512, "gen": 512, "ragged": False, "heads": 32},
        # a sparse step of one short request: a handful of rows
        {"name": "update_b1_256", "kind": "update", "batch": 1, "length": 256, "gen": 128, "ragged": False, "heads": 32, "rows": 7},
        # the at-scale batch (64 x (512 + 512)) with every tenth position salient
        {"name": "update_b64_1024", "kind": "update", "batch": 64, "length": 1024, "gen": 1024, "ragged": False, "heads": 32,
         "rows": 102},
        # requests of unequal lengths, the response rows alone
        {"name": "read_b6_ragged", "kind": "read", "batch": 6, "length": 397, "gen": 96, "ragged": True, "heads": 32},
        # the keys of one layer for a step of the at-scale batch
        {"name": "read_b64_1024", "kind": "read", "batch": 64, "length": 1024, "gen": 1024, "ragged": False, "heads": 32},
        # one short request: latency
        {"name": "attend_b1_256", "kind": "attend", "batch": 1, "length": 256, "gen": 128, "ragged": False, "heads": 32,
         "kv_heads": 32, "rows": 6, "at": "spread", "mask": "none", "cap": 0.0, "bias": False},
        # the headline batch, five of a hundred rows salient
        {"name": "attend_b16_512", "kind": "attend", "batch": 16, "length": 512, "gen": 512, "ragged": False, "heads": 32,
         "kv_heads": 32, "rows": 26, "at": "spread", "mask": "none", "cap": 0.0, "bias": False},
        # grouped-query heads, unequal lengths (one of them a single token, some without a row)
        {"name": "attend_gqa_b32", "kind": "attend", "batch": 32, "length": 601, "gen": 256, "ragged": True, "heads": 28,
         "kv_heads": 4, "rows": 12, "at": "spread", "mask": "none", "cap": 0.0, "bias": False},
        # one block of 32 rows decoded over long caches, distance bias
        {"name": "attend_long_b2", "kind": "attend", "batch": 2, "length": 32011, "gen": 32, "ragged": False, "heads": 32,
         "kv_heads": 8, "rows": 32, "at": "tail", "mask": "none", "cap": 0.0, "bias": True},
        # block-causal decoding of two blocks a sequence, capped scores
        {"name": "attend_prefix_b8", "kind": "attend", "batch": 8, "length": 4096, "gen": 64, "ragged": False, "heads": 16,
         "kv_heads": 16, "rows": 64, "at": "tail", "mask": "prefix", "cap": 30.0, "bias": False},
        # every row of packed documents (a dense step), with padding at the end
        {"name": "attend_docs_all", "kind": "attend", "batch": 4, "length": 2048, "gen": 2048, "ragged": False, "heads": 16,
         "kv_heads": 16, "rows": 2048, "at": "tail", "mask": "docs", "cap": 0.0, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(c):
    """What a case costs: elements of the caches it touches, and of the score matrix."""
    if c["kind"] != "attend":
        return c["batch"] * (c["rows"] if c["kind"] == "update" else c["gen"]) * c["heads"] * D, 0
    n = min(c["rows"] * (2 if c["ragged"] else 1), c["gen"], c["length"])
    return c["batch"] * c["length"] * c["kv_heads"] * D, c["batch"] * n * c["length"] * c["heads"]


def draw(rng):
    while True:
        kind = rng.choice(["write", "update", "read", "attend", "attend", "attend"])
        length = _log(rng, 1, 33000)
        c = {"kind": kind, "batch": _log(rng, 1, 70), "length": length, "gen": rng.choice([length, _log(rng, 1, length)]),
             "ragged": rng.random() < 0.6, "heads": rng.choice([1, 4, 8, 16, 32])}
        if kind == "update":
            c["rows"] = _log(rng, 1, 200)
        if kind == "attend":
            c["heads"], c["kv_heads"] = rng.choice([(32, 32), (16, 16), (28, 4), (32, 8), (7, 1), (8, 8), (5, 5), (16, 2)])
            c["rows"] = _log(rng, 1, rng.choice([20, 300, 2500]))
            c["mask"] = rng.choice(["none", "none", "prefix", "window", "docs"])
            c["at"] = rng.choice(["spread", "tail"]) if c["mask"] != "docs" else "spread"      # the last rows are padding
            c["cap"] = rng.choice([0.0, 0.0, 20.0, 50.0])
            c["bias"] = rng.random() < 0.3
        elements, scores = _size(c)
        if elements <= 64 * 1024 * 32 * D // (8 if kind == "attend" else 1) and scores <= 4 * 2048 * 2048 * 16:
            return c


# ---------------------------------------------------------------------------------------------------------------------
# geometry: follows from the case alone
# ---------------------------------------------------------------------------------------------------------------------
def _lens(c):
    """(cached positions, query rows) per sequence: the queries are a sequence's last rows."""
    n, length = c["batch"], c["length"]
    lens = [length] * n
    if c["ragged"]:
        lens = [length - (37 * i) % (1 + 3 * length // 4) for i in range(n)]
        if n > 2:
            lens[-1] = 1
    return lens, [min(c["gen"], v) for v in lens]


def _rows(c):
    """Listed rows per sequence."""
    _, q = _lens(c)
    if c["ragged"]:
        return [min((13 * i + c["rows"]) % (2 * c["rows"] + 1), v) for i, v in enumerate(q)]
    return [min(c["rows"], v) for v in q]


def _documents(length):
    """First position of every document of a sequence, and of the padding behind the last one."""
    pad = length - length // 16
    starts, pos, i = [], 0, 0
    while pos < pad:
        starts.append(pos)
        pos += 257 + (389 * i) % 700
        i += 1
    return starts + [pad]


def _ranges(c):
    """Visible keys [begin, end) of every query row (None: all of its sequence), as an int32 matrix on the CPU."""
    if c["mask"] == "none":
        return None
    lens, qs = _lens(c)
    got = []
    for length, q in zip(lens, qs):
        pos = torch.arange(length - q, length)
        if c["mask"] == "prefix":
            begin, end = torch.zeros_like(pos), ((pos // BLOCK + 1) * BLOCK).clamp_max(length)
        elif c["mask"] == "window":
            w = 1 + length // 8
            begin, end = (pos - w).clamp_min(0), (pos + w + 1).clamp_max(length)
        else:
            marks = torch.tensor(_documents(length) + [length])
            doc = torch.searchsorted(marks, pos, right=True) - 1
            pad = doc >= marks.numel() - 2
            begin, end = marks[doc].masked_fill(pad, 0), marks[(doc + 1).clamp_max(marks.numel() - 1)].masked_fill(pad, 0)
        got.append(torch.stack([begin, end], 1))
    return torch.cat(got).to(torch.int32)


def _cumulate(v):
    return [0] + torch.tensor(v).cumsum(0).tolist()


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _quantise(x):
    """(codes, scales) of x [..., heads, D]."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    part, exponent = torch.frexp(amax)                      # amax = part * 2^exponent, 0.5 <= part < 1; 448 = 0.875 * 2^9
    scale = torch.ldexp(torch.ones_like(amax), (exponent - 9 + (part > 0.875)).clamp_min(MIN_EXP))
    bad = ~torch.isfinite(amax)
    codes = torch.where(bad, 0.0, x / scale).to(torch.float8_e4m3fn)
    return codes, torch.where(bad, math.nan, scale).squeeze(-1)


def _values(codes, scales):
    return codes.float() * scales.unsqueeze(-1)


def prepare(case, seed):
    c, g = dict(case), torch.Generator(device=DEV).manual_seed(seed)
    lens, qs = _lens(c)
    cu_k, cu_q = _cumulate(lens), _cumulate(qs)
    batch, total_k, total_q = c["batch"], cu_k[-1], cu_q[-1]
    hkv = c.get("kv_heads", c["heads"])
    dev = lambda v, t: torch.tensor(v, dtype=t).to(DEV)     # noqa: E731

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def keys(n):        # a few channels of a head are much larger than the others
        return (randn(n, hkv, D) * torch.exp(0.8 * channels)).to(torch.bfloat16)

    def values(n):      # positions differ in size
        return (randn(n, hkv, D) * torch.exp(0.7 * randn(n, 1, 1))).to(torch.bfloat16)

    channels = randn(hkv, D)
    # the sequences lie in the cache in another order than in the batch; ids are arbitrary
    order = torch.randperm(batch, generator=g, device=DEV).tolist()
    seq_starts, pos = torch.full((4 * batch,), -1, dtype=torch.int64), FREE_ROWS
    ids = torch.randperm(4 * batch, generator=g, device=DEV)[:batch]
    ids_host = ids.tolist()
    for b in order:
        seq_starts[ids_host[b]] = pos
        pos += lens[b]
    s = {"kind": c["kind"], "cu_k": dev(cu_k, torch.int32), "cu_q": dev(cu_q, torch.int32), "starts": seq_starts.to(DEV),
         "ids": ids, "total_q": total_q, "total_k": total_k}
    rows = pos
    if c["kind"] == "write":
        s["x"] = torch.stack([keys(total_q), values(total_q)], 1)[:, 0]       # [rows, heads, D] inside the fused product
        s["codes"] = torch.zeros(rows, hkv * D, dtype=torch.float8_e4m3fn, device=DEV)
        s["scales"] = torch.zeros(rows, hkv, device=DEV)
        return s
    if c["kind"] == "read":
        codes, s["scales"] = _quantise(keys(rows))
        s["codes"] = codes.flatten(1)
        return s
    # lists of rows: ascending, grouped by sequence
    counts = _rows(c)
    picked, picked_k = [], []
    for b in range(batch):
        at = torch.arange(qs[b] - counts[b], qs[b])
        if c.get("at", "spread") == "spread":
            at = torch.randperm(qs[b], generator=g, device=DEV)[:counts[b]].sort().values.cpu()
        picked.append(at + cu_q[b])
        picked_k.append(at + cu_k[b] + lens[b] - qs[b])
    picked, picked_k = torch.cat(picked), torch.cat(picked_k)
    n = picked.numel()
    s["cu_rows"], s["count"] = dev(_cumulate(counts), torch.int32), n
    if c["kind"] == "update":
        s["rows_k"] = picked_k.to(torch.int64).to(DEV)
        s["pos_idx"] = picked.to(torch.int64).to(DEV)
        s["positions"] = torch.cat([torch.arange(a - b, a) for a, b in zip(lens, qs)]).to(DEV)
        angle = torch.outer(torch.arange(max(4096, c["length"]), dtype=torch.float64),
                            500000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().to(DEV)
        s["steps"] = [(keys(n), values(n)) for _ in range(2)]
        kc, s["k_scales"] = _quantise(keys(rows))
        v0 = values(rows)
        v0[_dest(s, s["rows_k"])] = s["steps"][1][1]         # the cache that the second step leaves
        vc, s["v_scales"] = _quantise(v0)
        s["k_codes"], s["v_codes"] = kc.flatten(1), vc.flatten(1)
        return s
    s["q"] = (2.0 * randn(total_q, c["heads"], D) * torch.exp(-0.8 * channels).repeat_interleave(c["heads"] // hkv, 0)).to(torch.bfloat16)
    s["rows"] = picked.to(torch.int32).to(DEV)
    s["max_rows"], s["max_k"] = max(max(counts), 1), max(lens)
    for name, x in (("k", keys(rows)), ("v", values(rows))):
        codes, s[name + "_scales"] = _quantise(x)
        s[name + "_codes"] = codes.flatten(1)
    ranges = _ranges(c)
    s["ranges"] = None if ranges is None else ranges.to(DEV)
    s["cap"] = c["cap"]
    s["slopes"] = torch.exp2(-8.0 * (torch.arange(c["heads"]) + 1) / c["heads"]).to(DEV) if c["bias"] else None
    return s


def _dest(s, rows_k):
    """Cache rows of packed key rows."""
    b = torch.searchsorted(s["cu_k"][1:].long(), rows_k, right=True)
    return s["starts"][s["ids"][b]] + rows_k - s["cu_k"].long()[b]


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)[state["kind"]](state)


def _last_rows(s):
    """Cache row of every packed query row (the last rows of each sequence)."""
    p = torch.arange(s["total_q"], device=DEV)
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    b = torch.searchsorted(cu_q[1:], p, right=True)
    return s["starts"][s["ids"][b]] + p - cu_q[b] + (cu_k[b + 1] - cu_k[b]) - (cu_q[b + 1] - cu_q[b])


def _write_plain(s):
    codes, scales = _quantise(s["x"])
    at = _last_rows(s)
    s["codes"][at] = codes.flatten(1)
    s["scales"][at] = scales
    return {"codes": s["codes"], "scales": s["scales"]}


def _read_plain(s):
    at = _last_rows(s)
    heads = s["scales"].size(1)
    return _values(s["codes"][at].view(-1, heads, D), s["scales"][at]).to(torch.bfloat16)


def _update_plain(s):
    at = _dest(s, s["rows_k"])
    cs = s["cos_sin"][s["positions"][s["pos_idx"]]].unsqueeze(1)
    cos, sin = cs[..., :64], cs[..., 64:]
    out = {}

    def step(name, k, v):
        a, b = k[..., :64].float(), k[..., 64:].float()
        kc, ks = _quantise(torch.cat([a * cos - b * sin, b * cos + a * sin], -1))
        vc, vs = _quantise(v)
        before = _values(s["v_codes"][at].view_as(vc), s["v_scales"][at])
        out[name] = (_values(vc, vs) - before).to(torch.bfloat16)
        s["k_codes"][at], s["k_scales"][at] = kc.flatten(1), ks
        s["v_codes"][at], s["v_scales"][at] = vc.flatten(1), vs

    step("dv_first", *s["steps"][0])
    step("dv_second", *s["steps"][1])
    return {**out, "k_codes": s["k_codes"], "k_scales": s["k_scales"], "v_codes": s["v_codes"], "v_scales": s["v_scales"]}


def _attend_plain(s):
    q, cu_q, cu_k, cu_r = s["q"], s["cu_q"].long(), s["cu_k"].long(), s["cu_rows"].long()
    heads, hkv = q.size(1), s["k_scales"].size(1)
    group, batch = heads // hkv, s["ids"].numel()
    n_max, l_max = s["max_rows"], s["max_k"]
    # keys and values of every sequence, padded to the longest; listed rows of every sequence, padded to the most
    key = torch.arange(l_max, device=DEV)
    there = key < (cu_k[1:] - cu_k[:-1]).unsqueeze(1)                                     # [B, L]
    at = torch.where(there, s["starts"][s["ids"]].unsqueeze(1) + key, 0)
    k = _values(s["k_codes"][at].view(batch, l_max, hkv, D), s["k_scales"][at]).permute(0, 2, 3, 1)    # [B, Hkv, D, L]
    v = _values(s["v_codes"][at].view(batch, l_max, hkv, D), s["v_scales"][at]).transpose(1, 2)        # [B, Hkv, L, D]
    slot = torch.arange(n_max, device=DEV) + cu_r[:-1].unsqueeze(1)
    live = slot < cu_r[1:].unsqueeze(1)                                                   # [B, N]
    row = s["rows"].long()[torch.where(live, slot, 0)]
    qs = q[row].float().view(batch, n_max, hkv, group, D).permute(0, 2, 3, 1, 4)          # [B, Hkv, G, N, D]
    t = torch.matmul(qs.reshape(batch, hkv, group * n_max, D), k).view(batch, hkv, group, n_max, l_max)
    t = t * D ** -0.5
    if s["cap"]:
        t = s["cap"] * torch.tanh(t / s["cap"])
    if s["slopes"] is not None:
        pos = row - cu_q[1:].unsqueeze(1) + (cu_k[1:] - cu_k[:-1]).unsqueeze(1)           # counted from the sequence's end
        away = (pos.unsqueeze(2) - key).abs().float()                                     # [B, N, L]
        t = t - s["slopes"].view(1, hkv, group, 1, 1) * away.view(batch, 1, 1, n_max, l_max)
    seen = there.unsqueeze(1) & live.unsqueeze(2)                                         # [B, N, L]
    if s["ranges"] is not None:
        r = s["ranges"][row].unsqueeze(2)                                                 # [B, N, 1, 2]
        seen = seen & (key >= r[..., 0]) & (key < r[..., 1])
    t = t.masked_fill(~seen.view(batch, 1, 1, n_max, l_max), -math.inf)
    top = t.amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, hkv, group * n_max, l_max), v).view(batch, hkv, group, n_max, D)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4)[live].reshape(-1, heads, D).to(torch.bfloat16)


_plain = {"write": _write_plain, "read": _read_plain, "update": _update_plain, "attend": _attend_plain}


def _write_own(s):
    from dyllm_b200 import ops
    ops.fp8_cache_write(s["x"], s["codes"], s["scales"], s["starts"], s["cu_q"], s["ids"], cu_seqlens_k=s["cu_k"])
    return {"codes": s["codes"], "scales": s["scales"]}


def _read_own(s):
    from dyllm_b200 import ops
    return ops.fp8_cache_read(s["codes"], s["scales"], s["starts"], s["cu_q"], s["ids"], s["total_q"], cu_seqlens_k=s["cu_k"])


def _update_own(s):
    from dyllm_b200 import ops
    out = {}
    for name, (k, v) in zip(("dv_first", "dv_second"), s["steps"]):
        out[name] = ops.fp8_kv_cache_update(k, v, s["rows_k"], s["positions"], s["pos_idx"], s["cos_sin"], s["cu_k"], s["starts"],
                                            s["starts"], s["ids"], (s["k_codes"], s["k_scales"]), (s["v_codes"], s["v_scales"]))
    return {**out, "k_codes": s["k_codes"], "k_scales": s["k_scales"], "v_codes": s["v_codes"], "v_scales": s["v_scales"]}


def _attend_own(s):
    from dyllm_b200.attention_ops import attention_salient_rows_fp8
    return attention_salient_rows_fp8(s["q"], (s["k_codes"], s["k_scales"]), (s["v_codes"], s["v_scales"]), s["starts"], s["starts"],
                                      s["ids"], s["cu_q"], s["cu_k"], s["cu_rows"], s["rows"], max_rows_per_seq=s["max_rows"],
                                      softcap=s["cap"], slopes=s["slopes"], key_ranges=s["ranges"])


_own = {"write": _write_own, "read": _read_own, "update": _update_own, "attend": _attend_own}


# ---------------------------------------------------------------------------------------------------------------------
# work and definition
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    hkv, row = c.get("kv_heads", c["heads"]), D + 4
    lens, qs = _lens(c)
    if c["kind"] in ("write", "read"):
        return {"bytes": sum(qs) * hkv * (2 * D + row), "flops": 0}
    n = sum(_rows(c))
    if c["kind"] == "update":
        # K: bf16 in, codes out; V: bf16 in, old codes in, codes out, difference out
        return {"bytes": 2 * n * hkv * (2 * D + row + 2 * D + 2 * row + 2 * D), "flops": 2 * n * hkv * D * 3}
    # pairs that see each other and keys that any row sees; of rows listed at random, the expected share
    ranges, counts, pairs, keys, pos = _ranges(c), _rows(c), 0.0, 0.0, 0
    for length, q, m in zip(lens, qs, counts):
        if ranges is None:
            pairs, keys = pairs + m * length, keys + (length if m else 0)
        elif m:
            r = ranges[pos:pos + q].long()
            r = r[q - m:] if c["at"] == "tail" else r
            pairs += float((r[:, 1] - r[:, 0]).sum()) * m / len(r)
            marks = torch.zeros(length + 1)
            marks.index_add_(0, r[:, 0], torch.ones(len(r)))
            marks.index_add_(0, r[:, 1], -torch.ones(len(r)))
            seen = marks.cumsum(0)[:length]
            keys += float((1 - (1 - seen / len(r)) ** m).sum())
        pos += q
    return {"bytes": keys * hkv * 2 * row + 2 * n * c["heads"] * 2 * D, "flops": 4 * D * c["heads"] * pairs}


def _exact_codes(x):
    """(codes, scales) in 64 bits: the nearest number of the e4m3 grid (3 bits behind the point, steps of 2^-9 below 2^-6)."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -200) / 448)).clamp_min(MIN_EXP)
    e = torch.where(amax > 448 * torch.exp2(e), e + 1, torch.where((amax <= 224 * torch.exp2(e)) & (e > MIN_EXP), e - 1, e))
    y = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step, torch.exp2(e).squeeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    starts, ids, lens_qs = s["starts"].tolist(), s["ids"].tolist(), list(zip(*_lens(case)))
    first = [starts[i] for i in ids]                                      # first cache row of every sequence
    last = [torch.arange(f + a - q, f + a, device=DEV) for f, (a, q) in zip(first, lens_qs)]
    if case["kind"] == "write":
        codes, scales = s["codes"].double(), s["scales"].double()
        at = torch.cat(last)
        y, e = _exact_codes(s["x"])
        codes[at], scales[at] = y.flatten(1), e
        return {"codes": codes, "scales": scales}
    if case["kind"] == "read":
        at = torch.cat(last)
        return s["codes"][at].double().view(len(at), -1, D) * s["scales"][at].double().unsqueeze(-1)
    counts = _rows(case)
    if case["kind"] == "update":
        begins, n = _cumulate([a for a, _ in lens_qs]), s["count"]
        at = torch.cat([s["rows_k"][o:o + m] - begins[b] + first[b]
                        for b, (o, m) in enumerate(zip(_cumulate(counts), counts))]) if n else s["rows_k"]
        angle = s["cos_sin"].double()[s["positions"][s["pos_idx"]]]
        turn = torch.complex(angle[:, :64], angle[:, 64:]).unsqueeze(1)
        held = s["v_codes"][at].double().view(n, -1, D) * s["v_scales"][at].double().unsqueeze(-1)
        dv = []
        for k, v in s["steps"]:
            k = k.double()
            z = torch.complex(k[..., :64].contiguous(), k[..., 64:].contiguous()) * turn
            ky, ke = _exact_codes(torch.cat([z.real, z.imag], -1))
            vy, ve = _exact_codes(v)
            now = vy * ve.unsqueeze(-1)
            dv.append(now - held)
            held = now
        out = {"dv_first": dv[0], "dv_second": dv[1]}
        for name, new in (("k_codes", ky.flatten(1)), ("k_scales", ke), ("v_codes", vy.flatten(1)), ("v_scales", ve)):
            out[name] = s[name].double()
            out[name][at] = new
        return out
    q, heads = s["q"].double(), s["q"].size(1)
    hkv = s["k_scales"].size(1)
    o = torch.zeros(s["count"], heads, D, dtype=torch.float64, device=DEV)
    cu_q, done = _cumulate([v for _, v in lens_qs]), 0
    for b, ((length, n_q), m) in enumerate(zip(lens_qs, counts)):
        if not m:
            continue
        held = slice(first[b], first[b] + length)
        rows = s["rows"][done:done + m].long()
        pos = rows - cu_q[b] + length - n_q
        away = (pos[:, None] - torch.arange(length, device=DEV)[None]).abs().double()
        seen = torch.ones_like(away, dtype=torch.bool)
        if s["ranges"] is not None:
            r, j = s["ranges"][rows].long(), torch.arange(length, device=DEV)
            seen = (j[None] >= r[:, :1]) & (j[None] < r[:, 1:])
        for h in range(heads):
            g = h // (heads // hkv)
            k = s["k_codes"][held, g * D:(g + 1) * D].double() * s["k_scales"][held, g:g + 1].double()
            v = s["v_codes"][held, g * D:(g + 1) * D].double() * s["v_scales"][held, g:g + 1].double()
            t = q[rows, h] @ k.T / math.sqrt(D)
            if s["cap"]:
                t = s["cap"] * torch.tanh(t / s["cap"])
            if s["slopes"] is not None:
                t = t - float(s["slopes"][h]) * away
            p = torch.softmax(t.masked_fill(~seen, -math.inf), -1)
            o[done:done + m, h] = torch.nan_to_num(p, nan=0.0) @ v
        done += m
    return o
