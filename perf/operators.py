"""The rotary positions and the paged 8-bit KV cache as calls whose time counts
for a user: listed() names them, draw() gives more of the same ranges,
prepare() makes one ready, run() makes one pass (in plain torch operations, or
with `own` through picolm_amd), exact() is the same result in 64 bits.

  tables   cos and sin of a run of positions, frequencies scaled for contexts
           longer than the trained one (angles in 64 bits)
  rope     q and k rows of any positions rotated by such tables, both pair
           layouts, all or part of a head
  store    rows appended to the cache (k rotated, k and v quantised, q rotated
           on the way), then the sequences' last rows read back as values
  attn     causal grouped-query attention of each sequence's last rows over
           its cached rows: single tokens, prompts, both mixed
  step     one layer of a serving step: append, then attention
  fork     sequences that share another's pages, then grow: allocation and
           copies of the shared last page
  compact  a cache with freed pages brought to its lowest page numbers

The cache.  A block is 32 tokens of one kv head; k and v of a block are int8
codes with one fp32 scale each (value = code * scale, scale = max|x| / 127).
A page is a multiple of 32 tokens of every layer and head:

  codes  int8 [n_pages][n_layers][n_kv_heads][page/32][2: k, v][Dp/32][1024]
  scales fp32 [n_pages][n_layers][n_kv_heads][page/32][2: k, v]

Dp is head_dim rounded up to 32.  A tile of 1024 codes holds 32 tokens x 32
elements in the order the matrix cores take: byte 256 g + 16 i + 8 h + j is
token 16 h + i, element 8 g + j of k, and token 16 (j / 4) + 4 g + j % 4,
element 16 h + i of v.  A sequence is a row of page numbers and a length; a
page counts the sequences that hold it (0: free), and new pages are the free
ones of the lowest numbers.

Appending rows to a block that has older ones keeps its scale where the new
rows fit; where they do not, the scale grows and the older codes are rounded
again to it.  Rotated values are rounded once to fp32, codes are rounded from
64-bit quotients.
"""
import math
import random

import torch

own = False

LLAMA, QWEN = 0, 1  # pairs (2i, 2i+1), pairs (i, i + rot/2)
BLOCK = 32


def listed():
    return [
        # the tables of a model at its full scaled context (Llama-3.2-1B's
        # head size and frequency base), built once when it is loaded
        _tables("tables_131072", 64, 5e5, "bands", 32.0, 8192, 1.0, 4.0, 0, 131072),
        # one generated token's rows: launch latency
        _rope("rope_token", 1, 32, 8, 64, 64, LLAMA, 8192),
        # a long prompt's rows, half of each head rotated (Qwen3-0.6B heads)
        _rope("rope_prompt", 8191, 16, 8, 128, 64, QWEN, 32768),
        # one token each of a batch (Qwen3-0.6B heads)
        _kv("store_tokens", "store", 64, 16, 8, 128, 64, (40, 8000), (1, 1), layout=QWEN, rot=128),
        # a few prompts at once (Llama-3.2-1B heads), new and continued
        _kv("store_prompts", "store", 5, 32, 8, 64, 64, (900, 4100), (700, 2100)),
        # a short chat turn's token (TinyLlama heads): latency
        _kv("attn_token_257", "attn", 1, 32, 4, 64, 64, (257, 257), (1, 1)),
        # a batch of tokens at many lengths (Qwen3-0.6B heads)
        _kv("attn_batch_64", "attn", 64, 16, 8, 128, 64, (1000, 8191), (1, 1)),
        # one token at a long context (Llama-3.2-1B heads)
        _kv("attn_token_130001", "attn", 1, 32, 8, 64, 128, (130001, 130001), (1, 1)),
        # prompts, one chunk each over what their sequences hold already
        _kv("attn_prompts", "attn", 3, 32, 8, 64, 64, (2000, 4001), (1000, 2047)),
        # a layer of a mixed step: two prompts among single tokens, a head
        # size between the usual ones (MHA, 80)
        _kv("step_mixed_d80", "step", 24, 32, 32, 80, 32, (30, 2000), (1, 1), prompts=2,
            prompt_rows=(200, 700), rot=80),
        # eight branches each of two prompts, a token further (TinyLlama,
        # every layer)
        _pages("fork_16", "fork", 18, 22, 4, 64, 64, (1500, 2040), parents=2, free=0.3),
        # a server's cache after half of its sequences ended (TinyLlama,
        # every layer)
        _pages("compact_48", "compact", 48, 22, 4, 64, 64, (300, 2040), parents=0, free=0.5),
    ]


def _case(name, kind, **kw):
    return dict({"name": name} if name else {}, kind=kind, **kw)


def _tables(name, rot, base, scaling, factor, orig, low, high, first, n):
    return _case(name, "tables", rot=rot, base=base, scaling=scaling, factor=factor, orig=orig,
                 low=low, high=high, first=first, n=n)


def _rope(name, rows, Hq, Hkv, D, rot, layout, n_pos):
    return _case(name, "rope", rows=rows, Hq=Hq, Hkv=Hkv, D=D, rot=rot, layout=layout,
                 n_pos=n_pos)


def _kv(name, kind, S, Hq, Hkv, D, page, lens, rows, prompts=0, prompt_rows=(1, 1), layout=LLAMA,
        rot=64, layers=1, lens_seed=7):
    return _case(name, kind, S=S, Hq=Hq, Hkv=Hkv, D=D, page=page, len_lo=lens[0], len_hi=lens[1],
                 rows_lo=rows[0], rows_hi=rows[1], prompts=prompts, prompt_lo=prompt_rows[0],
                 prompt_hi=prompt_rows[1], layout=layout, rot=rot, layers=layers,
                 lens_seed=lens_seed)


def _pages(name, kind, S, layers, Hkv, D, page, lens, parents, free, lens_seed=7):
    return _case(name, kind, S=S, layers=layers, Hkv=Hkv, D=D, page=page, len_lo=lens[0],
                 len_hi=lens[1], parents=parents, free=free, lens_seed=lens_seed)


# ---- more cases of the same ranges ------------------------------------------


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """Head sizes (the usual ones more often), kv heads, q heads."""
    D = rng.choice([64, 64, 64, 128, 128, 128, 32, 48, 80, 96, 100, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    return D, Hkv, Hkv * rng.choice([1, 2, 4, 5, 7, 8, 16])


def draw(rng):
    kind = rng.choice(["tables", "rope", "store", "store", "attn", "attn", "attn", "step", "fork",
                       "compact"])
    seed = rng.randrange(1 << 30)
    D, Hkv, Hq = _heads(rng)
    layout = rng.choice([LLAMA, QWEN])
    rot = rng.choice([D, D, D // 2])
    page = rng.choice([32, 64, 96, 128, 256])
    if kind == "tables":
        return _tables(None, rng.choice([32, 48, 64, 80, 96, 128]), rng.choice([1e4, 5e5, 1e6]),
                       rng.choice(["none", "linear", "ntk", "bands", "ramp"]),
                       rng.choice([2.0, 4.0, 8.0, 32.0]), rng.choice([2048, 4096, 8192]), 1.0,
                       rng.choice([4.0, 32.0]), rng.choice([0, 1, 100003, 900001]),
                       _log(rng, 100, 131072))
    if kind == "rope":
        most = min(8192, 200_000_000 // ((Hq + Hkv) * D * 8))
        return _rope(None, _log(rng, 1, most), Hq, Hkv, D, rot, layout, _log(rng, 4096, 65536))
    if kind == "store":
        if rng.random() < 0.5:
            hi = _log(rng, 64, 8192)
            return _kv(None, "store", _log(rng, 1, 96), Hq, Hkv, D, page, (1, hi), (1, 1),
                       layout=layout, rot=rot, lens_seed=seed)
        hi = _log(rng, 64, 4096)
        return _kv(None, "store", rng.randint(1, 6), Hq, Hkv, D, page, (hi // 3, hi),
                   (2, max(2, hi // 2)), layout=layout, rot=rot, lens_seed=seed)
    if kind == "attn":
        shape = rng.choice(["token", "batch", "prompt"])
        if shape == "token":
            n = _log(rng, 1, 131072)
            return _kv(None, "attn", 1, Hq, Hkv, D, page, (n, n), (1, 1), lens_seed=seed)
        if shape == "batch":
            hi = _log(rng, 64, 8192)
            return _kv(None, "attn", _log(rng, 2, 64), Hq, Hkv, min(D, 128), page,
                       (max(1, hi // 50), hi), (1, rng.choice([1, 1, 2, 5])), lens_seed=seed)
        hi = _log(rng, 200, 3000)
        return _kv(None, "attn", rng.randint(1, 4), min(Hq, 4 * Hkv), Hkv, min(D, 128), page,
                   (hi // 2, hi), (max(2, hi // 8), hi // 2), lens_seed=seed)
    if kind == "step":
        hi = _log(rng, 64, 2000)
        return _kv(None, "step", rng.randint(4, 24), Hq, Hkv, min(D, 128), page, (hi // 4, hi),
                   (1, 1), prompts=rng.randint(0, 3), prompt_rows=(2, max(2, hi // 3)),
                   layout=layout, rot=min(rot, 128), lens_seed=seed)
    layers = rng.choice([4, 12, 16, 22])
    hi = _log(rng, 200, 2040)
    if kind == "fork":
        parents = rng.randint(1, 3)
        return _pages(None, "fork", parents * rng.randint(2, 8), layers, min(Hkv, 4), min(D, 80),
                      page, (hi // 2, hi), parents, rng.uniform(0.0, 0.6), seed)
    return _pages(None, "compact", rng.randint(6, 48), layers, min(Hkv, 4), min(D, 64), page,
                  (hi // 4, hi), 0, rng.uniform(0.2, 0.8), seed)


# ---- what the sizes of a case come to ---------------------------------------


def _cdiv(a, b):
    return -(-a // b)


def _lens(c):
    """Lengths (the new rows included) and new rows of the sequences."""
    r = random.Random(c["lens_seed"])
    lens = [_log(r, c["len_lo"], c["len_hi"]) for _ in range(c["S"])]
    if c.get("prompts"):
        lo = min(c["prompt_hi"], c["len_hi"])
        lens[:c["prompts"]] = [_log(r, lo, c["len_hi"]) for _ in range(c["prompts"])]
    if "rows_lo" not in c:
        return lens, [0] * c["S"]
    rows = [_log(r, c["prompt_lo"], c["prompt_hi"]) if i < c["prompts"]
            else _log(r, c["rows_lo"], c["rows_hi"]) for i in range(c["S"])]
    return lens, [min(n, m) for n, m in zip(rows, lens)]


def _dp(c):
    return _cdiv(c["D"], 32) * 32


def _page_bytes(c):
    return c["layers"] * c["Hkv"] * c["page"] // BLOCK * 2 * (BLOCK * _dp(c) + 4)


def _moves(c):
    """Pages that compact moves: live ones at or above the number of live ones."""
    refs = _layout(c)[2]
    live = sum(1 for x in refs if x)
    return sum(1 for x in refs[live:] if x)


def work(c):
    if c["kind"] == "tables":
        return {"bytes": 4 * c["rot"] * c["n"], "flops": 40 * c["rot"] // 2 * c["n"]}
    if c["kind"] == "rope":
        n = c["rows"]
        return {"bytes": n * ((c["Hq"] + c["Hkv"]) * c["D"] * 8 + c["rot"] * 4 + 4),
                "flops": n * (c["Hq"] + c["Hkv"]) * c["rot"] * 3}
    lens, rows = _lens(c)
    if c["kind"] in ("store", "attn", "step"):
        n, kvd, qd = sum(rows), c["Hkv"] * c["D"], c["Hq"] * c["D"]
        scale = c["Hkv"] * 8 / BLOCK
        b = f = 0
        if c["kind"] != "attn":  # k and v read, codes written; q read and written; the table rows
            b += n * (kvd * 8 + 2 * kvd + scale + qd * 8 + c["rot"] * 4)
            f += n * (2 * kvd * 4 + (kvd + qd) * 3)
        if c["kind"] == "store":  # codes read, values written
            back = sum(min(x, y + 31) for x, y in zip(lens, rows))
            b += back * (2 * kvd + scale + kvd * 8)
            f += back * 2 * kvd
        else:
            b += sum(x * (2 * kvd + scale) for x, y in zip(lens, rows) if y) + n * qd * 8
            f += 4 * qd * sum(y * x - y * (y - 1) // 2 for x, y in zip(lens, rows))
        return {"bytes": b, "flops": f}
    table = 4 * c["S"] * _cdiv(max(lens) + 64, c["page"])
    if c["kind"] == "fork":
        copies = sum(1 for i in range(c["parents"], c["S"]) if lens[i % c["parents"]] % c["page"])
        return {"bytes": copies * 2 * _page_bytes(c) + 2 * table, "flops": 0}
    return {"bytes": _moves(c) * 2 * _page_bytes(c) + 2 * table + 8 * len(_layout(c)[2]),
            "flops": 0}


# ---- inputs -----------------------------------------------------------------


def _frequencies(c):
    """Angle per position of each pair, and what cos and sin are multiplied by."""
    rot, base, f = c["rot"], c["base"], c["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    if c["scaling"] == "ntk":
        base = base * f ** (rot / (rot - 2))
    theta = torch.pow(torch.tensor(base, dtype=torch.float64), -2 * i / rot)
    if c["scaling"] == "linear":
        return theta / f, 1.0
    if c["scaling"] == "bands":  # by how often a pair turns within the trained context
        turns = c["orig"] * theta / (2 * math.pi)
        s = ((turns - c["low"]) / (c["high"] - c["low"])).clamp(0, 1)
        return (1 - s) * theta / f + s * theta, 1.0
    if c["scaling"] == "ramp":  # the same, blended linearly over the pairs' numbers
        at = [rot * math.log(c["orig"] / (2 * math.pi * t)) / (2 * math.log(base))
              for t in (c["high"], c["low"])]
        lo, hi = max(0, math.floor(at[0])), min(rot - 1, math.ceil(at[1]))
        g = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return theta * (1 - g) + theta / f * g, 0.1 * math.log(f) + 1
    return theta, 1.0


def _layout(c):
    """Page numbers of each sequence, of pages that lie anywhere in the pool,
    and how many sequences hold each page.  fork: the sequences behind the
    parents are empty yet.  compact: some sequences have ended."""
    lens, _ = _lens(c)
    r = random.Random(c["lens_seed"] + 1)
    if c["kind"] == "fork":
        lens = [n if i < c["parents"] else 0 for i, n in enumerate(lens)]
    need = [_cdiv(n, c["page"]) for n in lens]
    spare = int(c["free"] * sum(need)) + 2 * c["S"] + 4 if c["kind"] == "fork" else 5
    ids = list(range(sum(need) + spare))
    r.shuffle(ids)
    refs, rows, at = [0] * len(ids), [], 0
    for i, n in enumerate(need):
        rows.append(ids[at:at + n])
        at += n
    if c["kind"] == "compact":
        gone = set(r.sample(range(c["S"]), int(c["free"] * c["S"])))
        rows = [[] if i in gone else p for i, p in enumerate(rows)]
        lens = [0 if i in gone else n for i, n in enumerate(lens)]
    for p in rows:
        for x in p:
            refs[x] = 1
    return rows, lens, refs


def _cuda(values, dtype):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(rows):
    s = [0]
    for n in rows:
        s.append(s[-1] + n)
    return s


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = {"case": c}

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if c["kind"] == "tables":
        # another seed starts at another position
        st["first"] = c["first"] + seed % 1009
        st["cos"], st["sin"] = (torch.empty(c["n"], c["rot"] // 2, device="cuda")
                                for _ in range(2))
        return st
    if c["kind"] == "rope":
        st["qkv"] = normal(c["rows"], (c["Hq"] + 2 * c["Hkv"]) * c["D"])
        st["pos"] = torch.randint(0, c["n_pos"], (c["rows"],), generator=g, device="cuda",
                                  dtype=torch.int32)
        st["q_out"] = torch.empty(c["rows"], c["Hq"] * c["D"], device="cuda")
        st["k_out"] = torch.empty(c["rows"], c["Hkv"] * c["D"], device="cuda")
        _prepare_tables(st, c["rot"], c["n_pos"])
        return st
    rows, lens, refs = _layout(c)
    P, B = len(refs), c["page"] // BLOCK
    width = _cdiv(max(max(lens), 1) + 64, c["page"])
    st["table"] = _cuda([p + [-1] * (width - len(p)) for p in rows], torch.int32)
    st["len"], st["refs"] = _cuda(lens, torch.int32), _cuda(refs, torch.int32)
    shape = (P, c["layers"], c["Hkv"], B, 2)
    st["codes"] = torch.empty(*shape, _dp(c) // 32, 1024, dtype=torch.int8, device="cuda")
    flat = st["codes"].view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        part = flat[at:at + (1 << 28)]
        part.copy_(torch.empty(part.shape, dtype=torch.float16, device="cuda")
                   .normal_(0, 36, generator=g).round_().clamp_(-127, 127))
    st["scales"] = (normal(*shape) * 0.2).exp() * 0.028
    if c["kind"] == "fork":
        st["parent"] = _cuda([-1 if i < c["parents"] else i % c["parents"]
                              for i in range(c["S"])], torch.int32)
        st["add"] = _cuda([0 if i < c["parents"] else 1 for i in range(c["S"])], torch.int32)
        st["status"] = _cuda([-1, -1], torch.int32)
        return st
    if c["kind"] == "compact":
        st["saved_table"], st["saved_refs"] = st["table"].clone(), st["refs"].clone()
        st["status"] = _cuda([-1, -1], torch.int32)
        return st
    n = _lens(c)[1]
    back = [min(x, y + 31) for x, y in zip(lens, n)]
    total = sum(n)
    st["n_rows"], st["longest"], st["most"] = total, max(lens), max(n)
    st["row_start"], st["back_start"] = (_cuda(_starts(x), torch.int32) for x in (n, back))
    qd, kvd = c["Hq"] * c["D"], c["Hkv"] * c["D"]
    st["n_back"] = sum(back)
    st["q"] = normal(total, qd)
    if c["kind"] != "attn":
        # some tokens are larger than their neighbours: scales that grow
        size = (normal(total, 1) * 0.3).exp()
        st["k"], st["v"] = normal(total, kvd) * size, normal(total, kvd) * size
        st["q_out"] = torch.empty_like(st["q"])
        st["back_k"], st["back_v"] = (torch.empty(st["n_back"], kvd, device="cuda")
                                      for _ in range(2))
        _prepare_tables(st, c["rot"], max(lens) + 1)
    st["out"] = torch.empty(total, qd, device="cuda")
    return st


def _prepare_tables(st, rot, n):
    theta = torch.pow(torch.tensor(1e4, dtype=torch.float64),
                      -torch.arange(0, rot, 2, dtype=torch.float64) / rot).cuda()
    angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * theta
    st["cos"], st["sin"], st["n_pos"] = angle.cos().float(), angle.sin().float(), n


# ---- one pass ---------------------------------------------------------------


def run(st):
    if own:
        return _RUN_OWN[st["case"]["kind"]](st, st["case"])
    return _RUN[st["case"]["kind"]](st, st["case"])


def _tables_plain(st, c):
    theta, m = _frequencies(c)
    pos = torch.arange(st["first"], st["first"] + c["n"], dtype=torch.float64, device="cuda")
    angle = pos[:, None] * theta.cuda()
    return (angle.cos() * m).float(), (angle.sin() * m).float()


def _rotate(x, cos, sin, layout, rot):
    """x [rows][heads][D] rotated by cos, sin [rows][rot/2]."""
    x = x.double()
    first = slice(0, rot, 2) if layout == LLAMA else slice(0, rot // 2)
    second = slice(1, rot, 2) if layout == LLAMA else slice(rot // 2, rot)
    a, b = x[..., first], x[..., second]
    c, s = cos.double()[:, None], sin.double()[:, None]
    out = x.clone()
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    return out.float()


def _rope_plain(st, c):
    n, D = c["rows"], c["D"]
    cos, sin = st["cos"][st["pos"].long()], st["sin"][st["pos"].long()]
    q, k, _ = st["qkv"].split([c["Hq"] * D, c["Hkv"] * D, c["Hkv"] * D], 1)
    return (_rotate(q.reshape(n, -1, D), cos, sin, c["layout"], c["rot"]).view(n, -1),
            _rotate(k.reshape(n, -1, D), cos, sin, c["layout"], c["rot"]).view(n, -1))


def _untile_k(t):
    """[..., Dp/32, 1024] codes of a block as [..., 32 tokens, Dp]."""
    lead, C = t.shape[:-2], t.shape[-2]
    n = len(lead)
    t = t.reshape(*lead, C, 4, 16, 2, 8)  # c g i h j
    return t.permute(*range(n), n + 3, n + 2, n, n + 1, n + 4).reshape(*lead, 32, C * 32)


def _untile_v(t):
    lead, C = t.shape[:-2], t.shape[-2]
    n = len(lead)
    t = t.reshape(*lead, C, 4, 16, 2, 2, 4)  # c g i h j/4 j%4
    return t.permute(*range(n), n + 4, n + 1, n + 5, n, n + 3, n + 2).reshape(*lead, 32, C * 32)


def _tile_k(x):
    lead, C = x.shape[:-2], x.shape[-1] // 32
    n = len(lead)
    x = x.reshape(*lead, 2, 16, C, 4, 8)  # h i c g j
    return x.permute(*range(n), n + 2, n + 3, n + 1, n, n + 4).reshape(*lead, C, 1024)


def _tile_v(x):
    lead, C = x.shape[:-2], x.shape[-1] // 32
    n = len(lead)
    x = x.reshape(*lead, 2, 4, 4, C, 2, 16)  # j/4 g j%4 c h i
    return x.permute(*range(n), n + 3, n + 1, n + 5, n + 4, n, n + 2).reshape(*lead, C, 1024)


def _places(st, row_start, total):
    """Sequence and position of every row of a batch: a sequence's rows are its last ones."""
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(row_start[1:].long(), row, right=True)
    return seq, st["len"][seq].long() - (row_start[seq + 1].long() - row)


def _append_plain(st, c):
    D, layer = c["D"], c["layers"] - 1
    n = st["n_rows"]
    seq, pos = _places(st, st["row_start"], n)
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _rotate(st["q"].view(n, -1, D), cos, sin, c["layout"], c["rot"]).view(n, -1)
    k = _rotate(st["k"].view(n, -1, D), cos, sin, c["layout"], c["rot"])
    x = torch.stack([k, st["v"].view(n, -1, D)], 2)  # [n][Hkv][2][D]
    x = torch.nn.functional.pad(x, (0, _dp(c) - D))
    key, block = torch.unique_consecutive(seq * (1 << 32) + pos // BLOCK, return_inverse=True)
    nb = key.numel()
    bs, bb = key >> 32, key & ((1 << 32) - 1)
    start = torch.full((nb,), BLOCK, device="cuda").scatter_reduce(0, block, pos % BLOCK, "amin")
    B = c["page"] // BLOCK
    page, b = st["table"][bs, bb // B].long(), bb % B
    tiles = st["codes"][page, layer, :, b]  # [nb][Hkv][2][C][1024]
    old = torch.stack([_untile_k(tiles[:, :, 0]), _untile_v(tiles[:, :, 1])], 2)
    old = old.double() * (start > 0).view(-1, 1, 1, 1, 1)
    was = st["scales"][page, layer, :, b] * (start > 0).view(-1, 1, 1)  # [nb][Hkv][2]
    most = x.abs().amax(-1)
    most = torch.zeros_like(was).scatter_reduce(0, block.view(-1, 1, 1).expand_as(most), most,
                                                "amax")
    now = torch.maximum(was, most / torch.full_like(most, 127))
    grown = (now > was)[..., None, None]
    ratio = torch.where(grown, old * was.double()[..., None, None]
                        / torch.where(now > 0, now, 1.0).double()[..., None, None], old)
    codes = ratio.round()
    div = torch.where(now > 0, now, torch.inf)[block][..., None].double()
    codes[block, :, :, pos % BLOCK] = (x.double() / div).round().clamp(-127, 127)
    codes = codes.to(torch.int8)
    st["codes"][page, layer, :, b] = torch.stack([_tile_k(codes[:, :, 0]), _tile_v(codes[:, :, 1])],
                                                 2)
    st["scales"][page, layer, :, b] = now
    return q


def _values(st, c, width):
    """k and v [S][Hkv][tokens][D] of the first `width` pages of every sequence."""
    layer, D = c["layers"] - 1, c["D"]
    page = st["table"][:, :width].long().clamp(min=0)
    codes, scales = st["codes"][page, layer], st["scales"][page, layer]
    S = page.shape[0]

    def of(t, s):  # [S][width][Hkv][B][32][Dp]
        x = t.float() * s[..., None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(S, c["Hkv"], -1, _dp(c))[..., :D]

    return (of(_untile_k(codes[:, :, :, :, 0]), scales[..., 0]),
            of(_untile_v(codes[:, :, :, :, 1]), scales[..., 1]))


def _store_plain(st, c):
    q = _append_plain(st, c)
    seq, pos = _places(st, st["back_start"], st["n_back"])
    B, layer, D = c["page"] // BLOCK, c["layers"] - 1, c["D"]
    key, block = torch.unique_consecutive(seq * (1 << 32) + pos // BLOCK, return_inverse=True)
    bs, bb = key >> 32, key & ((1 << 32) - 1)
    page, b = st["table"][bs, bb // B].long(), bb % B
    codes, scales = st["codes"][page, layer, :, b], st["scales"][page, layer, :, b]
    k = _untile_k(codes[:, :, 0]).float() * scales[:, :, 0, None, None]
    v = _untile_v(codes[:, :, 1]).float() * scales[:, :, 1, None, None]
    n = st["n_back"]
    return {"q": q, "k": k[block, :, pos % BLOCK][..., :D].reshape(n, -1),
            "v": v[block, :, pos % BLOCK][..., :D].reshape(n, -1)}


def _attn_plain(st, c, q):
    n, G, D = st["n_rows"], c["Hq"] // c["Hkv"], c["D"]
    k, v = _values(st, c, _cdiv(st["longest"], c["page"]))
    S, T = k.shape[0], k.shape[2]
    seq, pos = _places(st, st["row_start"], n)
    at = torch.arange(n, device="cuda") - st["row_start"][seq].long()
    most = st["most"]
    qs = q.new_zeros(S, most, c["Hkv"], G, D)
    qs[seq, at] = q.view(n, c["Hkv"], G, D)
    limit = torch.full((S, most), -1, device="cuda")
    limit[seq, at] = pos
    qs = qs.transpose(1, 2).reshape(S * c["Hkv"], most * G, D)
    s = torch.bmm(qs, k.reshape(-1, T, D).transpose(1, 2).contiguous())
    s = (s / math.sqrt(D)).view(S, c["Hkv"], most, G, T)
    seen = torch.arange(T, device="cuda") <= limit[:, None, :, None, None]
    s = s.masked_fill(~seen, -torch.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(S * c["Hkv"], most * G, T), v.reshape(-1, T, D).contiguous())
    o = o.view(S, c["Hkv"], most, G, D) / torch.where(total > 0, total, 1.0)
    return o.transpose(1, 2)[seq, at].reshape(n, -1)


def _step_plain(st, c):
    out = _attn_plain(st, c, _append_plain(st, c))
    return {"out": out, "codes": st["codes"], "scales": st["scales"]}


def _fork_plain(st, c):
    S, page = c["S"], c["page"]
    table, length, refs, parent = st["table"], st["len"], st["refs"], st["parent"].long()
    entry = torch.arange(table.shape[1], device="cuda")
    # each sequence with a parent gives its pages back and holds its parent's
    takes = (parent >= 0) & (parent != torch.arange(S, device="cuda"))
    source = torch.where(takes, parent, torch.arange(S, device="cuda"))
    taken, new_len = table[source], length[source]
    held = (entry < _pages_of(length, page)[:, None]) & takes[:, None]
    refs.scatter_add_(0, table.clamp(min=0).long().view(-1), -held.int().view(-1))
    held = (entry < _pages_of(new_len, page)[:, None]) & takes[:, None]
    refs.scatter_add_(0, taken.clamp(min=0).long().view(-1), held.int().view(-1))
    table.copy_(taken)
    length.copy_(new_len)
    # then room for the new tokens; who shares its last page gets a copy
    add = st["add"]
    have, want = _pages_of(length, page), _pages_of(length + add, page)
    grows = add > 0
    last = table.gather(1, (length // page).clamp(max=table.shape[1] - 1).long()[:, None])[:, 0]
    partial = grows & (length % page > 0)
    last = torch.where(partial, last, -1)
    before = ((last[:, None] == last[None, :]) & partial).tril(-1).sum(1)
    copies = partial & (refs[last.clamp(min=0).long()] - before > 1)
    count = torch.where(grows, want - have, 0) + copies
    first = count.cumsum(0) - count
    free = torch.argsort((refs > 0).int(), stable=True)
    short = (count.sum() - (refs == 0).sum()).clamp(min=0)
    over = want > table.shape[1]
    over = torch.where(over.any(), over.int().argmax() + 1, 0)
    fits = (short == 0) & (over == 0)
    copies, grows = copies & fits, grows & fits
    fresh = free[first.clamp(max=free.numel() - 1)]
    src, dst = last.clamp(min=0).long(), torch.where(copies, fresh, last.clamp(min=0).long())
    st["codes"][dst] = st["codes"][src]
    st["scales"][dst] = st["scales"][src]
    new = (entry >= have[:, None]) & (entry < want[:, None]) & grows[:, None]
    at = (first + copies)[:, None] + entry - have[:, None]
    got = torch.where(new, free[at.clamp(0, free.numel() - 1)].int(), table)
    got = torch.where((entry == (length // page)[:, None]) & copies[:, None], fresh[:, None].int(),
                      got)
    changed = got != table
    refs.scatter_add_(0, got.clamp(min=0).long().view(-1), changed.int().view(-1))
    refs.scatter_add_(0, src, -copies.int())
    table.copy_(got)
    length.add_(torch.where(grows, add, 0))
    st["status"].copy_(torch.stack([short, over]))
    return _page_state(st)


def _pages_of(n, page):
    return (n + page - 1) // page


def _page_state(st):
    return {n: st[n] for n in ("table", "len", "refs", "status", "codes", "scales")}


def _compact_plain(st, c):
    table, refs = st["table"], st["refs"]
    table.copy_(st["saved_table"])
    refs.copy_(st["saved_refs"])
    live = refs > 0
    n = live.sum()
    number = torch.arange(refs.numel(), device="cuda")
    moves, holes = torch.nonzero(live & (number >= n))[:, 0], torch.nonzero(~live & (number < n))[:, 0]
    st["codes"][holes] = st["codes"][moves]
    st["scales"][holes] = st["scales"][moves]
    to = number.clone()
    to[moves] = holes
    refs[holes] = refs[moves]
    refs[moves] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table))
    st["status"].copy_(torch.stack([n, torch.tensor(moves.numel(), device="cuda")]))
    return _page_state(st)


_RUN = {"tables": _tables_plain, "rope": _rope_plain, "store": _store_plain,
        "attn": lambda st, c: _attn_plain(st, c, st["q"]), "step": _step_plain,
        "fork": _fork_plain, "compact": _compact_plain}


# ---- the same through picolm_amd --------------------------------------------


def _p(t):
    return t.data_ptr()


def _package():
    import picolm_amd as P
    P.init(0)
    return P


def _cache(P, st, c):
    """The descriptors of the cache and its sequences, made once as a program does."""
    if "cache" not in st:
        st["cache"] = P.kv8.Cache(c["layers"], c["Hkv"], c["D"], st["refs"].numel(), c["page"],
                                  codes=_p(st["codes"]), scales=_p(st["scales"]))
        st["seqs"] = P.kv8.Sequences(c["S"], st["table"].shape[1], table=_p(st["table"]),
                                     lens=_p(st["len"]), refs=_p(st["refs"]))
        if "cos" in st:
            st["rope"] = P.rope.Tables(c["layout"], c["rot"], st["n_pos"], _p(st["cos"]),
                                       _p(st["sin"]))
    return st["cache"], st["seqs"]


def _tables_own(st, c):
    P = _package()
    spec = P.rope.Spec(c["rot"], c["base"], c["scaling"], c["factor"], c["orig"], c["low"],
                       c["high"])
    P.rope.make_tables(spec, st["first"], c["n"], _p(st["cos"]), _p(st["sin"]))
    return st["cos"], st["sin"]


def _rope_own(st, c):
    P = _package()
    tab = P.rope.Tables(c["layout"], c["rot"], st["n_pos"], _p(st["cos"]), _p(st["sin"]))
    width, q = st["qkv"].shape[1], _p(st["qkv"])
    P.rope.rotate(tab, c["rows"], _p(st["pos"]), c["D"],
                  q, c["Hq"], width, _p(st["q_out"]), c["Hq"] * c["D"],
                  q + 4 * c["Hq"] * c["D"], c["Hkv"], width, _p(st["k_out"]), c["Hkv"] * c["D"])
    return st["q_out"], st["k_out"]


def _append_own(P, st, c):
    cache, seqs = _cache(P, st, c)
    P.kv8.append(cache, seqs, c["layers"] - 1, st["n_rows"], _p(st["row_start"]), _p(st["k"]),
                 _p(st["v"]), rope=st["rope"], q=_p(st["q"]), n_heads=c["Hq"],
                 q_out=_p(st["q_out"]))


def _store_own(st, c):
    P = _package()
    _append_own(P, st, c)
    P.kv8.fetch(st["cache"], st["seqs"], c["layers"] - 1, st["n_back"], _p(st["back_start"]),
                _p(st["back_k"]), _p(st["back_v"]))
    return {"q": st["q_out"], "k": st["back_k"], "v": st["back_v"]}


def _attn_own(st, c):
    P = _package()
    cache, seqs = _cache(P, st, c)
    P.kv8.attend(cache, seqs, c["layers"] - 1, c["Hq"], st["n_rows"], _p(st["row_start"]),
                 _p(st["q"]), _p(st["out"]))
    return st["out"]


def _step_own(st, c):
    P = _package()
    _append_own(P, st, c)
    P.kv8.attend(st["cache"], st["seqs"], c["layers"] - 1, c["Hq"], st["n_rows"],
                 _p(st["row_start"]), _p(st["q_out"]), _p(st["out"]))
    return {"out": st["out"], "codes": st["codes"], "scales": st["scales"]}


def _fork_own(st, c):
    P = _package()
    cache, seqs = _cache(P, st, c)
    P.kv8.fork(cache, seqs, _p(st["parent"]))
    P.kv8.extend(cache, seqs, _p(st["add"]), _p(st["status"]))
    return _page_state(st)


def _compact_own(st, c):
    P = _package()
    cache, seqs = _cache(P, st, c)
    # back to the saved sequences
    P.check(P.lib.plh_memcpy_dtod(_p(st["table"]), _p(st["saved_table"]), st["table"].numel() * 4),
            "plh_memcpy_dtod")
    P.check(P.lib.plh_memcpy_dtod(_p(st["refs"]), _p(st["saved_refs"]), st["refs"].numel() * 4),
            "plh_memcpy_dtod")
    P.kv8.compact(cache, seqs, _p(st["status"]))
    return _page_state(st)


_RUN_OWN = {"tables": _tables_own, "rope": _rope_own, "store": _store_own, "attn": _attn_own,
            "step": _step_own, "fork": _fork_own, "compact": _compact_own}


# ---- 64-bit results ---------------------------------------------------------


def _turned(x, angle_cos, angle_sin, layout, rot):
    """Rows x [n][H][D] turned pair by pair as complex numbers, rounded to fp32."""
    x = x.to(torch.float64).clone()
    part = x[..., :rot]
    if layout == LLAMA:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], -1, 2).contiguous())
    else:
        z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous())
    z = z * torch.complex(angle_cos.double(), angle_sin.double())[:, None]
    x[..., :rot] = (torch.view_as_real(z).flatten(-2) if layout == LLAMA
                    else torch.cat([z.real, z.imag], -1))
    return x.float().double()


def _token_codes(st, c, kind, s, n):
    """Codes [Hkv][n][D] and scales [Hkv][n] of sequence s's first n tokens, token by token."""
    t = torch.arange(n, device="cuda")
    page = st["table"][s].long()[t // c["page"]]
    b = t % c["page"] // 32
    u, d = (t % 32)[:, None], torch.arange(c["D"], device="cuda")[None]
    if kind == 0:
        byte = d % 32 // 8 * 256 + u % 16 * 16 + u // 16 * 8 + d % 8
    else:
        byte = u % 16 // 4 * 256 + d % 16 * 16 + d % 32 // 16 * 8 + u // 16 * 4 + u % 4
    layer = c["layers"] - 1
    heads = torch.arange(c["Hkv"], device="cuda")[:, None]
    codes = st["codes"][page[None, :, None], layer, heads[..., None], b[None, :, None], kind,
                        (d // 32)[None], byte[None]]
    return codes, st["scales"][page[None], layer, heads, b[None], kind]


def _exact_cache(st, c):
    """[per sequence] codes and scales after the append, by k and v; and the rotated q."""
    D, sizes, n_new = c["D"], st["len"].tolist(), st["row_start"].tolist()
    q = st["q"].double().view(-1, c["Hq"], D).clone()
    kept = []
    for s, n in enumerate(sizes):
        a, z = n_new[s], n_new[s + 1]
        first = n - (z - a)
        pair = [[t.clone() for t in _token_codes(st, c, kind, s, n)] for kind in (0, 1)]
        if c["kind"] != "attn" and z > a:
            cos, sin = st["cos"][first:n], st["sin"][first:n]
            q[a:z] = _turned(st["q"][a:z].view(z - a, -1, D), cos, sin, c["layout"], c["rot"])
            new = (_turned(st["k"][a:z].view(z - a, -1, D), cos, sin, c["layout"], c["rot"]),
                   st["v"][a:z].double().view(z - a, -1, D))
            for kind in (0, 1):
                codes, scales = pair[kind][0].double(), pair[kind][1].double()
                rows = new[kind].transpose(0, 1)  # [Hkv][rows][D]
                for lo in range(first // 32 * 32, n, 32):
                    at, end = max(lo, first), min(lo + 32, n)
                    part = rows[:, at - first:end - first]
                    need = (part.abs().amax((1, 2)) / 127).float().double()
                    if at > lo:
                        was = scales[:, lo]
                        grow = (need > was)[:, None, None]
                        again = torch.round(codes[:, lo:at] * was[:, None, None]
                                            / need.clamp(min=1e-300)[:, None, None])
                        codes[:, lo:at] = torch.where(grow, again, codes[:, lo:at])
                        need = torch.maximum(need, was)
                    scales[:, lo:end] = need[:, None]
                    codes[:, at:end] = torch.round(part / need.clamp(min=1e-300)[:, None, None]
                                                   ).clamp(-127, 127)
                pair[kind] = [codes, scales]
        kept.append(pair)
    return kept, q


def _exact_attention(st, c, kept, q):
    G, starts = c["Hq"] // c["Hkv"], st["row_start"].tolist()
    out = torch.zeros(st["n_rows"], c["Hq"], c["D"], dtype=torch.float64, device="cuda")
    for s, n in enumerate(st["len"].tolist()):
        a, z = starts[s], starts[s + 1]
        if z == a:
            continue
        hidden = (torch.arange(n, device="cuda")[None]
                  > torch.arange(n - (z - a), n, device="cuda")[:, None])
        for h in range(c["Hq"]):
            k, v = (kept[s][kind][0][h // G].double() * kept[s][kind][1][h // G].double()[:, None]
                    for kind in (0, 1))
            w = (q[a:z, h] @ k.T.contiguous() / math.sqrt(c["D"])).masked_fill(hidden, -torch.inf)
            out[a:z, h] = torch.softmax(w, -1) @ v
    return out.view(st["n_rows"], -1)


def exact(c, seed):
    if c["kind"] in ("fork", "compact"):
        return None  # whole numbers and copies
    st = prepare(c, seed)
    if c["kind"] == "tables":
        pos = st["first"] + torch.arange(c["n"], dtype=torch.float64)
        theta, m = _frequencies(c)
        z = torch.polar(torch.full((1, 1), m, dtype=torch.float64),
                        torch.outer(pos, theta))
        return z.real.contiguous(), z.imag.contiguous()
    if c["kind"] == "rope":
        n, D, pos = c["rows"], c["D"], st["pos"].long()
        x = _turned(st["qkv"].view(n, -1, D), st["cos"][pos], st["sin"][pos], c["layout"],
                    c["rot"])
        return (x[:, :c["Hq"]].reshape(n, -1),
                x[:, c["Hq"]:c["Hq"] + c["Hkv"]].reshape(n, -1))
    if work(c)["flops"] > 1e13:
        return None
    kept, q = _exact_cache(st, c)
    if c["kind"] == "store":
        back = st["back_start"].tolist()
        rows = [[(p[0][:, len_ - m:].double() * p[1][:, len_ - m:].double()[..., None])
                 .transpose(0, 1).reshape(m, -1) for p in pair]
                for pair, len_, m in zip(kept, st["len"].tolist(),
                                         [b - a for a, b in zip(back, back[1:])])]
        return {"q": q.view(st["n_rows"], -1), "k": torch.cat([r[0] for r in rows]),
                "v": torch.cat([r[1] for r in rows])}
    out = _exact_attention(st, c, kept, q)
    return out if c["kind"] == "attn" else {"out": out, "codes": None, "scales": None}
