"""What a serving step needs around the quantized KV cache, as cases that can be timed: page tables and slot maps made from request lengths, and attention
of packed tokens with a window and first tokens that stay visible (sinks), or of trees of drafted tokens.

A case is a dict of plain values. ``op`` says what one pass does:

``reserve``
    ``QuantizedKVCache.reserve``: the page table of ``b`` requests brought from the lengths of the last step to those of this one. ``change``: "step" (every
    request one token longer) or "serve" (some end, some begin, some grow); ``window`` / ``sinks``: pages that no token sees any more are given back;
    ``shared``: every fourth request has its first pages in common with the one before; ``pool``: pages there are, as a share of those asked for.
``plan``
    ``.plan``: where the packed tokens of this step go, which position and sequence is each one's and, for trees, which tokens it sees.
``write``
    ``.plan``, the tokens' keys and values ``.store``d (``rope``: ``.rope_store`` of a fused projection's output), for trees the accepted path kept
    (``.keep``), and the written stretch read back.
``attend``
    ``.attend``.

``tokens``: how many each sequence brings. "one": one; "mixed": the first sequence ``s`` (a piece of its prompt), the others one; "prompts": up to ``s``;
"tree": trees of up to ``s`` drafted tokens (``shape``: "random", "chain", "star"; ``blank``: some of a tree's places are not used). ``ctx`` is the longest
sequence's length with its new tokens, ``ragged`` the share of it (and of ``s``) that others go down to, ``idle``: every 16th place of the batch is empty,
``pad``: rows behind the last sequence, as a captured step has them. "one" is called with a position for each sequence, the others with a plan.
"""
import math
import random

import numpy as np
import torch

own = False  # False: the operators in plain torch operations; True: the framework's

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32  # values that share a scale
CHUNK = 2048  # positions filled at a time while a cache is made


def _case(name, op, **kw):
    c = {"name": name, "op": op, "fmt": "q4_0", "dt": "bf16", "b": 1, "h": 32, "kv": 8, "hd": 128, "ctx": 512, "page": 0, "tokens": "one", "s": 1, "ragged": 1.0, "idle": False,
         "pad": 0, "shape": "random", "blank": False, "window": 0, "sinks": 0, "rope": False, "change": "step", "shared": False, "pool": 1.0}
    c.update(kw)
    return c


def listed():
    return [
        # page tables: between two decode steps of a server, where latency counts
        _case("reserve_step", "reserve", b=64, ctx=16384, page=64, ragged=0.02),
        # many long conversations that come, go and share their beginning; attention with a window lets go of what lies behind it
        _case("reserve_serve", "reserve", b=500, ctx=131072, page=64, ragged=0.05, change="serve", window=40000, sinks=100, shared=True, pool=1.1),
        # slot maps: drafted trees of a batch, and prompts of all lengths packed into one forward pass
        _case("plan_trees", "plan", b=48, ctx=8192, page=64, tokens="tree", s=61, ragged=0.4, idle=True, pad=100),
        _case("plan_prompts", "plan", b=200, ctx=8192, page=128, tokens="prompts", s=1500, ragged=0.01, pad=1000),
        # trees written as a decoder writes them, the accepted path kept
        _case("write_trees", "write", b=24, ctx=4096, page=64, tokens="tree", s=40, ragged=0.5, blank=True, rope=True),
        # packed prompts written
        _case("write_prompts", "write", fmt="q8_0", b=32, ctx=4096, page=128, tokens="prompts", s=2048, ragged=0.05, rope=True),
        # attention with a window and sinks: one token of one long conversation (the decoder's f32 queries), of a server's ragged batch, a piece of a prompt,
        # and a piece of a prompt beside other sequences' single tokens
        _case("sinks_token", "attend", dt="f32", ctx=8192, window=1024, sinks=4),
        _case("sinks_batch", "attend", b=64, ctx=16384, page=64, ragged=0.05, idle=True, window=4096, sinks=64),
        _case("sinks_prompt", "attend", fmt="q8_0", ctx=12288, tokens="prompts", s=2048, window=4096, sinks=128),
        _case("sinks_mixed", "attend", dt="f16", h=28, kv=4, hd=64, b=41, ctx=8000, page=32, tokens="mixed", s=777, ragged=0.1, window=2500, sinks=7),
        # attention of drafted trees: one conversation, and a server's batch
        _case("tree_one", "attend", dt="f16", ctx=4096, tokens="tree", s=26),
        _case("tree_batch", "attend", b=24, ctx=8192, page=64, tokens="tree", s=63, ragged=0.2, blank=True, pad=17),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["reserve", "plan", "write", "write", "attend", "attend", "attend", "attend"])
        kv = rng.choice([1, 2, 3, 4, 8, 8])
        c = _case("", op, fmt=rng.choice(["q4_0", "q4_0", "q8_0"]), dt=rng.choice(["f32", "f16", "bf16", "bf16"]), b=_log_int(rng, 1, 64), kv=kv, h=kv * rng.choice([1, 2, 4, 4, 5, 7, 8]),
                  hd=rng.choice([64, 128, 128]), page=rng.choice([0, 0, 32, 64, 128]), ragged=round(rng.uniform(0.02, 1.0), 3), idle=rng.random() < 0.3)
        del c["name"]
        if op == "reserve":
            c.update(b=_log_int(rng, 1, 500), ctx=_log_int(rng, 1, 131072), page=rng.choice([32, 64, 64, 128, 256]), change=rng.choice(["step", "serve"]),
                     shared=rng.random() < 0.3, pool=round(rng.uniform(0.7, 1.5), 3))
            if rng.random() < 0.4:
                c.update(window=_log_int(rng, 1, c["ctx"]), sinks=rng.choice([0, 1, 4, 100, 1000]))
            if 64 <= c["b"] * (c["ctx"] // c["page"]) <= 500 * 2048:
                return c
            continue
        c["tokens"] = rng.choice(["prompts", "tree"] if op in ("plan", "write") else ["one", "one", "mixed", "prompts", "tree", "tree"])
        if c["tokens"] == "tree":
            c["s"] = _log_int(rng, 1, 256) if rng.random() < 0.3 else rng.randint(2, 64)
            c["ctx"] = c["s"] + _log_int(rng, 1, 16384)
            c["shape"], c["blank"] = rng.choice(["random", "random", "chain", "star"]), rng.random() < 0.3
        elif c["tokens"] == "one":
            c["ctx"] = _log_int(rng, 1, 65536)
        else:
            c["s"] = _log_int(rng, 2, 2048)
            c["ctx"] = c["s"] + rng.choice([0, 1]) * _log_int(rng, 1, 8192)
        if c["tokens"] != "one":
            c["pad"] = rng.choice([0, 0, _log_int(rng, 1, 100)])
        if op == "write":
            c["rope"] = rng.random() < 0.6
        if op == "attend" and (c["tokens"] != "tree" or rng.random() < 0.3):
            c.update(window=_log_int(rng, c["s"] if c["tokens"] == "tree" else 1, 2 * c["ctx"]), sinks=rng.choice([0, 1, 4, 31, 64, 100, 1000]))
        if op == "plan":
            c["b"], c["ctx"] = _log_int(rng, 1, 300), c["s"] + _log_int(rng, 100, 8192)
        starts, counts = _requests(c)
        total = sum(counts)
        if total == 0 or total + c["pad"] > 65536 * 4 or c["b"] * c["kv"] * c["ctx"] * c["hd"] > 64 * 8 * 16384 * 128 and op != "plan":
            continue
        w = work(c)
        if op == "write" and (w["bytes"] > work(listed()[5])["bytes"] or c["b"] * c["s"] * c["kv"] * c["hd"] > 32 * 2048 * 8 * 128):
            continue
        if op == "attend" and (w["flops"] > work(listed()[8])["flops"] or w["bytes"] > work(listed()[7])["bytes"]):
            continue
        if op == "plan" and w["bytes"] > 8 * work(listed()[3])["bytes"]:
            continue
        return c


def _share(c, i, turn):
    return c["ragged"] + (1 - c["ragged"]) * ((i * turn + 0.5) % 1.0) if i else 1.0


def _requests(c, seed=0):
    """Positions that every sequence has in the cache, and new tokens that it brings. Slot maps hold nothing but these: there they differ from seed to seed."""
    starts, counts, rng = [], [], random.Random(seed)
    for i in range(c["b"]):
        if c["tokens"] in ("tree", "prompts"):
            n = max(1, int(c["s"] * _share(c, i, 0.7548776662)))
        else:
            n = c["s"] if c["tokens"] == "mixed" and i == 0 else 1
        length = max(n, int(c["ctx"] * _share(c, i, 0.6180339887)))
        if c["idle"] and i % 16 == 5:
            n, length = 0, 0
        starts.append(length - n - (rng.randint(0, length - n) if c["op"] == "plan" else 0)), counts.append(n)
    return starts, counts


def _longest(c):
    return c["s"] if c["tokens"] in ("tree", "prompts", "mixed") else 1


def _parents(c, seed):
    """A parent for every packed token: its index in its own tree, -1 for a child of what is in the cache, -2 for a place that is not used."""
    rng = random.Random(seed * 7919 + 1)
    out = []
    for n in _requests(c)[1]:
        for i in range(n):
            if c["blank"] and i > n * 0.8:
                out.append(-2)
            elif c["shape"] == "chain" or i == 0:
                out.append(i - 1)
            elif c["shape"] == "star":
                out.append(0)
            else:
                out.append(max(0, i - 1 - int(rng.expovariate(1 / 6))))
    return out + [-2] * c["pad"]


def _accepted(c, seed):
    """The last token of each tree that was taken over; -1: none."""
    rng = random.Random(seed * 104729 + 5)
    return [rng.randint(-1, max(0, int(n * 0.8) - 1)) if n else -1 for n in _requests(c)[1]]


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _kv_rows(g, c, *lead):
    """Keys (a few channels larger than the others, as after training) and values [*lead, kv, hd]."""
    gain = torch.exp(0.5 * torch.cos(torch.arange(c["hd"], device="cuda") * 2.4))
    shape = (*lead, c["kv"], c["hd"])
    return (_rand(g, *shape) * gain).to(DT[c["dt"]]), (_rand(g, *shape) * 0.7).to(DT[c["dt"]])


def _tables(c):
    """cos, sin [ctx, hd / 2]"""
    ang = torch.arange(c["ctx"], device="cuda")[:, None] / 10000.0 ** (torch.arange(0, c["hd"], 2, device="cuda") / c["hd"])[None]
    return ang.cos(), ang.sin()


def _reserve_inputs(c, seed):
    """The table of the last step (numpy int32), this step's lengths, the first position still seen, and how many pages there are."""
    rng = np.random.default_rng(seed)
    b, page = c["b"], c["page"]
    per = -(-c["ctx"] // page)
    top = np.array([max(1, int(c["ctx"] * _share(c, i, 0.6180339887))) for i in range(b)])
    if c["change"] == "step":
        old, new = top - 1, top
    else:
        kind = rng.integers(0, 8, b)  # 0: ends, 1: begins, else it grows by up to three pages
        old = np.where(kind == 1, 0, np.maximum(top - rng.integers(0, 3 * page + 1, b), 0))
        new = np.where(kind == 0, 0, top)
    first = np.maximum(new - c["window"], 0) if c["window"] else np.zeros_like(new)
    have = -(-old // page)
    pages = max(int(have.sum()), int(c["pool"] * int((-(-new // page)).sum())), 1)
    table = np.full((b, per), -1, np.int32)
    order = rng.permutation(pages).astype(np.int32)
    at = 0
    for i in range(b):
        n = int(have[i])
        table[i, :n] = order[at:at + n]
        at += n
        if c["shared"] and i % 4 == 3:
            same = min(n, int(have[i - 1])) // 2
            table[i, :same] = table[i - 1, :same]
    return table, new, first, pages


def prepare(case, seed):
    c = {"name": "", **case}
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    b, h, kv, hd = c["b"], c["h"], c["kv"], c["hd"]
    st = {"case": c}
    if own:
        from xn_b200.dtypes import GgmlDType
        from xn_b200.kv_cache import QuantizedKVCache

        def make(heads, dim, pages):
            paging = {"page_size": c["page"], "num_pages": pages} if c["page"] else {}
            return QuantizedKVCache(GgmlDType.Q4_0 if c["fmt"] == "q4_0" else GgmlDType.Q8_0, b, heads, c["ctx"], dim, torch.device("cuda"), **paging)
    if c["op"] == "reserve":
        table, new, first, pages = _reserve_inputs(c, seed)
        st["table"], st["length"], st["pages"] = torch.from_numpy(table).cuda(), torch.from_numpy(new).cuda(), pages
        st["first"] = torch.from_numpy(first).cuda() if c["window"] else None
        if own:
            st["cache"] = make(1, 64, pages)
        return st
    starts, counts = _requests(c, seed)
    st["starts"], st["counts"] = starts, counts
    st["n"] = sum(counts) + c["pad"]
    st["pos"], st["count"] = torch.tensor(starts, device="cuda"), torch.tensor(counts, device="cuda")
    st["parents"] = torch.tensor(_parents(c, seed), dtype=torch.int32, device="cuda") if c["tokens"] == "tree" else None
    st["rounds"] = max(1, math.ceil(math.log2(_longest(c) + 1)))
    table, pages = None, b
    if c["page"]:
        per = -(-c["ctx"] // c["page"])
        pages = b * per
        table = torch.randperm(pages, generator=g, device="cuda").view(b, per).to(torch.int32)
    st["table"] = table
    if c["op"] == "plan":
        if own:
            st["cache"] = make(1, 64, pages)
            if c["page"]:
                st["cache"].page_table.copy_(table)
        return st
    if own:
        cache = make(kv, hd, pages)
        if c["page"]:
            cache.page_table.copy_(table)
    else:
        cache = _PlainCache(c, table)
    for at in range(0, c["ctx"], CHUNK):  # every slot is written to its end: past a sequence's length lies what an earlier one has left
        k, v = _kv_rows(g, c, b, min(CHUNK, c["ctx"] - at))
        cache.store(k, v, torch.full((b,), at, device="cuda"))
    st["cache"] = cache
    if c["op"] == "write":
        k, v = _kv_rows(g, c, st["n"])
        st["k"], st["v"] = k, v
        if c["rope"]:
            q = _rand(g, st["n"], h, hd).to(DT[c["dt"]])
            st["qkv"] = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], -1)  # a fused projection's output
            st["cos"], st["sin"] = _tables(c)
        st["node"] = torch.tensor(_accepted(c, seed), device="cuda") if c["tokens"] == "tree" else None
        return st
    if c["tokens"] == "one":
        st["q"] = (_rand(g, b, 1, h, hd) * 1.5).to(DT[c["dt"]])
        st["pos"] = torch.where(st["count"] > 0, st["pos"], -1)  # an empty place's is negative
    else:
        st["q"] = (_rand(g, st["n"], h, hd) * 1.5).to(DT[c["dt"]])
        if own:
            st["plan"] = cache.plan(st["pos"], st["count"], st["n"], _longest(c), st["parents"])
        elif c["tokens"] == "tree":
            st["plan"] = _plain_plan(st)
    return st


# ---- the plain form ------------------------------------------------------------------------------------------------------------------------------

def _quantise(x, fmt):
    """f32 [.., hd] -> codes [.., hd / 32, 32] (f32 whole numbers) and scales [.., hd / 32] f16."""
    x = x.unflatten(-1, (-1, BLOCK))
    if fmt == "q4_0":
        d = x.gather(-1, x.abs().argmax(-1, keepdim=True)) / -8
    else:
        d = x.abs().amax(-1, keepdim=True) / 127
    inv = torch.where(d == 0, 0.0, 1 / d)
    if fmt == "q4_0":
        code = (x * inv + 8.5).trunc().clamp(0, 15)
    else:
        y = x * inv
        code = y.trunc()
        code = code + torch.sign(y) * ((y - code).abs() >= 0.5)
    return code, d.squeeze(-1).half()


class _PlainCache:
    """Codes and scales as dense tensors: [b, ctx, kv, ..], or by pages [pages, page, kv, ..]; the last row of all is written where nothing is to be."""

    def __init__(self, c, table):
        self.c, self.table = c, table
        self.size = c["page"] if table is not None else c["ctx"]
        rows = (table.numel() if table is not None else c["b"]) * self.size + 1
        width = c["hd"] // 2 if c["fmt"] == "q4_0" else c["hd"]
        kind = torch.uint8 if c["fmt"] == "q4_0" else torch.int8
        self.codes = [torch.zeros((rows, c["kv"], width), dtype=kind, device="cuda") for _ in range(2)]
        self.scales = [torch.zeros((rows, c["kv"], c["hd"] // BLOCK), dtype=torch.float16, device="cuda") for _ in range(2)]

    def rows(self, sequence, where):
        """The rows of positions, any shape (the last one for what is not there)."""
        at = where.clamp(0, self.c["ctx"] - 1)
        page = sequence.expand_as(at) if self.table is None else self.table[sequence.expand_as(at), at // self.size].long()
        return torch.where((where >= 0) & (where < self.c["ctx"]), page * self.size + at % self.size, -1)

    def put(self, k, v, rows):
        for i, x in enumerate((k, v)):
            code, d = _quantise(x.float(), self.c["fmt"])
            code = code.flatten(-2)
            code = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8) if self.c["fmt"] == "q4_0" else code.to(torch.int8)
            self.codes[i][rows], self.scales[i][rows] = code, d

    def store(self, k, v, pos):
        self.put(k, v, self.rows(torch.arange(k.shape[0], device="cuda")[:, None], pos[:, None] + torch.arange(k.shape[1], device="cuda")))

    def get(self, rows):
        """f32 keys and values [*rows, kv, hd]"""
        out = []
        for codes, scales in zip(self.codes, self.scales):
            code, d = codes[rows], scales[rows]
            if self.c["fmt"] == "q4_0":
                code = torch.stack([code & 15, code >> 4], -1).flatten(-2).float() - 8
            out.append((code.float().unflatten(-1, (-1, BLOCK)) * d.float()[..., None]).flatten(-2))
        return out


def _rotate(x, cos, sin):
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _plain_reserve(st):
    c, page, pages = st["case"], st["case"]["page"], st["pages"]
    table, length = st["table"], st["length"].clamp(0, c["ctx"])
    at = torch.arange(table.shape[1], device="cuda") * page
    needed = at < length[:, None]
    if st["first"] is not None:
        needed &= (at + page > st["first"][:, None]) | (at < c["sinks"])
    there = needed & (table >= 0) & (table < pages)
    used = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    used[torch.where(there, table, pages).flatten().long()] = 1
    order = torch.argsort(used[:pages], stable=True)  # the free pages first, in their order
    free = pages - used[:pages].sum()
    missing = needed & ~there
    rank = (missing.flatten().cumsum(0) - 1).view_as(table)
    taken = torch.where(missing & (rank < free), order[rank.clamp(0, pages - 1)].to(torch.int32), -1)
    new = torch.where(there, table, taken)
    short = needed & (new < 0)
    room = torch.where(short.any(1), short.int().argmax(1) * page, length)
    return [new, room, free - torch.minimum(free, missing.sum())]


def _plain_plan(st):
    """offsets, sequence, position, slot, which tokens of its tree a token sees (dense and as bits; None)"""
    c, pos, count, n, b = st["case"], st["pos"], st["count"], st["n"], st["case"]["b"]
    offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
    t = torch.arange(n, device="cuda")
    real = t < offsets[-1]
    sequence = torch.where(real, torch.searchsorted(offsets[1:], t, right=True), 0).clamp(max=b - 1)
    index = t - offsets[sequence]
    place = pos[sequence] + index
    position, sees, bits = place, None, None
    if c["tokens"] == "tree":
        longest = _longest(c)
        dense = torch.arange(longest, device="cuda")
        sees = dense == index[:, None]  # itself, and then its ancestors in steps of 1, 2, 4, ..
        up, ok = st["parents"].long(), real & (st["parents"] > -2) & (st["parents"] < index)
        for _ in range(st["rounds"]):
            to = torch.where(up >= 0, t - index + up, t)
            sees = sees | sees[to]
            ok = ok & ok[to]
            up = torch.where(up >= 0, up[to], up)
        real = real & ok
        sees = sees & real[:, None]
        position = pos[sequence] + sees.sum(1) - 1
        words = -(-longest // 32)
        padded = torch.zeros((n, words * 32), dtype=torch.int64, device="cuda")
        padded[:, :longest] = sees
        bits = (padded.view(n, words, 32) << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
    page = c["page"] or -(-c["ctx"] // 32) * 32
    slot = sequence * page + place
    if c["page"]:
        slot = st["table"][sequence, place.clamp(0, c["ctx"] - 1) // page].long() * page + place % page
    return [offsets, torch.where(t < offsets[-1], sequence, -1).to(torch.int32), torch.where(real, position, -1), torch.where(real, slot, -1), bits, sees]


def _plain_write(st):
    c, cache = st["case"], st["cache"]
    h, kv, hd = c["h"], c["kv"], c["hd"]
    offsets, sequence, position, _, _, sees = _plain_plan(st)
    real = position >= 0
    place = torch.where(real, st["pos"][sequence] + torch.arange(st["n"], device="cuda") - offsets[sequence], -1)
    rows = cache.rows(sequence.long(), place)
    q = []
    if c["rope"]:
        x = st["qkv"].float().unflatten(-1, (-1, hd))
        cos, sin = (t[position.clamp(min=0)][:, None] * real[:, None, None] for t in (st["cos"], st["sin"]))
        q = [_rotate(x[:, :h], cos, sin).to(DT[c["dt"]])]
        cache.put(_rotate(x[:, h:h + kv], cos, sin), x[:, h + kv:], rows)
    else:
        cache.put(st["k"], st["v"], rows)
    s = _longest(c)
    after = []
    if c["tokens"] == "tree":
        node = st["node"]
        path = sees[(offsets[:-1] + node.clamp(min=0)).clamp(max=st["n"] - 1)] & ((node >= 0) & (node < st["count"]))[:, None]  # [b, s]
        rank = path.cumsum(1) - 1
        which = torch.arange(c["b"], device="cuda")[:, None]
        source = cache.rows(which, torch.where(path, st["pos"][:, None] + torch.arange(s, device="cuda"), -1))
        target = cache.rows(which, torch.where(path, st["pos"][:, None] + rank, -1))
        for held in (*cache.codes, *cache.scales):
            held[target] = held[source]
        after = [st["pos"] + path.sum(1)]
    back = cache.rows(torch.arange(c["b"], device="cuda")[:, None], st["pos"][:, None] + torch.arange(s, device="cuda"))
    out = [x * (back >= 0)[..., None, None] for x in cache.get(back)]
    return q + after + [x.transpose(1, 2) for x in out]


def _plain_attend(st):
    c, cache = st["case"], st["cache"]
    h, kv, hd = c["h"], c["kv"], c["hd"]
    q_all = st["q"].reshape(-1, h, hd)
    out = torch.zeros((q_all.shape[0], h, hd), dtype=torch.float32, device="cuda")
    at = 0
    for i, (start, n) in enumerate(zip(st["starts"], st["counts"])):
        if c["tokens"] == "one":
            at = i
        if n == 0:
            continue
        end, low = start + n, max(0, start - c["window"] + 1) if c["window"] else 0
        where = torch.cat([torch.arange(0, min(c["sinks"], low), device="cuda"), torch.arange(low, end, device="cuda")])
        tree = st["plan"][5][at:at + n, :n] if c["tokens"] == "tree" else None
        p = start + (tree.sum(1) - 1 if tree is not None else torch.arange(n, device="cuda"))[:, None]
        seen = where <= p
        if c["window"]:
            seen = seen & ((where > p - c["window"]) | (where < c["sinks"]))
        if tree is not None:
            seen = torch.cat([seen[:, :-n] & tree.any(1, keepdim=True), tree], 1)
        k, v = (x.transpose(0, 1) for x in cache.get(cache.rows(torch.full_like(where, i), where)))
        q = q_all[at:at + n].float().view(n, kv, h // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)
        score = (q @ k.transpose(-1, -2) * (1 / math.sqrt(hd))).view(kv, h // kv, n, -1)
        score = torch.where(seen, score, -torch.inf)
        top = score.amax(-1, keepdim=True)
        weight = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
        total = weight.sum(-1, keepdim=True)
        got = (weight.view(kv, -1, where.numel()) @ v).view(kv, h // kv, n, hd) / torch.where(total == 0, 1.0, total)
        out[at:at + n] = got.permute(2, 0, 1, 3).reshape(n, h, hd)
        at += n
    return out.view(st["q"].shape).to(st["q"].dtype)


def run(st):
    c = st["case"]
    if not own:
        if c["op"] == "plan":
            return [x for x in _plain_plan(st)[:5] if x is not None]
        return {"reserve": _plain_reserve, "write": _plain_write, "attend": _plain_attend}[c["op"]](st)
    cache = st["cache"]
    if c["op"] == "reserve":
        room, free = cache.reserve(st["length"], first=st["first"], sinks=c["sinks"], table=st["table"])
        return [cache.page_table, room, free]
    if c["op"] == "attend":
        return cache.attend(st["q"], st["pos"] if c["tokens"] == "one" else st["plan"], window=c["window"], sinks=c["sinks"])
    plan = cache.plan(st["pos"], st["count"], st["n"], _longest(c), st["parents"])
    if c["op"] == "plan":
        return [x for x in (plan.offsets, plan.sequence, plan.position, plan.slot, plan.sees) if x is not None]
    out = []
    if c["rope"]:
        out.append(cache.rope_store(st["qkv"], st["cos"], st["sin"], plan, c["h"]))
    else:
        cache.store(st["k"], st["v"], plan)
    if c["tokens"] == "tree":
        out.append(cache.keep(plan, st["node"]))
    return out + list(cache.load(st["pos"], _longest(c), dtype=torch.float32))


def work(case):
    c = {"name": "", **case}
    e = {"f32": 4, "f16": 2, "bf16": 2}[c["dt"]]
    b = c["b"]
    if c["op"] == "reserve":
        cells = b * -(-c["ctx"] // c["page"])
        return {"bytes": 8 * cells + (24 if c["window"] else 16) * b, "flops": 4 * cells}
    starts, counts = _requests(c)
    n = sum(counts) + c["pad"]
    words = -(-_longest(c) // 32)
    maps = 24 * b + n * (20 + (4 + 4 * words if c["tokens"] == "tree" else 0))
    if c["op"] == "plan":
        return {"bytes": maps, "flops": 8 * n}
    row = (c["hd"] // 2 if c["fmt"] == "q4_0" else c["hd"]) + c["hd"] // 16  # codes and scales of one head's position
    if c["op"] == "write":
        new, back = 2 * c["kv"] * n, 2 * c["kv"] * b * _longest(c)
        rotated = 2 * n * c["h"] * c["hd"] * e if c["rope"] else 0
        return {"bytes": new * (c["hd"] * e + row) + back * (row + c["hd"] * 4) + rotated + maps, "flops": 6 * (new + back) * c["hd"]}
    read, pairs = 0, 0
    for start, k in zip(starts, counts):
        if k == 0:
            continue
        w, end = c["window"] or start + k, start + k
        low = max(0, start - w + 1)
        read += end - low + min(c["sinks"] if c["window"] else 0, low)
        for i in range(k):
            p = start + (int(math.log2(i + 1)) if c["tokens"] == "tree" else i)
            low = max(0, p - w + 1)
            pairs += p + 1 - low + min(c["sinks"] if c["window"] else 0, low)
    return {"bytes": 2 * c["kv"] * read * row + 2 * n * c["h"] * c["hd"] * e, "flops": 4 * c["h"] * c["hd"] * pairs}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------------------------

def _stands_for(x, fmt):
    """The values, in 64 bits, that the block format holds for x [.., hd]. The format is defined by f32 arithmetic up to its codes."""
    y = x.to(torch.float32).reshape(-1, BLOCK)
    size = y.abs()
    if fmt == "q4_0":
        first = (size == size.max(1, keepdim=True).values).int().cumsum(1).cumsum(1) == 1  # the first of equal magnitudes
        step = (y * first).sum(1, keepdim=True) * -0.125
        code = torch.minimum(torch.floor(y * torch.where(step != 0, step.reciprocal(), step) + 8.5), torch.full_like(y, 15)).double() - 8
    else:
        step = size.max(1, keepdim=True).values / 127
        z = (y * torch.where(step != 0, step.reciprocal(), step)).double()
        code = torch.where(z < 0, -torch.floor(0.5 - z), torch.floor(z + 0.5))
    return (code * step.half().double()).reshape(x.shape)


def _exact_reserve(c, seed):
    table, length, first, pages = _reserve_inputs(c, seed)
    page, out, room = c["page"], np.full_like(table, -1), []
    wanted = []
    for i in range(c["b"]):
        n = -(-int(length[i]) // page)
        keep = [j for j in range(n) if j * page < c["sinks"] or (j + 1) * page > int(first[i])]
        wanted.append(keep)
        for j in keep:
            if 0 <= table[i, j] < pages:
                out[i, j] = table[i, j]
    free = np.setdiff1d(np.arange(pages), out[out >= 0])
    at = 0
    for i, keep in enumerate(wanted):
        end = int(length[i])
        for j in keep:
            if out[i, j] < 0 and at < len(free):
                out[i, j] = free[at]
                at += 1
            elif out[i, j] < 0:
                end = j * page
                break
        room.append(end)
    return [torch.from_numpy(out), torch.tensor(room), torch.tensor(len(free) - at)]


def _paths(c, seed):
    """For every packed token its place in its sequence's tree and the list of tokens from the tree's root to it (None: no token)."""
    if c["tokens"] != "tree":
        return [[range(i + 1) for i in range(n)] for n in _requests(c)[1]]
    parents, out = iter(_parents(c, seed)), []
    for n in _requests(c)[1]:
        mine = []
        for i in range(n):
            up = next(parents)
            mine.append([i] if up == -1 else mine[up] + [i] if up >= 0 and mine[up] is not None else None)
        out.append(mine)
    return out


def _exact_plan(c, seed):
    starts, counts = _requests(c, seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    page = c["page"] or -(-c["ctx"] // 32) * 32
    per = -(-c["ctx"] // page)
    table = torch.randperm(c["b"] * per, generator=g, device="cuda").view(c["b"], per).tolist() if c["page"] else [[i] for i in range(c["b"])]
    words = -(-_longest(c) // 32)
    sequence, position, slot, sees = [], [], [], []
    paths = _paths(c, seed) if c["tokens"] == "tree" else None
    for i, n in enumerate(counts):
        for j in range(n):
            place, path = starts[i] + j, paths[i][j] if paths else None
            real = paths is None or path is not None
            sequence.append(i)
            position.append((starts[i] + len(path) - 1 if paths else place) if real else -1)
            slot.append(table[i][place // page] * page + place % page if real else -1)
            if paths:
                whole = sum(1 << x for x in path) if real else 0
                sees.append([((whole >> (32 * w)) + 2 ** 31) % 2 ** 32 - 2 ** 31 for w in range(words)])
    for x in (sequence, position, slot):
        x += [-1] * c["pad"]
    sees += [[0] * words] * c["pad"]
    offsets = [sum(counts[:i]) for i in range(len(counts))] + [sum(counts)]
    out = [torch.tensor(offsets), torch.tensor(sequence, dtype=torch.int32), torch.tensor(position), torch.tensor(slot)]
    return out + ([torch.tensor(sees, dtype=torch.int32)] if paths else [])


def exact(case, seed):
    c = {"name": "", **case}
    if c["op"] == "reserve":
        return _exact_reserve(c, seed)
    if c["op"] == "plan":
        return _exact_plan(c, seed)
    starts, counts = _requests(c)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    b, h, kv, hd, dt = c["b"], c["h"], c["kv"], c["hd"], DT[c["dt"]]
    n, s = sum(counts) + c["pad"], _longest(c)
    if c["page"]:
        torch.randperm(b * -(-c["ctx"] // c["page"]), generator=g, device="cuda")
    filled = []
    for at in range(0, c["ctx"], CHUNK):
        filled.append(_kv_rows(g, c, b, min(CHUNK, c["ctx"] - at)))
    paths = _paths(c, seed)
    if c["op"] == "write":
        new = _kv_rows(g, c, n)
        out, after = [], []
        turn = [torch.zeros((n, 1, hd // 2), dtype=torch.float64, device="cuda") for _ in range(2)]
        if c["rope"]:
            where, angle, t = [], [], 0
            for i in range(b):
                for path in paths[i]:
                    if path is not None:
                        where.append(t), angle.append(starts[i] + len(path) - 1)
                    t += 1
            where, angle = torch.tensor(where, device="cuda"), torch.tensor(angle, device="cuda")
            for to, table in zip(turn, _tables(c)):
                to[where] = table[angle][:, None].double()

            def turned(x, rounded=lambda y: y):
                a, z = x[..., :hd // 2].double(), x[..., hd // 2:].double()
                return torch.cat((rounded(a * turn[0]) - rounded(z * turn[1]), rounded(z * turn[0]) + rounded(a * turn[1])), -1)
            out.append(turned(_rand(g, n, h, hd).to(dt)))
            # Which code a key gets is defined by f32 arithmetic, its rotation's included: products and sums rounded once each. (In 64 bits throughout, 1 code in
            # 100000 of Q8_0 is another one, where a value lies next to the border of two.)
            new = (turned(new[0], lambda y: y.float().double()), new[1])
        accepted = _accepted(c, seed)
        back = [torch.zeros((b, s, kv, hd), dtype=torch.float64, device="cuda") for _ in range(2)]
        for x in range(2):
            held = _stands_for(new[x], c["fmt"])
            t = 0
            for i in range(b):
                end = min(starts[i] + s, c["ctx"])  # what lay there before
                for at in range(starts[i] // CHUNK * CHUNK, end, CHUNK):
                    low = max(at, starts[i])
                    back[x][i, low - starts[i]:at + CHUNK - starts[i]][:end - low] = _stands_for(filled[at // CHUNK][x][i, low - at:end - at], c["fmt"])
                fresh = [j for j in range(counts[i]) if paths[i][j] is not None]
                if fresh:
                    back[x][i, fresh] = held[[t + j for j in fresh]]
                if c["tokens"] == "tree" and accepted[i] >= 0 and paths[i][accepted[i]] is not None:
                    path = paths[i][accepted[i]]
                    back[x][i, :len(path)] = held[[t + j for j in path]]
                t += counts[i]
        if c["tokens"] == "tree":
            after = [torch.tensor([starts[i] + (len(paths[i][accepted[i]] or []) if accepted[i] >= 0 else 0) for i in range(b)])]
        return out + after + [x.transpose(1, 2) for x in back]
    shape = (b, 1, h, hd) if c["tokens"] == "one" else (n, h, hd)
    q = (_rand(g, *shape) * 1.5).to(dt).view(-1, h, hd)
    out = torch.zeros((q.shape[0], h, hd), dtype=torch.float64, device="cuda")
    where = torch.arange(c["ctx"], device="cuda")
    t = 0
    for i, (start, m) in enumerate(zip(starts, counts)):
        if c["tokens"] == "one":
            t = i
        if m == 0:
            continue
        hidden = torch.ones((m, start + m), dtype=torch.bool, device="cuda")
        if c["tokens"] == "tree":
            for j, path in enumerate(paths[i]):
                if path is None:
                    continue
                p = start + len(path) - 1
                hidden[j, max(0, p - c["window"] + 1) if c["window"] else 0:start] = False
                hidden[j, :min(start, c["sinks"])] = False
                hidden[j, [start + x for x in path]] = False
        else:
            last = (start + torch.arange(m, device="cuda"))[:, None]
            hidden = where[:start + m] > last
            if c["window"]:
                hidden |= (where[:start + m] <= last - c["window"]) & (where[:start + m] >= c["sinks"])
        none = hidden.all(1, keepdim=True)
        for j in range(kv):
            key, value = (torch.cat([_stands_for(x[w][i, :, j], c["fmt"]) for x in filled])[:start + m] for w in range(2))
            for head in range(j * (h // kv), (j + 1) * (h // kv)):
                logit = q[t:t + m, head].double() @ key.T / math.sqrt(hd)
                weight = torch.softmax(logit.masked_fill(hidden, -torch.inf).masked_fill(none, 0.0), 1).masked_fill(none, 0.0)
                out[t:t + m, head] = weight @ value
        t += m
    return out.view(shape)
