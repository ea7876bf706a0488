"""The quantized KV cache's operators, as cases that can be timed: the cache written and read back, and attention over it.

A case is a dict of plain values. ``op`` says what one pass does:

``store``
    ``QuantizedKVCache.rope_store`` (``rope``: the rotated queries come back) or ``.store`` of ``s`` new tokens of each of ``b`` sequences, then
    ``.load`` of the rows that were written.
``load``
    ``.load`` of the first ``ctx`` positions of every sequence.
``attend``
    ``.attend``: ``s`` query tokens of every sequence over its cache, ``ctx`` positions long with them (``ragged``: sequences of other lengths down
    to that share of ``ctx``; ``idle``: every 16th slot of the batch has no sequence).

``fmt`` is the cache's block format, ``dt`` the type of the activations, ``page`` the positions of a page (0: one run of memory per sequence),
``window`` a sliding window (0: none).
"""
import math

import torch

own = False  # False: the operators in plain torch operations; True: the framework's

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32  # values that share a scale
CHUNK = 2048  # positions filled at a time while a cache is made


def _case(name, op, fmt, dt, b, h, kv, hd, ctx, s=1, page=0, window=0, ragged=1.0, idle=False, rope=False):
    return {"name": name, "op": op, "fmt": fmt, "dt": dt, "b": b, "h": h, "kv": kv, "hd": hd, "ctx": ctx, "s": s, "page": page, "window": window,
            "ragged": ragged, "idle": idle, "rope": rope}


def listed():
    return [
        # the cache written as a decoder writes it, and read back
        _case("store_token", "store", "q4_0", "f32", 1, 32, 8, 128, 512, rope=True),                     # one token of one sequence: latency
        _case("store_drafts_paged", "store", "q8_0", "bf16", 13, 8, 2, 64, 1501, s=7, page=64, ragged=0.3),  # a few tokens of many sequences, anywhere
        _case("store_prompts", "store", "q4_0", "bf16", 8, 32, 8, 128, 4096, s=4096, rope=True),          # long prompts of a batch
        _case("load_prefix", "load", "q8_0", "f16", 1, 16, 4, 128, 1000),                                # a prefix handed to another program
        _case("load_batch", "load", "q4_0", "bf16", 16, 32, 8, 128, 8192, page=128),                      # a batch's caches for a dense kernel
        # one token of every sequence
        _case("attend_ctx512", "attend", "q4_0", "f32", 1, 32, 8, 128, 512),                             # the decoder's step, batch 1
        _case("attend_batch16", "attend", "q8_0", "f32", 16, 32, 8, 128, 200),                           # and batch 16
        _case("attend_ctx131072", "attend", "q4_0", "bf16", 1, 32, 8, 128, 131072),                      # one long document
        _case("attend_batch64_paged", "attend", "q4_0", "bf16", 64, 32, 8, 128, 16384, page=64, ragged=0.02, idle=True),  # a server's ragged batch
        # a few drafted tokens to verify, with a window
        _case("attend_drafts", "attend", "q8_0", "f16", 9, 28, 4, 64, 4001, s=5, window=3000, ragged=0.4),
        # prompts
        _case("attend_prompt", "attend", "q4_0", "bf16", 1, 32, 8, 128, 512, s=512),                     # a prompt of its own
        _case("attend_chunk", "attend", "q4_0", "bf16", 1, 32, 8, 128, 8192, s=2048),                    # a piece of a long prompt
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["store", "store", "load", "attend", "attend", "attend", "attend"])
        kv = rng.choice([1, 2, 3, 4, 8, 8])
        c = _case("", op, rng.choice(["q4_0", "q4_0", "q8_0"]), rng.choice(["f32", "f16", "bf16", "bf16"]), _log_int(rng, 1, 64), kv * rng.choice([1, 2, 4, 4, 5, 7, 8]), kv,
                  rng.choice([64, 128, 128]), 0, page=rng.choice([0, 0, 32, 64, 128]), ragged=round(rng.uniform(0.02, 1.0), 3), idle=rng.random() < 0.3)
        del c["name"]
        if op == "attend":
            kind = rng.random()
            if kind < 0.6:
                c["ctx"] = _log_int(rng, 1, 131072)
            elif kind < 0.8:  # drafts
                c["s"] = rng.randint(2, 9)
                c["ctx"] = _log_int(rng, c["s"], 16384)
            else:  # prompts, or pieces of them; a model in 16 bits
                c["s"] = _log_int(rng, 17, 2048)
                c["ctx"] = c["s"] + rng.choice([0, 1]) * _log_int(rng, 1, 6144)
                c["b"] = min(c["b"], 4)
                c["dt"] = rng.choice(["f16", "bf16"])
                c["ragged"], c["idle"] = 1.0, False
            if rng.random() < 0.2:
                c["window"] = _log_int(rng, 1, 2 * c["ctx"])
        else:
            c["ctx"], c["idle"] = _log_int(rng, 1, 16384), False
            if op == "store":
                c["s"] = min(c["ctx"], rng.choice([1, _log_int(rng, 2, 16), c["ctx"]]))
                c["rope"] = rng.random() < 0.5
        # no more memory to move than load_batch, attend_batch64_paged, or store_prompts, and no more products than attend_chunk
        rows = c["b"] * c["kv"] * (c["s"] if op == "store" else c["ctx"]) * c["hd"]
        if rows > (16 * 8 * 8192 * 128 if op == "load" else 8 * 8 * 4096 * 128 if op == "store" else 32 * 8 * 16384 * 128) or c["b"] * c["kv"] * c["ctx"] * c["hd"] > 64 * 8 * 16384 * 128:
            continue
        if c["b"] * c["h"] * c["s"] * c["ctx"] * c["hd"] > 32 * 2048 * 8192 * 128 and op == "attend":
            continue
        if 2 * rows < 4096:
            continue
        return c


def _lengths(c):
    """Positions in every sequence's cache, the new or asking tokens among them; 0: no sequence in this slot."""
    out = []
    for i in range(c["b"]):
        share = c["ragged"] + (1 - c["ragged"]) * ((i * 0.6180339887 + 0.5) % 1.0) if i else 1.0
        out.append(0 if c["idle"] and i % 16 == 5 else max(c["s"], int(c["ctx"] * share)))
    return out


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _kv_rows(g, c, n):
    """Keys (a few channels larger than the others, as after training) and values of `n` positions of every sequence: [b, n, kv, hd]."""
    gain = torch.exp(0.5 * torch.cos(torch.arange(c["hd"], device="cuda") * 2.4))
    shape = (c["b"], n, c["kv"], c["hd"])
    return (_rand(g, *shape) * gain).to(DT[c["dt"]]), (_rand(g, *shape) * 0.7).to(DT[c["dt"]])


def prepare(case, seed):
    c = {"name": "", **case}
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    b, h, kv, hd, s = c["b"], c["h"], c["kv"], c["hd"], c["s"]
    st = {"case": c}
    lengths = torch.tensor(_lengths(c), device="cuda")
    st["pos"] = torch.where(lengths > 0, lengths - s, -s)  # of the first of the s tokens; an idle slot's is negative
    table = None
    if c["page"]:
        per = -(-c["ctx"] // c["page"])
        table = torch.randperm(b * per, generator=g, device="cuda").view(b, per).to(torch.int32)
    if own:
        from xn_b200.dtypes import GgmlDType
        from xn_b200.kv_cache import QuantizedKVCache
        paging = {"page_size": c["page"], "num_pages": table.numel()} if c["page"] else {}
        cache = QuantizedKVCache(GgmlDType.Q4_0 if c["fmt"] == "q4_0" else GgmlDType.Q8_0, b, kv, c["ctx"], hd, torch.device("cuda"), **paging)
        if c["page"]:
            cache.page_table.copy_(table)
    else:
        cache = _PlainCache(c, table)
    for at in range(0, c["ctx"], CHUNK):  # every slot is written to its end: past a sequence's length lies what an earlier one has left
        k, v = _kv_rows(g, c, min(CHUNK, c["ctx"] - at))
        cache.store(k, v, torch.full((b,), at, device="cuda"))
    st["cache"] = cache
    if c["op"] == "store":
        k, v = _kv_rows(g, c, s)
        st["k"], st["v"] = k, v
        if c["rope"]:
            q = (_rand(g, b, s, h, hd)).to(DT[c["dt"]])
            st["qkv"] = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)  # a fused projection's output
            ang = torch.arange(c["ctx"], device="cuda")[:, None] / 10000.0 ** (torch.arange(0, hd, 2, device="cuda") / hd)[None]
            st["cos"], st["sin"] = ang.cos(), ang.sin()
    if c["op"] == "attend":
        st["q"] = (_rand(g, b, s, h, hd) * 1.5).to(DT[c["dt"]])
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
    """Codes and scales as dense tensors: [b, kv, ctx, ..], or by pages [pages, kv, page, ..]."""

    def __init__(self, c, table):
        self.c, self.table = c, table
        pages, size = (table.numel(), c["page"]) if table is not None else (c["b"], c["ctx"])
        width = c["hd"] // 2 if c["fmt"] == "q4_0" else c["hd"]
        kind = torch.uint8 if c["fmt"] == "q4_0" else torch.int8
        self.codes = [torch.zeros((pages, c["kv"], size, width), dtype=kind, device="cuda") for _ in range(2)]
        self.scales = [torch.zeros((pages, c["kv"], size, c["hd"] // BLOCK), dtype=torch.float16, device="cuda") for _ in range(2)]

    def _at(self, where):
        """Page and place in it of positions [b, n]."""
        row = torch.arange(where.shape[0], device="cuda")[:, None]
        if self.table is None:
            return row.expand_as(where), where
        return self.table[row, where // self.c["page"]].long(), where % self.c["page"]

    def store(self, k, v, pos):
        page, place = self._at(pos[:, None] + torch.arange(k.shape[1], device="cuda"))
        for i, x in enumerate((k, v)):
            code, d = _quantise(x.float(), self.c["fmt"])
            code = code.flatten(-2)
            code = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8) if self.c["fmt"] == "q4_0" else code.to(torch.int8)
            self.codes[i][page, :, place] = code
            self.scales[i][page, :, place] = d

    def load(self, start, length):
        """f32 keys and values [b, kv, length, hd] from position `start` on, a number or one for every sequence."""
        out = []
        for codes, scales in zip(self.codes, self.scales):
            if self.table is None and isinstance(start, int):
                code, d = codes[:, :, start:start + length], scales[:, :, start:start + length]
            else:
                first = start[:, None] if torch.is_tensor(start) else torch.full((self.c["b"], 1), start, device="cuda")
                page, place = self._at(first + torch.arange(length, device="cuda"))
                code, d = codes[page, :, place].transpose(1, 2), scales[page, :, place].transpose(1, 2)
            if self.c["fmt"] == "q4_0":
                code = torch.stack([code & 15, code >> 4], -1).flatten(-2).float() - 8
            out.append((code.float().unflatten(-1, (-1, BLOCK)) * d.float()[..., None]).flatten(-2))
        return out


def _rotate(x, cos, sin):
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _plain(st):
    c, cache = st["case"], st["cache"]
    b, h, kv, hd, s = c["b"], c["h"], c["kv"], c["hd"], c["s"]
    if c["op"] == "load":
        return [x.to(DT[c["dt"]]) for x in cache.load(0, c["ctx"])]
    if c["op"] == "store":
        q = []
        if c["rope"]:
            x = st["qkv"].float().unflatten(-1, (-1, hd))
            at = st["pos"][:, None] + torch.arange(s, device="cuda")
            cos, sin = st["cos"][at][:, :, None], st["sin"][at][:, :, None]
            q = [_rotate(x[:, :, :h], cos, sin).to(DT[c["dt"]])]
            cache.store(_rotate(x[:, :, h:h + kv], cos, sin), x[:, :, h + kv:], st["pos"])
        else:
            cache.store(st["k"], st["v"], st["pos"])
        return q + cache.load(st["pos"], s)
    k, v = cache.load(0, c["ctx"])
    q = st["q"].float().view(b, s, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, hd)
    score = (q @ k.transpose(-1, -2) * (1 / math.sqrt(hd))).view(b, kv, h // kv, s, -1)
    at, last = torch.arange(c["ctx"], device="cuda"), st["pos"][:, None] + torch.arange(s, device="cuda")
    seen = at <= last[..., None]
    if c["window"]:
        seen &= at > last[..., None] - c["window"]
    seen = seen[:, None, None]
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(b, kv, -1, c["ctx"]) @ v).view(b, kv, h // kv, s, hd) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 3, 1, 2, 4).reshape(b, s, h, hd).to(DT[c["dt"]])


def run(st):
    if not own:
        return _plain(st)
    c, cache = st["case"], st["cache"]
    if c["op"] == "load":
        return list(cache.load(0, c["ctx"], dtype=DT[c["dt"]]))
    if c["op"] == "attend":
        return cache.attend(st["q"], st["pos"], window=c["window"])
    q = []
    if c["rope"]:
        q = [cache.rope_store(st["qkv"], st["cos"], st["sin"], st["pos"], c["h"])]
    else:
        cache.store(st["k"], st["v"], st["pos"])
    return q + list(cache.load(st["pos"], c["s"], dtype=torch.float32))


def work(case):
    c = case
    e = {"f32": 4, "f16": 2, "bf16": 2}[c["dt"]]
    row = (c["hd"] // 2 if c["fmt"] == "q4_0" else c["hd"]) + c["hd"] // 16  # codes and scales of one head's position
    rows = 2 * c["b"] * c["kv"]
    if c["op"] == "load":
        return {"bytes": rows * c["ctx"] * (row + c["hd"] * e), "flops": rows * c["ctx"] * c["hd"]}
    if c["op"] == "store":
        new = rows * c["s"]
        rotated = 2 * c["b"] * c["s"] * c["h"] * c["hd"] * e if c["rope"] else 0
        return {"bytes": new * (c["hd"] * e + row + c["hd"] * 4) + rotated, "flops": 6 * new * c["hd"]}
    read, pairs = 0, 0
    for n in _lengths(c):
        if not n:
            continue
        w = c["window"] or n
        read += min(n, w + c["s"] - 1)
        pairs += sum(min(n - i, w) for i in range(c["s"]))
    return {"bytes": 2 * c["kv"] * read * row + 2 * c["b"] * c["s"] * c["h"] * c["hd"] * e, "flops": 4 * c["h"] * c["hd"] * pairs}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------------------------

def _stands_for(x, fmt):
    """The values, in 64 bits, that the block format holds for x [n, hd]. The format is defined by f32 arithmetic up to its codes."""
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


def exact(case, seed):
    c = {"name": "", **case}
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    b, h, kv, hd, s, dt = c["b"], c["h"], c["kv"], c["hd"], c["s"], DT[c["dt"]]
    if c["page"]:
        torch.randperm(b * -(-c["ctx"] // c["page"]), generator=g, device="cuda")
    ks, vs = [], []
    for at in range(0, c["ctx"], CHUNK):
        k, v = _kv_rows(g, c, min(CHUNK, c["ctx"] - at))
        if c["op"] != "store":
            ks.append(k), vs.append(v)
    if c["op"] == "store":
        k, v = (x.transpose(1, 2) for x in _kv_rows(g, c, s))
        out = []
        if c["rope"]:
            q = _rand(g, b, s, h, hd).to(dt).transpose(1, 2)
            ang = torch.arange(c["ctx"], device="cuda")[:, None] / 10000.0 ** (torch.arange(0, hd, 2, device="cuda") / hd)[None]
            at = torch.tensor([list(range(n - s, n)) for n in _lengths(c)], device="cuda")
            cos, sin = (t[at][:, None].double() for t in (ang.cos(), ang.sin()))

            def turned(x):
                a, z = x[..., :hd // 2].double(), x[..., hd // 2:].double()
                return torch.cat((a * cos - z * sin, z * cos + a * sin), -1)
            out.append(turned(q).transpose(1, 2))
            k = turned(k)
        for x in (k, v):
            out.append(torch.stack([_stands_for(x[i], c["fmt"]) for i in range(b)]))
        return out
    if c["op"] == "load":
        return [torch.cat([torch.stack([_stands_for(x[i].transpose(0, 1), c["fmt"]) for i in range(b)]) for x in xs], 2) for xs in (ks, vs)] \
            if b * kv * c["ctx"] * hd <= 16 * 8 * 8192 * 128 else None
    q = (_rand(g, b, s, h, hd) * 1.5).to(dt)
    out = torch.zeros((b, s, h, hd), dtype=torch.float64, device="cuda")
    where = torch.arange(c["ctx"], device="cuda")
    for i, n in enumerate(_lengths(c)):
        if not n:
            continue
        for j in range(kv):
            key, value = (torch.cat([_stands_for(x[i, :, j], c["fmt"]) for x in xs])[:n] for xs in (ks, vs))
            for head in range(j * (h // kv), (j + 1) * (h // kv)):
                logit = q[i, :, head].double() @ key.T / math.sqrt(hd)
                last = (n - s + torch.arange(s, device="cuda"))[:, None]
                hidden = where[:n] > last
                if c["window"]:
                    hidden |= where[:n] <= last - c["window"]
                out[i, :, head] = torch.softmax(logit.masked_fill(hidden, -torch.inf), 1) @ value
    return out
