"""Page tables from lengths, packed tokens, sinks beside a window, trees of drafted tokens and the accepted path kept: whole numbers against plain Python, stored
blocks against the calls for rectangles, attention against plain 64-bit arithmetic on what the blocks stand for (tolerances: test_gpu_kv_cache.py)."""
import math
import random

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import DEV, TYPES, _cache, _check, _filled, _init, _pos, _rand, _status  # noqa: F401 (_init: the module's fixture)

pytestmark = pytest.mark.gpu
PAST_STORE, PAST_ATTEND, NO_PAGE, CUT = 1 << 27, 1 << 28, 1 << 29, 1 << 31


@pytest.fixture(autouse=True)
def _clean():
    from xn_b200 import _lib
    _lib.check(_lib.lib().xnq_init(0))


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- page tables ----

def _reserved(table, length, first, sinks, page, pages, max_seq):
    out, wanted, room = np.full_like(table, -1), [], []
    for b in range(table.shape[0]):
        n = min(max(int(length[b]), 0), max_seq)
        f = 0 if first is None else min(max(int(first[b]), 0), max_seq)
        need = [i for i in range(table.shape[1]) if i * page < n and ((i + 1) * page > f or i * page < sinks)]
        wanted.append((n, need))
        for i in need:
            if 0 <= table[b, i] < pages:
                out[b, i] = table[b, i]
    left = sorted(set(range(pages)) - set(out[out >= 0].tolist()))
    left.reverse()
    for b, (n, need) in enumerate(wanted):
        end = n
        for i in need:
            if out[b, i] < 0:
                if left:
                    out[b, i] = left.pop()
                else:
                    end = min(end, i * page)
        room.append(end)
    return out, room, len(left)


def _paged(batch, max_seq, page, pages):
    from xn_b200.dtypes import GgmlDType
    from xn_b200.kv_cache import QuantizedKVCache
    return QuantizedKVCache(GgmlDType.Q4_0, batch, 1, max_seq, 64, DEV, page_size=page, num_pages=pages)


RESERVE = [  # batch, max_seq, page, pages
    (1, 1, 32, 1), (1, 33, 32, 3), (3, 1000, 32, 40), (7, 4097, 64, 500), (1, 200000, 32, 6251), (33, 31, 32, 20), (300, 100, 64, 1000), (64, 8192, 64, 8192),
    (64, 8193, 64, 9001), (100, 20000, 64, 31248), (257, 2047, 32, 16385), (40, 65536, 64, 70000)]


@pytest.mark.parametrize("batch,max_seq,page,pages", RESERVE)
@pytest.mark.parametrize("kind", ["plain", "window", "sinks", "scarce"])
def test_page_tables(batch, max_seq, page, pages, kind):
    rng = np.random.default_rng(batch * 7 + max_seq)
    c = _paged(batch, max_seq, page, pages)
    per = c.page_table.shape[1]
    for step in range(4):
        table = c.page_table.cpu().numpy().copy()
        if step == 1 and pages > 4:   # entries that are no page, pages that two rows name
            table[rng.integers(0, batch), rng.integers(0, per)] = pages
            table[rng.integers(0, batch), rng.integers(0, per)] = -7
            table[0] = table[-1]
            c.page_table.copy_(torch.from_numpy(table))
        most = max_seq if kind == "scarce" else max(1, min(max_seq, pages * page // batch))
        length = rng.integers(-3, most + 5, batch)
        length[rng.integers(0, batch)] = 0
        first = None if kind == "plain" else np.maximum(length - rng.integers(0, 300, batch), -5)
        sinks = int(rng.integers(0, 100)) if kind == "sinks" else 0
        room, free = c.reserve(torch.from_numpy(length).to(DEV), first=None if first is None else torch.from_numpy(first).to(DEV), sinks=sinks)
        want, want_room, want_free = _reserved(table, length, first, sinks, page, pages, max_seq)
        assert np.array_equal(c.page_table.cpu().numpy(), want)
        assert room.tolist() == want_room and int(free) == want_free and free.shape == () and room.dtype is torch.int64
    before = c.page_table.clone()
    again = c.reserve(torch.from_numpy(length).to(DEV), first=None if first is None else torch.from_numpy(first).to(DEV), sinks=sinks)   # nothing left to do
    if kind != "scarce":
        assert torch.equal(c.page_table, before)
    assert int(again[1]) == want_free and again[0].tolist() == want_room
    assert _status() == 0


def test_a_page_table_from_another_and_in_a_graph():
    c = _paged(5, 700, 32, 60)
    length, source = _pos(700, 0, 33, 64, 65), _i32([[(7 * b + i) % 60 if i < 3 else -1 for i in range(22)] for b in range(5)])
    kept = source.clone()
    room, free = c.reserve(length, table=source)
    want, want_room, want_free = _reserved(source.cpu().numpy(), length.tolist(), None, 0, 32, 60, 700)
    assert np.array_equal(c.page_table.cpu().numpy(), want) and room.tolist() == want_room and int(free) == want_free and torch.equal(source, kept)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        c.reserve(length)
        with torch.cuda.graph(g, stream=s):
            room, free = c.reserve(length)
    for step in range(3):
        length.copy_(_pos(*(100 * step + 31 * b for b in range(5))))
        table = c.page_table.cpu().numpy()
        g.replay()
        want, want_room, want_free = _reserved(table, length.tolist(), None, 0, 32, 60, 700)
        assert np.array_equal(c.page_table.cpu().numpy(), want) and room.tolist() == want_room and int(free) == want_free


# ---- plans ----

def _planned(cache, pos, count, tokens, longest, parents):
    table = None if cache.page_table is None else cache.page_table.tolist()
    words = -(-longest // 32)
    out = dict(offsets=[], sequence=[-1] * tokens, position=[-1] * tokens, slot=[-1] * tokens, sees=[[0] * words for _ in range(tokens)])
    at = 0
    for b, n in enumerate(count):
        n = min(max(n, 0), longest, tokens - at)
        out["offsets"].append(at)
        paths = []
        for i in range(n):
            place, t = pos[b] + i, at + i
            out["sequence"][t] = b
            if parents is None:
                path = [i] if 0 <= place < cache.max_seq else None
                position = place
            else:
                up = parents[t]
                path = None if up < -1 or up >= i or pos[b] < 0 or place >= cache.max_seq or (up >= 0 and paths[up] is None) else ([] if up < 0 else paths[up]) + [i]
                position = pos[b] + len(path or []) - 1
            paths.append(path)
            if path is None:
                continue
            out["position"][t] = position
            page = b if table is None else table[b][place // cache.page_size]
            if 0 <= page < cache.num_pages:
                out["slot"][t] = page * cache.page_size + (place if table is None else place % cache.page_size)
            for j in path:
                out["sees"][t][j // 32] |= 1 << (j % 32)
        at += n
    out["offsets"].append(at)
    return out


def _tree(rng, n, shape, blank=0.0):
    if shape == "chain":
        up = [i - 1 for i in range(n)]
    elif shape == "star":
        up = [-1] + [0] * (n - 1)
    elif shape == "roots":
        up = [-1] * n
    else:
        up = [-1 if i == 0 else rng.randint(max(-1, i - 9), i - 1) for i in range(n)]
    return [-2 if rng.random() < blank else x for x in up]


def _same_plan(plan, want, tree):
    for name in ("offsets", "sequence", "position", "slot"):
        assert getattr(plan, name).tolist() == want[name], name
    if tree:
        assert [[x % 2 ** 32 for x in row] for row in plan.sees.tolist()] == want["sees"]


@pytest.mark.parametrize("page", [None, 32, 96])
@pytest.mark.parametrize("pos,count,tokens,longest", [
    ([5], [1], 1, None), ([0], [0], 3, None), ([7], [3], 0, None), ([0, 60, 3], [70, 2, 0], 72, 70), ([1, 2, 3, 90], [-4, 0, 5, 9], 20, 9), ([-3, 95, 50], [6, 9, 1], 17, None),
    ([0] * 40, [i % 3 for i in range(40)], 50, 2), (list(range(90)) * 4, [(i * 7) % 5 for i in range(360)], 800, 3)])
def test_slot_maps(page, pos, count, tokens, longest):
    c = _cache("q4_0", len(pos), 1, 100, 64, page)
    if page and len(pos) > 2:
        c.page_table[1, 0], c.page_table[2, 0] = -1, 100000   # no page
    plan = c.plan(_pos(*pos), _pos(*count), tokens, longest)
    limit = max(1, min(tokens, longest or tokens))
    _same_plan(plan, _planned(c, pos, count, tokens, limit, None), False)
    assert plan.start.tolist() == pos and plan.sees is None and plan.nodes is None
    cut = any(n < 0 or n > limit for n in count) or sum(min(max(n, 0), limit) for n in count) > tokens
    assert bool(_status() & CUT) == cut


@pytest.mark.parametrize("page", [None, 32])
@pytest.mark.parametrize("shape", ["chain", "star", "roots", "random"])
@pytest.mark.parametrize("count,longest,pad,blank", [([1], 1, 0, 0.0), ([256], 256, 3, 0.0), ([33, 0, 64, 31, 32], 64, 5, 0.1), ([7, 255, 9, 200], 255, 0, 0.02), ([5, 4, 3] * 50, 5, 70, 0.2)])
def test_trees(page, shape, count, longest, pad, blank):
    rng = random.Random(len(count) + longest)
    c = _cache("q4_0", len(count), 1, 700, 64, page)
    pos = [rng.choice([0, 31, 400, 640, 699, -2]) if i else 3 for i in range(len(count))]
    parents = [x for n in count for x in _tree(rng, n, shape, blank)] + [-2] * pad
    plan = c.plan(_pos(*pos), _pos(*count), len(parents), longest, _i32(parents))
    want = _planned(c, pos, count, len(parents), longest, parents)
    _same_plan(plan, want, True)
    for b, n in enumerate(count):
        there = sum(1 << i for i in range(n) if want["position"][want["offsets"][b] + i] >= 0)
        assert [x % 2 ** 32 for x in plan.nodes[b].tolist()] == [there >> (32 * w) & 0xffffffff for w in range(-(-longest // 32))]
    past = any(p >= 0 and p + n > 700 for p, n in zip(pos, count) if n)
    off = want["offsets"]
    cut = any(up != -2 and not -1 <= up < i for b, n in enumerate(count) for i, up in enumerate(parents[off[b]:off[b + 1]]))   # (a star of no tokens has one parent too many: the others are shifted)
    assert _status() & ~PAST_STORE == (CUT if cut else 0) and (past or not _status() & PAST_STORE)


def test_parents_that_are_none():
    c = _cache("q4_0", 2, 1, 64, 64)
    parents = [-1, 0, 1, 3, -1, 4, 2, -3, -1, 99, 0]   # of the first tree 3 -> itself, 5 -> 4; of the second 0 -> out of range ..
    plan = c.plan(_pos(4, 9), _pos(7, 4), 11, 7, _i32(parents))
    _same_plan(plan, _planned(c, [4, 9], [7, 4], 11, 7, parents), True)
    assert _status() == CUT


def test_one_position_for_all_and_a_plan_keeps_it():
    c = _cache("q8_0", 3, 1, 64, 64)
    pos = _pos(9)
    plan = c.plan(pos, _pos(1, 2, 0), 3)
    pos.fill_(50)
    assert plan.start.tolist() == [9, 9, 9] and plan.position.tolist() == [9, 9, 10]


# ---- stored ----

@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,KV,H,page,S,starts", [(64, 1, 1, None, 1, [0]), (128, 3, 6, 32, 7, [1, 30, 64]), (64, 8, 8, 64, 40, [0, 31, 17, 59]), (128, 2, 8, None, 5, [3, 95, 2, -2, 70]),
                                                   (128, 1, 4, 32, 4000, [0, 1, 33])])
def test_packed_rows_are_stored_as_rectangles_are(fmt, dt, hd, KV, H, page, S, starts):
    B, L = len(starts), max(100, S + 40)
    one, other = (_cache(fmt, B, KV, L, hd, page, seed=2) for _ in range(2))
    qkv = _rand(3, B, S, (H + 2 * KV) * hd, gain=2.0).to(TYPES[dt]).to(DEV)
    cos, sin = _rand(4, L, hd // 2).to(DEV), _rand(5, L, hd // 2).to(DEV)
    count = [S - i % 2 if S > 1 else 1 for i in range(B)]   # odd and even lengths: rows of the next sequence begin at either parity
    rows = torch.cat([torch.arange(n) + b * S for b, n in enumerate(count)]).to(DEV)
    packed = qkv.flatten(0, 1)[rows]
    kv = qkv.unflatten(2, (-1, hd))
    for rope in (False, True):
        for c in (one, other):
            c.pages.zero_()
        plan = other.plan(_pos(*starts), _pos(*count), len(rows) + 3, S)
        tail = torch.cat([packed, packed[:1].expand(3, -1)])
        for b in range(B):   # sequence by sequence, as one of the batch
            n, pos = count[b], torch.full((B,), -10 ** 6, dtype=torch.int64, device=DEV)
            pos[b] = starts[b]
            if rope:
                q = one.rope_store(qkv[:, :n], cos, sin, pos, H)[b]
                got = other.rope_store(tail, cos, sin, plan, H) if b == 0 else got
                assert torch.equal(got[sum(count[:b]):sum(count[:b]) + n], q)
            else:
                one.store(kv[:, :n, H:H + KV], kv[:, :n, H + KV:], pos)
        if rope:
            assert got.shape == (len(rows) + 3, H, hd) and not got[-3:].any()
            f = other.rope_store(tail, cos, sin, plan, H, out_dtype=torch.float32)
            assert f.dtype is torch.float32 and torch.equal(f.to(TYPES[dt]), got)
        else:
            t = tail.unflatten(1, (-1, hd))
            other.store(t[:, H:H + KV], t[:, H + KV:], plan)
        assert torch.equal(one.pages, other.pages)
    past = any(s + n > L for s, n in zip(starts, count))
    assert bool(_status() & PAST_STORE) == past


def test_strides_and_tables_that_are_short():
    c, d = _cache("q4_0", 2, 2, 64, 64, 32), _cache("q4_0", 2, 2, 64, 64, 32)
    plan = c.plan(_pos(5, 20), _pos(9, 4), 13)
    k, v = (_rand(i, 13, 3, 80).to(torch.bfloat16).to(DEV) for i in (0, 1))
    c.store(k[:, :2, :64], v[:, 1:, 3:67], plan)   # rows apart, and rows that are not 16-byte aligned
    d.store(k[:, :2, :64].contiguous(), v[:, 1:, 3:67].contiguous(), d.plan(_pos(5, 20), _pos(9, 4), 13))
    assert torch.equal(c.pages, d.pages) and _status() == 0
    qkv = _rand(7, 13, 6 * 64).to(DEV)
    cos = _rand(8, 22, 32).to(DEV)
    before = c.pages.clone()
    q = c.rope_store(qkv, cos, cos, plan, 2)   # positions 22 and 23 are not in the tables
    assert _status() == PAST_STORE and not q[11:].any() and q[:11].any(-1).all()
    k2, v2 = c.load(22, 2)
    c.pages.copy_(before)
    assert torch.equal(k2[1], c.load(22, 2)[0][1]) and torch.equal(v2[1], c.load(22, 2)[1][1])


# ---- attended to ----

def _packed_reference(c, q, plan, causal=True, window=0, sinks=0, scale=None):
    """f64: (out, lse, the f32 tolerance, the largest sum of |scale q_i k_i| of a visible pair), from the plan's own offsets and positions (which other tests hold)."""
    L, hd = c.max_seq, c.head_dim
    k, v = (x.double() for x in c.load(0, L, dtype=torch.float32))
    n, H = q.shape[:2]
    g, scale = H // c.kv_heads, hd ** -0.5 if scale is None else scale
    out, lse = torch.zeros(n, H, hd, dtype=torch.float64, device=DEV), torch.full((n, H), -math.inf, dtype=torch.float64, device=DEV)
    off, start, position = plan.offsets.tolist(), plan.start.tolist(), plan.position
    j, size = torch.arange(L, device=DEV), 0.0
    here = None
    if c.page_table is not None:
        per = c.page_table.shape[1]
        here = ((c.page_table >= 0) & (c.page_table < c.num_pages))[:, :, None].expand(-1, -1, c.page_size).reshape(c.batch, per * c.page_size)[:, :L]
    for b in range(c.batch):
        r = slice(off[b], off[b + 1])
        m = off[b + 1] - off[b]
        if m == 0:
            continue
        p = position[r][:, None]
        hi = p if causal else torch.full_like(p, start[b] + m - 1)
        if plan.sees is not None:
            hi = torch.full_like(p, start[b] - 1)
        seen = j <= hi
        if window:
            seen = seen & ((j > p - window) | (j < sinks))
        if plan.sees is not None:
            bits = (plan.sees[r].long()[:, :, None] >> torch.arange(32, device=DEV) & 1).bool().flatten(1)[:, :m]
            end = min(m, L - start[b])
            if start[b] >= 0 and end > 0:
                seen[:, start[b]:start[b] + end] |= bits[:, :end]
        seen = seen & (p >= 0)
        if here is not None:
            seen = seen & here[b]
        qq = q[r].double().transpose(0, 1)
        kk, vv = (x[b].repeat_interleave(g, 0) for x in (k, v))
        score = (qq @ kk.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
        sums = torch.logsumexp(score, -1)
        w = torch.where(seen, torch.exp(score - sums.masked_fill(sums == -math.inf, 0.0)[..., None]), 0.0)
        size = max(size, float(((qq.abs() @ kk.abs().transpose(-1, -2)) * abs(scale)).masked_fill(~seen, 0.0).max()))
        out[r], lse[r] = (w @ vv).transpose(0, 1), sums.transpose(0, 1)
    u = 2.0 ** -24
    return out, lse, float(v.abs().max()) * (4 * u * (hd / 16 + 16) * size + 64 * u), size


def _attends(c, q, plan, what, **kw):
    """Attention into a given result and into one of its own, with logarithms; returns the result."""
    lse, out = torch.full(q.shape[:2], 7.0, device=DEV), torch.full_like(q, math.nan)
    c.attend(q, plan, out=out, lse=lse, **kw)
    want, want_lse, tol, size = _packed_reference(c, q, plan, **kw)
    total = int(plan.offsets[-1])
    assert torch.isnan(out[total:]).all() and (lse[total:] == 7.0).all()   # rows behind the last sequence are left as they were
    _check(out[:total], want[:total], tol, what)
    seen = torch.isfinite(want_lse[:total])
    assert torch.equal(torch.isfinite(lse[:total]), seen) and bool((lse[:total][~seen] == -math.inf).all()) and not out[:total][~seen].any()
    if seen.any():
        # f32: the sums' own rounding. 16-bit rows: a key's value is rounded to f16, by at most 2^-11 of it (half a step), so that a score is off by no more than
        # 2^-11 of the sum of |scale q_i k_i|, and so is the logarithm of a sum of exponentials, whose derivative by its scores is a mean's.
        near = 2e-5 * max(1.0, float(want_lse[:total][seen].abs().max())) + (0.0 if q.dtype is torch.float32 else 2.0 ** -11 * size)
        assert float((lse[:total] - want_lse[:total])[seen].abs().max()) <= near, what
    own = c.attend(q, plan, **kw)
    assert torch.equal(own[:total], out[:total]) and not own[total:].any()
    return out


MIX = [  # heads, KV, hd, L, page, starts, counts, pad
    (1, 1, 128, 1, None, [0], [1], 0), (8, 2, 64, 100, 32, [99, 0, 40, 7], [1, 1, 0, 1], 2), (32, 8, 128, 600, 64, [500, 31, 0, 599], [9, 1, 33, 1], 0),
    (4, 4, 128, 300, None, [0, 100, 299], [150, 70, 1], 5), (28, 4, 64, 1500, 32, [1000, 3, 700], [257, 5, 2], 0), (6, 1, 64, 900, 64, [0, 500, 13, 890], [300, 12, 40, 10], 9),
    (16, 2, 128, 5000, None, [4000], [300], 0), (7, 7, 64, 77, 32, [-3, 10], [20, 67], 1)]


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd,L,page,starts,counts,pad", MIX)
def test_packed_attention(fmt, dt, H, KV, hd, L, page, starts, counts, pad):
    c = _filled(fmt, len(starts), KV, L, hd, page, seed=H + L)
    n = sum(counts) + pad
    plan = c.plan(_pos(*starts), _pos(*counts), n, max(counts))
    q = _rand(5, n, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    for kw in ({}, dict(window=1, sinks=1), dict(window=50, sinks=4), dict(window=L // 3 + 1, sinks=40), dict(window=300), dict(window=20, sinks=10 ** 6), dict(causal=False, window=64, sinks=33),
               dict(scale=-0.07, window=200, sinks=64)):
        _attends(c, q, plan, (fmt, dt, H, L, kw), **kw)
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd,L,page,starts,counts,pad,shape", [
    (8, 2, 128, 64, None, [10], [1], 0, "chain"), (8, 8, 64, 500, 32, [400, 0, 31, 77], [7, 33, 20, 0], 3, "random"), (32, 8, 128, 2000, 64, [1900, 700, 32], [60, 17, 33], 0, "random"),
    (4, 1, 64, 900, None, [600, 1], [256, 250], 6, "random"), (16, 4, 128, 3000, 64, [2900, 100, 1500, 60, 2000], [64, 4, 40, 30, 8], 0, "star"), (6, 2, 64, 300, 32, [50, 200], [90, 100], 2, "chain"),
    (12, 3, 128, 400, 32, [13, 399], [40, 1], 0, "roots")])
def test_trees_of_drafts(fmt, dt, H, KV, hd, L, page, starts, counts, pad, shape):
    rng = random.Random(L)
    c = _filled(fmt, len(starts), KV, L, hd, page, seed=H + L)
    parents = [x for n in counts for x in _tree(rng, n, shape, 0.1 if shape == "random" else 0.0)] + [-2] * pad
    longest = max(counts)
    plan = c.plan(_pos(*starts), _pos(*counts), len(parents), longest, _i32(parents))
    q = _rand(6, len(parents), H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    for kw in ({}, dict(window=longest, sinks=3), dict(window=longest + 100, sinks=64), dict(window=L), dict(scale=0.3)):
        out = _attends(c, q, plan, (fmt, dt, H, L, shape, kw), **kw)
        none = plan.position[:int(plan.offsets[-1])] < 0
        assert not out[:len(none)][none].any()
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt,S", [("f32", 1), ("bf16", 1), ("f16", 6), ("bf16", 40), ("f16", 200), ("f32", 90)])
def test_sinks_without_a_plan(fmt, dt, S):
    B, H, KV, hd, L = 3, 8, 2, 128, 1000
    c = _filled(fmt, B, KV, L, hd, 64)
    q = _rand(5, B, S, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    starts = [L - S, 300, -S]
    plan = c.plan(_pos(*starts), _pos(S, S, S), B * S, S)
    for window, sinks in ((1, 1), (33, 4), (70, 100), (500, 64), (50, 0), (0, 9)):
        lse, out = torch.full((B, S, H), 7.0, device=DEV), torch.full_like(q, math.nan)
        c.attend(q, _pos(*starts), window=window, sinks=sinks, out=out, lse=lse)
        want, want_lse, tol, _ = _packed_reference(c, q.flatten(0, 1), plan, window=window, sinks=sinks)
        _check(out.flatten(0, 1), want, tol, (fmt, dt, S, window, sinks))
        assert not out[2].any() and bool((lse[2] == -math.inf).all())
        assert torch.equal(c.attend(q, _pos(*starts), window=window, sinks=sinks), out)
    assert torch.equal(c.attend(q, _pos(*starts), sinks=9), c.attend(q, _pos(*starts)))   # all of it is seen anyway
    assert _status() == 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B,most,KV", [(65, 40, 1), (300, 3, 2), (300, 70, 1), (700, 9, 1)])
def test_many_sequences(dt, B, most, KV):
    rng = random.Random(B)
    L, hd, H = 700, 64, 4 * KV
    c = _filled("q4_0", B, KV, L, hd, 32)
    counts = [rng.choice([0, 1, 1, rng.randint(1, most)]) for _ in range(B)]
    starts = [rng.randint(0, L - most) for _ in range(B)]
    n = sum(counts) + 4
    q = _rand(9, n, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    plan = c.plan(_pos(*starts), _pos(*counts), n, most)
    _attends(c, q, plan, (dt, B, most), window=100, sinks=5)
    parents = [x for m in counts for x in _tree(rng, m, "random", 0.05)] + [-2] * 4
    _attends(c, q, c.plan(_pos(*starts), _pos(*counts), n, most, _i32(parents)), (dt, B, most, "tree"))
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
def test_one_long_sequence_among_short_ones(fmt):
    """Parts: of the long one many, of the others none; and of one that has fewer rows than the grid."""
    L, H, KV, hd = 20000, 4, 1, 64
    c = _filled(fmt, 4, KV, L, hd, 128)
    for counts, starts in (([64, 70, 1, 64], [19900, 300, 5000, 0]), ([20, 100, 3, 0], [19980, 100, 9000, 4]), ([130, 0, 0, 0], [19870, 0, 0, 0])):
        n = sum(counts)
        q = _rand(9, n, H, hd, gain=1.5).to(torch.bfloat16).to(DEV)
        plan = c.plan(_pos(*starts), _pos(*counts), n, 130)
        for kw in ({}, dict(window=7000, sinks=50)):
            out = _attends(c, q, plan, (fmt, counts, kw), **kw)
            for _ in range(10):
                assert torch.equal(c.attend(q, plan, **kw), out)   # whoever came first
    one = _filled(fmt, 1, KV, 3000, hd)
    plan = one.plan(_pos(2900), _pos(33), 200, 200)   # room for 200 tokens, 33 came
    _attends(one, _rand(3, 200, 8, hd).to(torch.float16).to(DEV), plan, "fewer than there is room for")
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt,n", [("f32", 5), ("bf16", 5), ("f16", 9), ("bf16", 40), ("f16", 90), ("f32", 40)])
def test_what_is_not_seen_changes_no_bit(fmt, dt, n):
    """Between the first positions and the window, behind the tokens, drafts that are not ancestors, places that are not used: infinite and NaN scales."""
    L, H, KV, hd, start, window, sinks = 700, 8, 2, 128, 500, 100, 40
    c = _filled(fmt, 2, KV, L, hd, 32)
    q = _rand(5, 2 * n, H, hd).to(TYPES[dt]).to(DEV)
    parents = [-1 if i == 0 else -2 if i % 5 == 4 else (i - 1) // 2 if (i - 1) // 2 % 5 != 4 else 0 for i in range(n)] * 2
    plans = [(c.plan(_pos(start, 90), _pos(n, n), 2 * n, n), window), (c.plan(_pos(start, 90), _pos(n, n), 2 * n, n, _i32(parents)), max(window, n))]
    for plan, w in plans:
        want = c.attend(q, plan, window=w, sinks=sinks)
        k, v = c.load(0, L, dtype=torch.float32)
        d = _cache(fmt, 2, KV, L, hd, 32, seed=11)
        d.pages.fill_(0xff)   # every scale a NaN
        mine = d.plan(_pos(start, 90), _pos(n, n), 2 * n, n, _i32(parents) if plan.sees is not None else None)
        for b, s in ((0, start), (1, 90)):
            live = [i for i in range(n) if int(plan.position[b * n + i]) >= 0]
            at = sorted(set(range(min(sinks, s))) | set(range(max(0, s - w + 1), s)) | {s + i for i in live})
            for lo in range(0, len(at)):
                one = torch.full((2,), -10, dtype=torch.int64, device=DEV)
                one[b] = at[lo]
                d.store(k[:, :, at[lo]:at[lo] + 1].transpose(1, 2), v[:, :, at[lo]:at[lo] + 1].transpose(1, 2), one)
        if plan.sees is not None:
            q[plan.position < 0] = math.nan   # nor is the query of a place that is not used
        assert torch.equal(d.attend(q, mine, window=w, sinks=sinks), want)   # (blocks of what blocks stand for are the same blocks)
    assert _status() == 0


def test_a_row_that_sees_a_scale_that_is_not_finite():
    L, H, KV, hd = 300, 4, 1, 64
    for dt, n in (("f32", 6), ("bf16", 6), ("bf16", 40)):
        c = _filled("q4_0", 1, KV, L, hd)
        parents = [-1] + [0] * (n - 1)
        plan = c.plan(_pos(200), _pos(n), n, n, _i32(parents))
        bad = torch.full((1, 1, KV, hd), math.inf, device=DEV)
        c.store(bad, bad, _pos(203))   # the fourth draft: seen by itself alone
        out = c.attend(_rand(1, n, H, hd).to(TYPES[dt]).to(DEV), plan)
        assert torch.isnan(out[3]).all() and torch.isfinite(torch.cat([out[:3], out[4:]])).all()


def test_pages_that_are_gone():
    """A window's pages given back: nothing is missed, and what lies there now is another sequence's."""
    L, H, KV, hd, page = 2000, 8, 2, 64, 64
    for dt in ("f32", "bf16"):
        c = _filled("q4_0", 2, KV, L, hd, page)
        q = _rand(3, 2, 8, hd).to(TYPES[dt]).to(DEV)[:, :H]
        plan = c.plan(_pos(1500, 900), _pos(1, 1), 2, 1)
        want = c.attend(q, plan, window=300, sinks=70)
        length, first = _pos(1501, 901), _pos(1501 - 300, 901 - 300)
        room, free = c.reserve(length, first=first, sinks=70)
        assert room.tolist() == [1501, 901] and int((c.page_table[0] >= 0).sum()) == 2 + (1500 // 64 - 1201 // 64 + 1) and int((c.page_table[0, 2:18] >= 0).sum()) == 0
        assert torch.equal(c.attend(q, c.plan(_pos(1500, 900), _pos(1, 1), 2, 1), window=300, sinks=70), want)
        assert _status() == 0


# ---- kept ----

@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [None, 32])
@pytest.mark.parametrize("shape,counts", [("chain", [1, 5, 70]), ("random", [40, 9, 0, 64]), ("star", [256, 3]), ("random", [200, 255, 256])])
def test_the_accepted_path_stays(fmt, hd, page, shape, counts):
    rng = random.Random(hd + len(counts))
    B, KV, L = len(counts), 3, 700
    c = _filled(fmt, B, KV, L, hd, page)
    starts = [rng.choice([0, 31, 33, 100, L - n]) for n in counts]
    trees = [_tree(rng, n, shape, 0.05) for n in counts]
    plan = c.plan(_pos(*starts), _pos(*counts), sum(counts) + 1, max(counts), _i32([x for t in trees for x in t] + [-2]))
    node = [rng.randint(-1, n - 1) if n else rng.randint(-1, 3) for n in counts]
    node[0] = counts[0] - 1
    k, v = c.load(0, L, dtype=torch.float32)
    pos = c.keep(plan, _pos(*node))
    want = []
    for b, n in enumerate(counts):
        path, at = [], node[b] if 0 <= node[b] < n else -1
        while at >= 0:
            path.append(at)
            at = trees[b][at]
        if at == -2:
            path = []   # the token, or one that it follows, is none
        path.reverse()
        want.append(starts[b] + len(path))
        for x in (k, v):
            x[b, :, starts[b]:starts[b] + len(path)] = x[b, :, [starts[b] + i for i in path]].clone()
    assert pos.tolist() == want
    got = c.load(0, L, dtype=torch.float32)
    assert torch.equal(got[0], k) and torch.equal(got[1], v) and _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_a_server_between_its_steps(fmt, dt):
    """Prompts packed into pages, drafted trees attended to and kept, sequences that end and begin: what each sequence has in the end, and what its tokens saw, is
    what it has when its tokens come one after the other."""
    rng = random.Random(4)
    B, KV, H, hd, L, page = 4, 2, 8, 64, 500, 32
    c, plain = _cache(fmt, B, KV, L, hd, page), _cache(fmt, B, KV, L, hd)
    c.page_table.fill_(-1)
    ang = torch.arange(L, device=DEV)[:, None] / 10000.0 ** (torch.arange(0, hd, 2, device=DEV) / hd)[None]
    cos, sin = ang.cos(), ang.sin()
    rows = lambda n: torch.randn(n, (H + 2 * KV) * hd, device=DEV).to(TYPES[dt])

    def alone(b, qkv, at):   # one sequence's tokens, one after the other
        out = []
        for i in range(qkv.shape[0]):
            pos = torch.full((B,), -1, dtype=torch.int64, device=DEV)
            pos[b] = at + i
            q = plain.rope_store(qkv[i:i + 1].expand(B, 1, -1), cos, sin, pos, H)
            out.append(plain.attend(q, pos)[b, 0])
        return torch.stack(out)

    def near(got, want):
        assert float((got.double() - want.double()).norm()) <= (2.0 ** -7 if dt == "bf16" else 2e-6) * float(want.double().norm())

    counts = [70, 1, 0, 130]
    pos = torch.zeros(B, dtype=torch.int64, device=DEV)
    room, free = c.reserve(_pos(*counts))
    assert room.tolist() == counts
    plan = c.plan(pos, _pos(*counts), sum(counts), max(counts))
    qkv = rows(sum(counts))
    out = c.attend(c.rope_store(qkv, cos, sin, plan, H), plan)
    off = 0
    for b, n in enumerate(counts):
        if n:
            near(out[off:off + n], alone(b, qkv[off:off + n], 0))
        off += n
    pos = _pos(*counts)
    for step in range(3):
        sizes = [rng.randint(1, 40) if b != 2 or step else 0 for b in range(B)]
        trees = [_tree(rng, n, "random") for n in sizes]
        n = sum(sizes)
        c.reserve(pos + _pos(*sizes))
        plan = c.plan(pos, _pos(*sizes), n, 40, _i32([x for t in trees for x in t]))
        qkv = rows(n)
        out = c.attend(c.rope_store(qkv, cos, sin, plan, H), plan)
        node = [rng.randint(0, m - 1) if m else -1 for m in sizes]
        after = c.keep(plan, _pos(*node))
        off = 0
        for b, m in enumerate(sizes):
            path, at = [], node[b]
            while at >= 0:
                path.append(off + at)
                at = trees[b][at]
            path.reverse()
            if path:
                near(out[path], alone(b, qkv[path], int(pos[b])))
            assert int(after[b]) == int(pos[b]) + len(path)
            off += m
        pos = after
        c.reserve(pos)   # what only drafts that were not taken needed goes back
        for b in range(B):
            n = int(pos[b])
            for x, y in zip(c.load(0, max(n, 1), dtype=torch.float32), plain.load(0, max(n, 1), dtype=torch.float32)):
                assert torch.equal(x[b, :, :n], y[b, :, :n])
        if step == 1:   # a request ends, another takes its place
            pos[3] = 0
            c.reserve(pos)
            assert not (c.page_table[3] >= 0).any()
    assert _status() & ~(PAST_STORE | NO_PAGE) == 0   # (the read-backs above ask for more than some sequences have)


# ---- streams, graphs, layers, refusals ----

def test_a_step_in_a_graph():
    """reserve, plan, rope_store, attend and keep captured once, replayed for other requests; two graphs and an eager call beside one another."""
    B, KV, H, hd, L, page, n = 5, 2, 16, 64, 600, 32, 90
    c = _cache("q4_0", B, KV, L, hd, page)
    state = dict(pos=_pos(0, 50, 33, 7, 400), count=_pos(20, 1, 40, 0, 3), node=_pos(4, 0, 39, -1, 2), parents=_i32([i - 1 if i else -1 for i in range(n)]), qkv=torch.randn(n, (H + 2 * KV) * hd, device=DEV).to(torch.bfloat16))
    cos, sin = _rand(4, L, hd // 2).to(DEV), _rand(5, L, hd // 2).to(DEV)

    def step():
        room, free = c.reserve(state["pos"] + state["count"])
        plan = c.plan(state["pos"], state["count"], n, 40, state["parents"])
        out = c.attend(c.rope_store(state["qkv"], cos, sin, plan, H), plan)
        return room, free, plan.offsets, out, c.keep(plan, state["node"])

    s = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(s):
        step()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                res = step()
            graphs.append((g, res))
    torch.cuda.synchronize()
    for turn in range(4):
        state["count"].copy_(_pos(*((7 * turn + 11 * b) % 19 for b in range(B))))
        state["pos"].copy_(_pos(*((31 * turn + 60 * b) % 500 for b in range(B))))
        state["node"].copy_(_pos(*((turn + b) % 9 - 1 for b in range(B))))
        # every sequence's tokens are a chain
        off = np.concatenate([[0], np.cumsum(state["count"].tolist())])
        up = np.full(n, -2)
        for b in range(B):
            up[off[b]:off[b + 1]] = np.arange(off[b + 1] - off[b]) - 1
        state["parents"].copy_(torch.from_numpy(up))
        state["qkv"].normal_()
        table, pages = c.page_table.clone(), c.pages.clone()
        want = [x.clone() for x in step()]
        after = c.pages.clone()
        for g, res in graphs:
            c.page_table.copy_(table)
            c.pages.copy_(pages)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(res, want):
                assert torch.equal(x, y)
            assert torch.equal(c.pages, after)


def test_on_another_stream_and_under_a_mode():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    c = _filled("q4_0", 2, 2, 300, 64, 32)
    parents = _i32([-1, 0, 0, 1, -1, 0, -2])
    q, qkv = _rand(1, 7, 4, 64).to(DEV), _rand(2, 7, 8 * 64).to(DEV)
    cos = _rand(4, 300, 32).to(DEV)

    def all_of_it():
        c.page_table.copy_(table)
        room, free = c.reserve(_pos(200, 150), first=_pos(100, 0), sinks=5)
        plan = c.plan(_pos(100, 60), _pos(4, 3), 7, 4, parents)
        lse = torch.empty(7, 4, device=DEV)
        a = c.rope_store(qkv, cos, cos, plan, 4)
        c.store(qkv.view(7, 8, 64)[:, :2], qkv.view(7, 8, 64)[:, 2:4], plan)
        b = c.attend(q, plan, window=50, sinks=3)
        d = c.attend(q, plan, window=50, sinks=3, lse=lse)
        return [x.clone() for x in (room, free, plan.start, plan.offsets, plan.sequence, plan.position, plan.slot, plan.sees, plan.nodes, a, b, d, lse, c.keep(plan, _pos(3, 1)), c.page_table)]
    table = c.page_table.clone()
    want = all_of_it()
    with Watch():
        for x, y in zip(all_of_it(), want):
            assert torch.equal(x, y)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = all_of_it()
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_layers_share_a_table_and_a_plan():
    from xn_b200.dtypes import GgmlDType
    from xn_b200.kv_cache import QuantizedKVCache
    first = QuantizedKVCache(GgmlDType.Q4_0, 2, 2, 200, 64, DEV, page_size=32, num_pages=20)
    second = QuantizedKVCache(GgmlDType.Q8_0, 2, 1, 200, 128, DEV, page_size=32, num_pages=20, page_table=first.page_table)
    first.reserve(_pos(100, 50))
    assert second.page_table.data_ptr() == first.page_table.data_ptr() and int((second.page_table >= 0).sum()) == 4 + 2
    plan = first.plan(_pos(90, 40), _pos(3, 2), 5)
    x = _rand(0, 5, 1, 128).to(DEV)
    second.store(x, x, plan)
    k, _ = second.load(90, 3, dtype=torch.float32)
    assert float((k[0, 0] - x[:3, 0]).abs().max()) < 0.05
    with pytest.raises(ValueError, match="page_table"):
        QuantizedKVCache(GgmlDType.Q4_0, 3, 2, 200, 64, DEV, page_size=32, num_pages=20, page_table=first.page_table)
    with pytest.raises(ValueError, match="page_table"):
        QuantizedKVCache(GgmlDType.Q4_0, 2, 2, 200, 64, DEV, page_table=first.page_table)


def test_refusals():
    c, other, flat = _cache("q4_0", 2, 2, 100, 64, 32), _cache("q4_0", 2, 2, 100, 64, 32), _cache("q4_0", 2, 2, 100, 64)
    pos, count = _pos(0, 5), _pos(3, 4)
    with pytest.raises(ValueError, match="no pages"):
        flat.reserve(pos)
    for kw in (dict(length=pos.int()), dict(length=_pos(1)), dict(length=pos.cpu()), dict(length=pos, first=_pos(1, 2, 3)), dict(length=pos, sinks=-1), dict(length=pos, table=c.page_table[:1]),
               dict(length=pos, table=c.page_table.long()), dict(length=_pos(1, 2, 3, 4)[::2])):
        with pytest.raises(ValueError, match="reserve"):
            c.reserve(**kw)
    for args in ((pos, count, -1), (pos, count, 7, 0), (pos, count.int(), 7), (pos, _pos(1), 7), (pos, count, 7, 4, _i32([0] * 6)), (pos, count, 7, 4, _pos(*[0] * 7)), (pos.int(), count, 7), (_pos(1, 2, 3), count, 7),
                 (pos, count, 700, 257, _i32([0] * 700)), (pos, count, 7, 4, _i32([0] * 14)[::2])):
        with pytest.raises(ValueError):
            c.plan(*args)
    plan, tree = c.plan(pos, count, 7), c.plan(pos, count, 7, 4, _i32([-1] * 7))
    x, q, qkv = torch.zeros(7, 2, 64, device=DEV), torch.zeros(7, 4, 64, device=DEV), torch.zeros(7, 8 * 64, device=DEV)
    cos = torch.zeros(100, 32, device=DEV)
    for call in (lambda: other.store(x, x, plan), lambda: flat.attend(q, plan), lambda: other.rope_store(qkv, cos, cos, plan, 4), lambda: other.keep(tree, pos)):
        with pytest.raises(ValueError, match="another cache"):
            call()
    for call in (lambda: c.store(x[:6], x[:6], plan), lambda: c.store(x, x.half(), plan), lambda: c.store(q, q, plan), lambda: c.store(x[None], x[None], plan), lambda: c.attend(q[:, :3], plan),
                 lambda: c.attend(q[None], plan), lambda: c.attend(q.double(), plan), lambda: c.attend(q.cpu(), plan), lambda: c.attend(q, plan, window=-1), lambda: c.attend(q, plan, window=5, sinks=-1),
                 lambda: c.attend(q, tree, window=3), lambda: c.attend(q, plan, out=q[:6]), lambda: c.attend(q, plan, lse=torch.empty(7, 3, device=DEV)), lambda: c.rope_store(qkv[None], cos, cos, plan, 4),
                 lambda: c.rope_store(qkv, cos, cos, plan, 3), lambda: c.rope_store(qkv, cos[:, :16], cos, plan, 4), lambda: c.keep(plan, pos), lambda: c.keep(tree, pos.int()), lambda: c.keep(tree, _pos(1))):
        with pytest.raises(ValueError):
            call()
    leaf = torch.zeros(7, 4, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no derivative"):
        c.attend(leaf, plan)
    with pytest.raises(RuntimeError, match="no derivative"):
        c.store(leaf[:, :2], x, plan)
    with pytest.raises(AttributeError, match="fixed"):
        c.page_table = other.page_table
    empty = c.plan(pos, _pos(0, 0), 0)
    assert c.attend(q[:0], empty).shape == (0, 4, 64) and c.store(x[:0], x[:0], empty) is None and c.rope_store(qkv[:0], cos, cos, empty, 4).shape == (0, 4, 64)
    assert c.keep(c.plan(pos, _pos(0, 0), 0, 1, _i32([])), _pos(-1, 0)).tolist() == [0, 5] and empty.offsets.tolist() == [0, 0, 0]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [3, 70])
def test_rows_that_lie_apart(dt, n):
    """Queries with heads and tokens apart, one query for all tokens, results between other values."""
    c = _filled("q4_0", 2, 2, 400, 64, 32)
    plan = c.plan(_pos(300, 9), _pos(n - 1, 1), n + 2, n)
    wide = _rand(3, 8, n + 2, 80).to(TYPES[dt]).to(DEV)
    q = wide[:, :, :64].transpose(0, 1)
    want = c.attend(q.contiguous(), plan, window=70, sinks=9)
    assert torch.equal(c.attend(q, plan, window=70, sinks=9), want)
    assert torch.equal(c.attend(wide[:, :, 3:67].transpose(0, 1), plan), c.attend(wide[:, :, 3:67].transpose(0, 1).contiguous(), plan))   # not 16-byte aligned
    one = q[:1].expand(n + 2, -1, -1)
    assert torch.equal(c.attend(one, plan), c.attend(one.contiguous(), plan))
    room = torch.full((n + 2, 8, 3, 64), 5.0, dtype=TYPES[dt], device=DEV)
    c.attend(q, plan, window=70, sinks=9, out=room[:, :, 1])
    assert torch.equal(room[:n, :, 1], want[:n]) and (room[:, :, ::2] == 5.0).all() and (room[n:] == 5.0).all()
    with pytest.raises(ValueError, match="apart"):
        c.attend(q, plan, out=room[:1, :, 1].expand(n + 2, -1, -1))


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("H,KV,counts", [(64, 1, [1, 1, 2]), (96, 2, [1, 0, 1]), (5, 5, [1, 2, 1])])
def test_wide_and_odd_groups(fmt, dt, H, KV, counts):
    c = _filled(fmt, 3, KV, 500, 128, 64)
    plan = c.plan(_pos(499 - counts[0], 7, 250), _pos(*counts), sum(counts), max(counts))
    q = _rand(4, sum(counts), H, 128, gain=1.5).to(TYPES[dt]).to(DEV)
    for kw in ({}, dict(window=90, sinks=33)):
        _attends(c, q, plan, (fmt, dt, H, KV, kw), **kw)


def test_more_requests_than_pages():
    batch, pages = 40000, 1000
    c = _paged(batch, 32, 32, pages)
    length = torch.arange(batch, device=DEV) % 33   # every 33rd has none
    room, free = c.reserve(length)
    need = (length > 0).cumsum(0)
    there = (length > 0) & (need <= pages)
    assert torch.equal(room, torch.where(there, length, 0)) and int(free) == 0
    assert torch.equal(c.page_table[:, 0][there].long(), torch.arange(pages, device=DEV)) and (c.page_table[:, 0][~there] == -1).all()


def test_sequences_that_share_their_beginning():
    """A shared page is read by both, and free when the second lets go."""
    c = _filled("q8_0", 2, 2, 300, 64, 32)
    c.page_table[1, :3] = c.page_table[0, :3]
    q = _rand(1, 2, 4, 64).to(DEV)
    plan = c.plan(_pos(95, 95), _pos(1, 1), 2, 1)
    out = c.attend(torch.cat([q[:1], q[:1]]), plan)
    assert torch.equal(out[0], out[1])
    free = [int(c.reserve(_pos(*n))[1]) for n in ((96, 96), (0, 96), (0, 0))]
    assert free == [c.num_pages - 3, c.num_pages - 3, c.num_pages]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("others,rows", [(99, 64), (60, 130), (147, 64), (299, 64)])
def test_parts_of_one_and_units_of_many(dt, others, rows):
    """One sequence is most of the work and is cut into many parts; the others are a step each: CTAs for all of them."""
    L, H, KV, hd = 20000, 4, 1, 64
    B = others + 1
    c = _cache("q4_0", B, KV, L, hd, 64)
    c.page_table.fill_(-1)
    n = rows // H
    c.reserve(_pos(*([L] + [n] * others)))
    for at in range(0, L, 2000):
        pos = torch.full((B,), -10 ** 6, dtype=torch.int64, device=DEV)
        pos[0] = at
        x = _rand(at, 1, 2000, KV, hd).to(DEV).expand(B, -1, -1, -1)
        c.store(x, x, pos)
    plan = c.plan(_pos(*([L - n] + [0] * others)), _pos(*([n] * B)), B * n, n)
    x = _rand(5, B * n, KV, hd).to(DEV)
    c.store(x, x, plan)
    q = _rand(6, B * n, H, hd).to(TYPES[dt]).to(DEV)
    out = torch.full_like(q, math.nan)
    c.attend(q, plan, out=out)
    one = c.plan(_pos(*([L - n] + [0] * others)), _pos(*([n] + [0] * others)), n, n)   # the long one by itself
    want, _, tol, _ = _packed_reference_of(c, q, plan, [0, 1, others // 2, others])
    for b, w in want.items():
        _check(out[b * n:(b + 1) * n], w, tol, (dt, others, rows, b))
    assert torch.isfinite(out.float()).all()
    _check(c.attend(q[:n], one), want[0], tol, (dt, others, rows))


def _packed_reference_of(c, q, plan, which):
    """f64 results of some sequences of a plan without trees (causal, everything seen)."""
    off, start, out = plan.offsets.tolist(), plan.start.tolist(), {}
    for b in which:
        m = off[b + 1] - off[b]
        k, v = (x[b].double().repeat_interleave(q.shape[1] // c.kv_heads, 0)[:, :start[b] + m] for x in c.load(0, start[b] + m, dtype=torch.float32))
        score = q[off[b]:off[b + 1]].double().transpose(0, 1) @ k.transpose(-1, -2) * c.head_dim ** -0.5
        j, p = torch.arange(start[b] + m, device=DEV), (start[b] + torch.arange(m, device=DEV))[:, None]
        out[b] = (torch.softmax(score.masked_fill(j > p, -math.inf), -1) @ v).transpose(0, 1)
    return out, None, 0.0, None


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_sinks_in_a_graph_at_other_positions(dt):
    c = _filled("q4_0", 3, 2, 900, 64, 32)
    for S in (1, 40):
        q, pos = _rand(1, 3, S, 8, 64).to(TYPES[dt]).to(DEV), _pos(800, 100, -S)
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            c.attend(q, pos, window=70, sinks=5)
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=s):
                out = c.attend(q, pos, window=70, sinks=5)
        for at in ([800, 100, -S], [3, 859, 500], [0, -1, 31]):
            pos.copy_(_pos(*at))
            q.normal_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, c.attend(q, pos, window=70, sinks=5))


def test_threads_with_streams_of_their_own():
    """Plans, packed attention of few and of many rows and page tables from four threads at once: as one after the other."""
    import threading
    c = _filled("q8_0", 6, 2, 1200, 64, 32)
    counts = [[1, 1, 150, 1, 0, 2], [40, 1, 1, 33, 20, 1], [1] * 6, [200, 100, 3, 1, 1, 60]]
    jobs = []
    for i, n in enumerate(counts):
        pos = _pos(*((100 * b + 37 * i) % 900 for b in range(6)))
        jobs.append((pos, _pos(*n), sum(n), max(n), _rand(i, sum(n), 8, 64).to(torch.bfloat16 if i % 2 else torch.float16).to(DEV)))

    def work(job):
        pos, n, tokens, longest, q = job
        plan = c.plan(pos, n, tokens, longest)
        return c.attend(q, plan, window=300, sinks=9), c.attend(q, plan)
    want = [[x.clone() for x in work(job)] for job in jobs]
    torch.cuda.synchronize()
    wrong, errors = [], []

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    got = work(jobs[i])
                    torch.cuda.current_stream().synchronize()
                    wrong.extend(i for x, y in zip(got, want[i]) if not torch.equal(x, y))
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=thread, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not errors and not wrong and _status() == 0
