"""The quantized KV cache between requests: calls that lie at the edge of what is served, and closer looks at results of which test_gpu_kv_packed.py takes one norm."""
import math
import random
import threading

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import DEV, TYPES, _cache, _check, _filled, _init, _pos, _rand, _status  # noqa: F401 (_init: the module's fixture)
from test_gpu_kv_packed import CUT, PAST_STORE, _attends, _clean, _i32, _packed_reference, _paged, _tree  # noqa: F401 (_clean: before each test)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,page", [(6, 500, 32), (40, 4000, 32)])
def test_steps_without_a_wait_in_between(dt, B, L, page):
    """A server's steps enqueued one after the other, the page table another one in each: as with a wait behind every call. (40 rows of 125 entries: the table by
    several kernels.)"""
    KV, H, hd, n, steps = 2, 8, 64, 200 if B == 6 else 400, 25
    rng = random.Random(B)
    c = _cache("q4_0", B, KV, L, hd, page)
    cos, sin = _rand(4, L, hd // 2).to(DEV), _rand(5, L, hd // 2).to(DEV)
    at, todo = [0] * B, []
    for step in range(steps):
        at = [0 if rng.random() < 0.3 else a for a in at]   # requests end, others begin in their places
        counts = [min(rng.choice([0, 1, 1, rng.randint(1, 60)]), L - a) for a in at]
        while sum(counts) > n:
            counts[counts.index(max(counts))] = 1
        todo.append((_pos(*at), _pos(*counts), _pos(*(a + m for a, m in zip(at, counts))), (torch.randn(n, (H + 2 * KV) * hd, device=DEV)).to(TYPES[dt])))
        at = [a + m for a, m in zip(at, counts)]
    start = torch.randperm(c.num_pages, generator=torch.Generator().manual_seed(1))[:c.page_table.numel()].view(c.page_table.shape).to(torch.int32).to(DEV)

    def run(wait):
        c.page_table.copy_(start)
        c.pages.zero_()
        out = []
        torch.cuda.synchronize()
        for pos, count, length, qkv in todo:
            room, free = c.reserve(length)
            wait()
            plan = c.plan(pos, count, n)
            wait()
            q = c.rope_store(qkv, cos, sin, plan, H)
            wait()
            out += [room, free, plan.slot, plan.position, q, c.attend(q, plan, window=300, sinks=5)]
            wait()
            out += [c.attend(q, plan), *c.load(0, 64, dtype=torch.float32), c.page_table.clone()]
            wait()
        torch.cuda.synchronize()
        return out
    want = run(torch.cuda.synchronize)
    for _ in range(3):
        for i, (x, y) in enumerate(zip(run(lambda: None), want)):
            assert torch.equal(x, y), i
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run(lambda: None)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("B,L,tokens", [(256, 200, 32768), (200, 600, 100000)])
def test_f32_tokens_of_many_sequences(B, L, tokens):
    """No more is said of the sequences' lengths than that they are as many tokens as there are: any of them could be as long as all."""
    KV, H, hd, n = 1, 8, 64, tokens // B
    c = _filled("q4_0", B, KV, L, hd, 32)
    counts = [n + (-1) ** b * (b % 37) for b in range(B)]
    counts[-1] += tokens - sum(counts)
    starts = [(b * 7) % (L - m) if m < L else 0 for b, m in enumerate(counts)]
    plan = c.plan(_pos(*starts), _pos(*counts), tokens)
    assert plan.longest == tokens
    _attends(c, _rand(2, tokens, H, hd, gain=1.5).to(DEV), plan, (B, tokens))
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt,counts", [("f16", [1, 5, 15, 16, 64]), ("bf16", [1, 7, 8, 40])])
def test_a_plan_of_one_sequence_with_room_for_more(fmt, dt, counts):
    """Which arithmetic a sequence gets goes by its own rows, not by the room: below 64 rows of a KV head (bf16: 32) keys and weights keep their bits."""
    L, H, KV, hd = 3000, 8, 2, 128
    c = _filled(fmt, 1, KV, L, hd, 64)
    q = _rand(5, 64, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    for n in counts:
        plan = c.plan(_pos(2900 - n), _pos(n), 64)
        for kw in ({}, dict(window=700, sinks=40)):
            lse, out = torch.full((64, H), 7.0, device=DEV), torch.full_like(q, math.nan)
            c.attend(q, plan, out=out, lse=lse, **kw)
            want, want_lse, tol, size = _packed_reference(c, q, plan, **kw)
            _check(out[:n], want[:n], tol, (fmt, dt, n, kw))
            assert torch.isnan(out[n:]).all() and (lse[n:] == 7.0).all()
            rows = n * H // KV
            # as test_gpu_kv_cache.py has it where the scores are products of the codes themselves; else a key's rounding to f16, half a step of 2^-10 at most
            near = 2e-5 * max(1.0, float(want_lse[:n].abs().max())) + (0.0 if rows < (64 if dt == "f16" else 32) else 2.0 ** -11 * size)
            assert float((lse[:n] - want_lse[:n]).abs().max()) <= near, (fmt, dt, n, kw)
            own = c.attend(q, plan, **kw)
            assert torch.equal(own[:n], out[:n]) and not own[n:].any()
    assert _status() == 0


def test_one_sequence_of_few_and_of_many_tokens_in_a_graph():
    """One captured step with room for 90 tokens, replayed for a single token, for none and for all of them."""
    L, H, KV, hd, n = 1200, 8, 1, 64, 90
    c = _filled("q4_0", 1, KV, L, hd, 32)
    pos, count, q = _pos(100), _pos(n), _rand(1, n, H, hd).to(torch.float16).to(DEV)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attend(q, c.plan(pos, count, n))
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            plan = c.plan(pos, count, n)
            out = c.attend(q, plan)
    torch.cuda.synchronize()
    for at, m in ((1199, 1), (3, 90), (0, 0), (800, 7), (1000, 8), (7, 1), (1110, 90)):
        pos.fill_(at), count.fill_(m), q.normal_()
        g.replay()
        torch.cuda.synchronize()
        mine = c.plan(pos, count, n)
        assert torch.equal(out, c.attend(q, mine)) and not out[m:].any()
        if m:
            want, _, tol, _ = _packed_reference(c, q, mine)
            _check(out[:m], want[:m], tol, (at, m))
    assert _status() == 0


@pytest.mark.parametrize("page", [None, 32])
@pytest.mark.parametrize("at", [2 ** 63 - 1, 2 ** 63 - 3, 2 ** 62, 2 ** 31, 2 ** 32 + 5, -2 ** 63, -2 ** 63 + 2])
def test_positions_far_outside_the_cache(page, at):
    """A sequence at a position that no cache reaches (a server's mark of an unused place) brings tokens that are none: no sum of positions wraps round into the cache."""
    B, KV, H, hd, L, n = 3, 1, 4, 64, 100, 7
    c = _filled("q4_0", B, KV, L, hd, page)
    before = c.pages.clone()
    x, q = _rand(1, 3 * n, KV, hd).to(DEV), _rand(2, 3 * n, H, hd).to(DEV)
    for parents in (None, _i32([i - 1 for i in range(n)] * 3), _i32([-1] + [0] * (n - 1) + [-1] * n + [-1] + [0] * (n - 1))):
        plan = c.plan(_pos(5, at, 60), _pos(n, n, n), 3 * n, n, parents)
        assert plan.position[n:2 * n].tolist() == [-1] * n and plan.slot[n:2 * n].tolist() == [-1] * n and plan.start.tolist() == [5, at, 60]
        assert (plan.position[:n] >= 0).all() and (plan.position[2 * n:] >= 0).all()
        if parents is not None:
            assert not plan.sees[n:2 * n].any() and plan.nodes[:, 0].tolist() == [127, 0, 127]
        c.store(x, x, plan)
        for dt in ("f32", "bf16"):
            for kw in ({}, dict(window=20, sinks=5)):
                out = c.attend(q.to(TYPES[dt]), plan, **kw)
                assert not out[n:2 * n].any() and out[:n].any(-1).all() and out[2 * n:].any(-1).all()
        if parents is not None:
            assert c.keep(plan, _pos(2, 3, -1))[1:].tolist() == [at, 60]
        assert torch.equal(c.load(0, L)[0][1], _restored(c, before, 1))
    assert _status() & ~PAST_STORE == 0 and bool(_status() & PAST_STORE) == (at > 0)


def _restored(c, pages, b):
    """Sequence b's keys as another state of the memory has them."""
    now = c.pages.clone()
    c.pages.copy_(pages)
    k = c.load(0, c.max_seq)[0][b]
    c.pages.copy_(now)
    return k



@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("S,H", [(1, 4), (3, 4), (40, 256)])
def test_rectangles_far_outside_the_cache(dt, S, H):
    """The calls with a position a sequence, next to one that is served; a query past the cache sees all of it, or what its window leaves."""
    c = _filled("q4_0", 2, 1, 37, 64)
    q = _rand(3, 2, S, H, 64).to(TYPES[dt]).to(DEV)
    end = c.attend(q, _pos(20, 37 + 40))
    for at in (2 ** 62, 2 ** 63 - 1, 2 ** 63 - 2):
        for kw in ({}, dict(causal=False)):
            out = c.attend(q, _pos(20, at), **kw)
            assert torch.equal(out[1], end[1]) and out[0].any(-1).all(), (at, kw)
        for kw in (dict(window=9), dict(window=9, causal=False)):
            assert not c.attend(q, _pos(20, at), **kw)[1].any()
        assert torch.equal(c.attend(q, _pos(20, at), window=9, sinks=37)[1], c.attend(q, _pos(20, 37 + 40), window=9, sinks=37)[1])


@pytest.mark.parametrize("batch", [2, 4000])
def test_a_page_that_ends_behind_the_last_position_is_given_back(batch):
    """Rows of one page and a bit: `first` is compared with where the last page ends, which is past max_seq."""
    c = _paged(batch, 100, 64, 2 * batch)
    length = torch.full((batch,), 100, dtype=torch.int64, device=DEV)
    room, free = c.reserve(length)
    assert int(free) == 0 and (room == 100).all()
    before = c.page_table.clone()
    for first, needed in ((63, [True, True]), (64, [False, True]), (100, [False, True]), (127, [False, True]), (128, [False, False]), (2 ** 62, [False, False]), (2 ** 63 - 1, [False, False])):
        for sinks in (0, 64, 65):
            keep = torch.tensor([needed[0] or sinks > 0, needed[1] or sinks > 64], device=DEV)
            room, free = c.reserve(length, first=torch.full_like(length, first), sinks=sinks, table=before)
            assert torch.equal(c.page_table, torch.where(keep, before, -1)), (first, sinks)
            assert (room == 100).all() and int(free) == batch * (2 - int(keep.sum()))
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_each_sequence_by_itself(fmt, dt):
    """A norm and a logarithm's bound a sequence, by the kernel that serves its rows: of a long sequence among short ones no part is lost or taken twice, whose share of
    one norm over all rows is small."""
    L, H, KV, hd = 20000, 8, 2, 64
    c = _filled(fmt, 4, KV, L, hd, 128)
    for counts, starts in (([64, 70, 1, 64], [19900, 300, 5000, 0]), ([20, 100, 3, 0], [19980, 100, 9000, 4]), ([130, 0, 0, 0], [19870, 0, 0, 0]), ([6, 7, 1, 2], [19000, 12000, 19999, 6])):
        n = sum(counts)
        q = _rand(9, n, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
        plan = c.plan(_pos(*starts), _pos(*counts), n, 130)
        for kw in ({}, dict(window=7000, sinks=50)):
            lse, out = torch.full((n, H), 7.0, device=DEV), torch.full_like(q, math.nan)
            c.attend(q, plan, out=out, lse=lse, **kw)
            want, want_lse, tol, size = _packed_reference(c, q, plan, **kw)
            off = plan.offsets.tolist()
            for b, m in enumerate(counts):
                if m == 0:
                    continue
                r = slice(off[b], off[b + 1])
                _check(out[r], want[r], tol, (fmt, dt, counts, b, kw))
                # few rows: scores of the codes' own products, as test_gpu_kv_cache.py has it; many: a key's rounding to f16 is half a step, 2^-11 of it at most
                few = m * H // KV < (64 if dt == "f16" else 32)
                near = 2e-5 * max(1.0, float(want_lse[r].abs().max())) + (0.0 if few else 2.0 ** -11 * size)
                assert float((lse[r] - want_lse[r]).abs().max()) <= near, (fmt, dt, counts, b, kw)
    assert _status() == 0


def test_every_thread_has_compared_its_results():
    """Plans, packed attention of few and of many rows and page tables from four threads with streams of their own: all of them come to their end."""
    tables = [_paged(9, 700, 32, 100 + i) for i in range(4)]
    c = _filled("q4_0", 5, 2, 1000, 64, 32)
    counts = [[1, 1, 120, 0, 2], [30, 1, 17, 33, 1], [1] * 5, [150, 90, 3, 1, 40]]
    jobs = [(_pos(*((100 * b + 31 * i) % 800 for b in range(5))), _pos(*n), sum(n) + 2, _rand(i, sum(n) + 2, 8, 64).to(torch.float16 if i % 2 else torch.bfloat16).to(DEV),
             _pos(*((70 * b + 211 * i) % 700 for b in range(9)))) for i, n in enumerate(counts)]

    def work(i):
        pos, n, tokens, q, length = jobs[i]
        tables[i].page_table.fill_(-1)
        plan = c.plan(pos, n, tokens)
        return [c.attend(q, plan, window=200, sinks=9), c.attend(q, plan), plan.slot, *tables[i].reserve(length), tables[i].page_table.clone()]
    want = [[x.clone() for x in work(i)] for i in range(4)]
    torch.cuda.synchronize()
    compared, errors = [0] * 4, []

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    got = work(i)
                    torch.cuda.current_stream().synchronize()
                    compared[i] += all(torch.equal(x, y) for x, y in zip(got, want[i]))
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not errors and not any(t.is_alive() for t in threads) and compared == [60] * 4 and _status() == 0


@pytest.mark.parametrize("L", [120, 1000])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("starts,counts,room", [([900], [1], 1), ([900], [3], 80), ([10], [80], 80), ([700], [90], 300), ([0], [0], 70), ([900, 3], [1, 70], 90), ([5, 800, 60, 400], [1, 90, 8, 9], 200),
                                                ([-4], [3], 64), ([-70, 20], [70, 2], 80)])
def test_results_in_the_place_of_the_queries(L, dt, starts, counts, room):
    """Every row's query is read before its result is written, by whichever kernel has it."""
    c, starts = _filled("q4_0", len(starts), 2, L, 64, 32), [min(s, L - n) for s, n in zip(starts, counts)]
    q = _rand(3, room, 8, 64).to(TYPES[dt]).to(DEV)
    plan = c.plan(_pos(*starts), _pos(*counts), room)
    for kw in ({}, dict(window=200, sinks=9)):
        want, lse, mine = c.attend(q, plan, **kw), torch.full((room, 8), 7.0, device=DEV), q.clone()
        c.attend(mine, plan, out=mine, lse=lse, **kw)
        n = sum(counts)
        assert torch.equal(mine[:n], want[:n]) and torch.equal(mine[n:], q[n:]) and (lse[n:] == 7.0).all()
        assert torch.equal(torch.isfinite(lse[:n]), (plan.position[:n] >= 0)[:, None].expand(-1, 8))


def test_a_table_of_one_row_whatever_its_stride():
    """Of a dimension of one entry a stride means nothing, in the ordinary call as under a mode that looks at torch's operators."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from xn_b200.dtypes import GgmlDType
    from xn_b200.kv_cache import QuantizedKVCache

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    own = torch.full((4,), -1, dtype=torch.int32, device=DEV).as_strided((1, 4), (0, 1))
    c = QuantizedKVCache(GgmlDType.Q4_0, 1, 1, 128, 64, DEV, page_size=32, num_pages=9, page_table=own)
    table = _i32([5, 7, -1, 3]).as_strided((1, 4), (0, 1))
    assert table.stride(0) == 0 and table.is_contiguous()
    x = _rand(0, 3, 1, 64).to(DEV)
    for mode in (None, Watch()):
        c.page_table.fill_(-1)
        with mode if mode is not None else torch.no_grad():
            room, free = c.reserve(_pos(128), table=table)
            plan = c.plan(_pos(60), _pos(3), 3)
            c.store(x, x, plan)
        assert c.page_table.tolist() == [[5, 7, 0, 3]] and room.tolist() == [128] and int(free) == 5 and plan.slot.tolist() == [7 * 32 + 28 + i for i in range(3)]
    assert float((c.load(60, 3, torch.float32)[0][0, 0] - x[:, 0]).abs().max()) <= float(x.abs().max()) / 8 and _status() == 0
