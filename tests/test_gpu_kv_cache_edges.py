"""The quantized KV cache where it can go wrong between items, warps, halves and calls. Tolerances are those of test_gpu_kv_cache.py."""
import math
import sys
import threading
import time

import pytest
import torch

from test_gpu_kv_cache import DEV, TYPES, _cache, _check, _filled, _fmt, _init, _pos, _rand, _reference, _status  # noqa: F401 (_init: the module's fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,dt,S,H,group_of,lse", [("q4_0", "bf16", 1, 8, 4, True), ("q8_0", "bf16", 1, 8, 4, False), ("q4_0", "f32", 3, 8, 2, True), ("q8_0", "f16", 5, 12, 3, True)])
def test_rows_of_items_that_follow_one_another(fmt, dt, S, H, group_of, lse):
    """Ragged sequences, so that a CTA's run goes on from item to item: every row is stored where it belongs, in every call of many."""
    B, KV, L, hd = 96, H // group_of, 1500, 64
    c = _filled(fmt, B, KV, L, hd, 32)
    first = [int(S + (L - S) * ((i * 0.6180339887 + 0.5) % 1.0)) - S if i % 16 != 5 else -S for i in range(B)]
    q = _rand(9, B, S, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    pos = _pos(*first)
    k, v = c.load(0, L, dtype=torch.float32)
    want, want_lse, tol = _reference(k, v, q, first)
    made = []
    for _ in range(300):
        out = torch.full_like(q, math.nan)
        sums = torch.full((B, S, H), math.nan, device=DEV) if lse else None
        c.attend(q, pos, out=out, lse=sums)
        made.append((out, sums))
    _check(made[0][0], want, tol, (fmt, dt, S))
    if lse:
        seen = torch.isfinite(want_lse)
        assert float((made[0][1] - want_lse)[seen].abs().max()) <= 2e-5 * max(1.0, float(want_lse[seen].abs().max())) and bool((made[0][1][~seen] == -math.inf).all())
    for out, sums in made[1:]:
        assert torch.equal(out, made[0][0]) and (not lse or torch.equal(sums, made[0][1]))
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("S,hd", [(20, 128), (150, 128), (150, 64)])
def test_weights_stored_before_a_half_renews_its_reference(fmt, dt, S, hd):
    """Scores rise by some 13 (weights by 2^19) from the first tile of 32 of a half to the second, twice: the second tile asks for another reference when the
    first one's weights are already stored, and they are brought to it. The keys are whole multiples of a power of two, so that scores are exact however large:
    what is left is the tolerance's own terms."""
    B, H, KV, L = 2, 16, 4, 512
    c = _cache(fmt, B, KV, L, hd)
    level = ((torch.arange(L) >= 32).int() + (torch.arange(L) >= 160))[None, :, None, None]
    code = 3 * level + torch.randint(-1, 2, (B, L, KV, hd), generator=torch.Generator().manual_seed(4))
    code[..., ::32] = -8 if fmt == "q4_0" else 127        # a block's largest: its scale is 1/2
    c.store((code * 0.5).to(DEV), _rand(5, B, L, KV, hd).to(DEV), _pos(0))
    k, v = c.load(0, L, dtype=torch.float32)
    assert torch.equal(k.transpose(1, 2), (code * 0.5).to(DEV))
    q = _rand(6, B, S, H, hd, gain=1.0 if hd == 128 else 1.4).abs()
    q[..., ::32] = 0
    q = q.to(TYPES[dt]).to(DEV)
    first = [L - S, L - S - 45]
    got = c.attend(q, _pos(*first))
    want, _, tol = _reference(k, v, q, first)
    _check(got, want, tol, (fmt, dt, S))
    for _ in range(100):
        assert torch.equal(c.attend(q, _pos(*first)), got)
    assert _status() == 0


@pytest.mark.parametrize("S,own", [(64, True), (3, True), (64, False)])
def test_two_threads_on_one_stream(S, own):
    """Each call's parts stay its own, with results that it makes (C++) and with given ones (Python): the interpreter's lock is free while a call launches.
    A kernel that takes its time comes first, and the calls are more than the device's queue holds, so that launches block."""
    B, H, KV, hd, L = 1, 8, 2, 128, 16384
    c = _filled("q4_0", B, KV, L, hd)
    qs = [_rand(20 + i, B, S, H, hd).to(torch.bfloat16).to(DEV) for i in range(4)]
    pos = _pos(L - S)
    call = lambda q: c.attend(q, pos, out=torch.empty_like(q)) if own else c.attend(q, pos)
    want = [call(q) for q in qs]
    wrong, start = [], threading.Barrier(4)

    def work(i):
        for n in range(3):
            torch.cuda._sleep(100_000_000 if i == 0 else 1)
            start.wait()
            got = [call(qs[i]) for _ in range(400)]
            wrong.extend((i, n) for g in got if not torch.equal(g, want[i]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    assert not wrong, (len(wrong), wrong[:5])


def test_one_call_at_a_time_uses_a_workspace(monkeypatch):
    """The Python path: a call's kernels (two, where parts are joined) are enqueued before another call may use the same scratch."""
    from xn_b200 import kv_cache
    real, inside, together = kv_cache._lib.lib(), [], []

    class Slow:
        def __getattr__(self, name):
            return getattr(real, name)

        def xnq_kv_attend(self, *args):
            ws, here = args[12].value, threading.get_ident()
            inside.append((ws, here))
            time.sleep(0.005)
            together.extend(other for other in list(inside) if other[0] == ws and other[1] != here)
            rc = real.xnq_kv_attend(*args)
            inside.remove((ws, here))
            return rc
    c = _filled("q4_0", 1, 2, 256, 64)
    q, pos = _rand(2, 1, 1, 4, 64).to(DEV), _pos(255)
    c.attend(q, pos, out=torch.empty_like(q))
    monkeypatch.setattr(kv_cache._lib, "lib", Slow)
    threads = [threading.Thread(target=lambda: [c.attend(q, pos, out=torch.empty_like(q)) for _ in range(5)]) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not together and not inside


def test_scratch_is_kept_for_a_few_streams():
    from xn_b200 import kv_cache
    B, S, H, KV, hd, L = 1, 3, 8, 2, 64, 600
    c = _filled("q8_0", B, KV, L, hd)
    q, pos = _rand(3, B, S, H, hd).to(DEV), _pos(L - S)
    want = c.attend(q, pos, out=torch.empty_like(q))
    streams = [torch.cuda.Stream() for _ in range(40)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = c.attend(q, pos, out=torch.empty_like(q))
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
    assert len(kv_cache._workspaces) <= 16


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_blocks_with_infinities_and_nans_are_the_oracles(O, fmt, dt):
    inf, nan = math.inf, math.nan
    x = _rand(12, 16, 32)
    x[0], x[1], x[2], x[3] = inf, -inf, nan, 0.0
    x[4, ::2], x[4, 1::2] = -inf, nan
    x[5, ::2], x[5, 1::2] = inf, nan
    x[6, :16], x[6, 16:] = -inf, inf
    x[7, :16], x[7, 16:] = inf, -inf
    x[8, 31], x[9, 31], x[10, 31] = inf, -inf, nan
    x[11, 0], x[11, 31] = nan, -inf
    x[12], x[12, 5] = nan, 2.0
    x[13], x[13, 30] = nan, -2.0
    x[14], x[15] = -0.0, -1e-30
    x = x.view(1, 4, 2, 64).to(TYPES[dt])
    c = _cache(fmt, 1, 2, 4, 64)
    c.store(x.to(DEV), x.flip(1).contiguous().to(DEV), _pos(0))
    got = c.load(0, 4, dtype=torch.float32)
    for g, w in zip(got, (x, x.flip(1))):
        a = w.float().numpy()
        want = torch.from_numpy(O.to_float(int(_fmt(fmt)), O.from_float(int(_fmt(fmt)), a), a.size).reshape(a.shape)).transpose(1, 2).to(DEV)
        near = torch.equal if fmt == "q4_0" else lambda p, q: torch.allclose(p, q, rtol=2.0 ** -7, atol=0.0)   # (Q8_0's scale: a product with 1 / 127)
        assert torch.equal(torch.isnan(g), torch.isnan(want)) and near(torch.nan_to_num(g, nan=0.0), torch.nan_to_num(want, nan=0.0))


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("S", [20, 70, 300])
@pytest.mark.parametrize("k_gain,v_gain,q_gain", [(1e-3, 1e-6, 1e3), (300.0, 3e3, 1e-2), (1.0, 1e-3, 1.0), (1.0, 1e-6, 1.0), (1e-6, 1.0, 1.0)])
def test_scales_far_from_one_with_many_rows(fmt, dt, S, k_gain, v_gain, q_gain):
    """f16 results below its smallest normal number, 2^-14, keep that number's rounding: 2^-25 each."""
    B, KV, H, hd, L = 1, 2, 8, 128, 700
    c = _filled(fmt, B, KV, L, hd, k_gain=k_gain, v_gain=v_gain)
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(9, B, S, H, hd, gain=q_gain).to(TYPES[dt]).to(DEV)
    want, _, tol = _reference(k, v, q, [L - S])
    got = c.attend(q, _pos(L - S))
    if dt == "f16" and v_gain < 1e-2:
        assert float((got.double() - want).norm()) <= 2.0 ** -10 * float(want.norm()) + 2.0 ** -25 * want.numel() ** 0.5
    else:
        _check(got, want, tol, (fmt, dt, S, k_gain, v_gain, q_gain))


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("S", [1, 70, 300])
@pytest.mark.parametrize("gains", [(0.0, 1e-5, 1.0, 1e-3), (1.0, 1e-5, 30.0, 0.0), (1e-5, 0.0, 1e-3, 1e-5), (1e-4, 1e-5, 1e-4, 1e-6)])
def test_values_whose_size_changes_from_tile_to_tile(fmt, S, gains):
    """A whole tile of 32 positions after another, of zeros too, growing and shrinking."""
    B, KV, H, hd, L = 1, 2, 8, 128, 700
    c = _cache(fmt, B, KV, L, hd)
    size = torch.tensor(gains)[torch.arange(L) // 32 % 4][None, :, None, None]
    c.store(_rand(3, B, L, KV, hd).to(DEV), (_rand(4, B, L, KV, hd) * size).to(DEV), _pos(0))
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(9, B, S, H, hd, gain=1.5).to(torch.bfloat16).to(DEV)
    want, _, tol = _reference(k, v, q, [L - S])
    _check(c.attend(q, _pos(L - S)), want, tol, (fmt, S, gains))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("S", [1, 70])
@pytest.mark.parametrize("scale", [0.0, 1e-30, -1e-38, 1e-45])
def test_a_scale_near_nothing_averages_what_is_seen(dt, S, scale):
    """Also with queries near nothing: a hidden position's weight stays zero however small a score's factor is."""
    B, KV, H, hd, L = 2, 2, 8, 64, 200
    c = _filled("q4_0", B, KV, L, hd)
    k, v = c.load(0, L, dtype=torch.float32)
    for gain in (1.0, 1e-30):
        q = _rand(9, B, S, H, hd, gain=gain).to(TYPES[dt]).to(DEV)
        first = [L - S, 40 - S // 2]
        want, _, tol = _reference(k, v, q, first, scale=0.0)
        _check(c.attend(q, _pos(*first), scale=scale), want, tol, (dt, S, scale, gain))


def test_what_a_cache_is_made_of_is_not_replaced():
    """The kernels hold the addresses of its memory and its page table: both are filled in, never exchanged for others."""
    c = _cache("q4_0", 2, 2, 64, 64, 32)
    for name in ("pages", "page_table", "max_seq", "batch", "kv_heads", "head_dim", "page_size", "num_pages", "dtype", "device"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name))
    c.page_table.copy_(torch.arange(4).view(2, 2))
    assert c.page_table.data_ptr() == c._view.page_table and c.pages.data_ptr() == c._view.pages


def test_calls_that_torch_would_have_to_see_through_are_refused():
    """No gradient, tangent or trace comes out of these calls: with tensors that ask for one they say so."""
    from torch.autograd import forward_ad
    B, S, KV, H, hd, L = 1, 2, 2, 4, 64, 64
    c = _filled("q8_0", B, KV, L, hd)
    q, k, pos = _rand(1, B, S, H, hd).to(DEV), _rand(2, B, S, KV, hd).to(DEV), _pos(10)
    qkv, table = _rand(3, B, S, (H + 2 * KV) * hd).to(DEV), torch.zeros(L, hd // 2, device=DEV)
    want, before = c.attend(q, pos), c.pages.clone()
    ask = lambda t: t.clone().requires_grad_()
    calls = [lambda: c.attend(ask(q), pos), lambda: c.attend(ask(q), pos, out=torch.empty_like(q)), lambda: c.attend(ask(q).half(), pos), lambda: c.store(ask(k), k, pos),
             lambda: c.store(k, ask(k), pos), lambda: c.rope_store(ask(qkv), table, table, pos, H), lambda: c.rope_store(qkv, ask(table), table, pos, H),
             lambda: torch.func.vmap(lambda t: c.attend(t, pos))(q[None]), lambda: torch.func.grad(lambda t: c.attend(t, pos).sum())(q),
             lambda: torch.func.jvp(lambda t: c.attend(t, pos), (q,), (q,)), lambda: torch.jit.trace(lambda t: c.attend(t, pos), q, check_trace=False),
             lambda: torch.jit.trace(lambda t: (c.store(t, k, pos), t + 1)[1], k, check_trace=False)]

    def dual():
        with forward_ad.dual_level():
            c.attend(forward_ad.make_dual(q, q), pos)
    for i, call in enumerate(calls + [dual]):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i}")
    assert torch.equal(c.pages, before)
    with torch.no_grad():
        assert torch.equal(c.attend(ask(q), pos), want) and torch.equal(c.attend(ask(q), pos, out=torch.empty_like(q)), want)
    with torch.inference_mode():
        assert torch.equal(c.attend(ask(q), pos), want)
    assert torch.equal(c.attend(ask(q).detach(), pos), want) and not c.attend(q, pos).requires_grad


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("S", [1, 6, 70])
@pytest.mark.parametrize("sizes", [(0.3,), (0.05,), (0.05, 0.7, 0.02, 260.0, 0.3), (300.0, 0.05)])
def test_values_of_ordinary_and_other_sizes(fmt, dt, S, sizes):
    """On both sides of the ranges in which scales are taken as they are, and from one side to the other."""
    B, KV, H, hd, L = 2, 2, 8, 128, 500
    c = _cache(fmt, B, KV, L, hd)
    size = torch.tensor(sizes)[torch.arange(L) // 32 % len(sizes)][None, :, None, None]
    c.store((_rand(3, B, L, KV, hd) * size.clamp(max=1.0)).to(DEV), (_rand(4, B, L, KV, hd) * size).to(DEV), _pos(0))
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(9, B, S, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    first = [L - S, 333 - S]
    want, _, tol = _reference(k, v, q, first)
    _check(c.attend(q, _pos(*first)), want, tol, (fmt, dt, S, sizes))
    assert _status() == 0
