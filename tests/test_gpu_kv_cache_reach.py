"""The quantized KV cache's kernels where other tests do not reach: parts of many sizes and numbers, more sequences than a CTA has threads, scales that are
not finite in every place that some query does not see, Q8_0's blocks beside the oracle's. Tolerances are those of test_gpu_kv_cache.py."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import DEV, TYPES, _cache, _check, _filled, _init, _pos, _rand, _reference, _status  # noqa: F401 (_init: the module's fixture)

pytestmark = pytest.mark.gpu


def _log_sums(got, want, dt, many):
    seen = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), seen) and bool((got[~seen] == -math.inf).all())
    near = 2e-5 if not many or dt == "f32" else 2e-3 if dt == "bf16" else 2e-4
    assert float((got - want)[seen].abs().max()) <= near * max(1.0, float(want[seen].abs().max()))


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("B,S,H,KV,hd,L,window,first", [
    (1, 64, 1, 1, 64, 16384, 0, [16320]),        # 64 parts of one row tile: more than a warp has lanes
    (1, 100, 1, 1, 128, 16384, 0, [16284]),      # the same, an odd number of rows
    (1, 128, 1, 1, 128, 16384, 0, [500]),        # a short sequence in a large cache: most parts have no step
    (1, 128, 2, 1, 64, 8192, 300, [7000]),       # a window: few steps for many parts
    (2, 33, 4, 2, 64, 3000, 0, [2967, -10]),     # five to twelve parts; a sequence that begins in the call
    (3, 70, 2, 2, 128, 2600, 1, [2000, -70, 64]),
    (1, 513, 4, 4, 64, 2048, 0, [1000]),         # several row tiles and parts
])
def test_parts_of_many_rows(fmt, dt, B, S, H, KV, hd, L, window, first):
    c = _filled(fmt, B, KV, L, hd, seed=S)
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(31, B, S, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    lse, out = torch.full((B, S, H), 7.0, device=DEV), torch.full_like(q, math.nan)
    c.attend(q, _pos(*first), window=window, out=out, lse=lse)
    want, want_lse, tol = _reference(k, v, q, first, window=window)
    _check(out, want, tol, (fmt, dt, B, S, H, KV, hd, L))
    _log_sums(lse, want_lse, dt, True)
    for _ in range(20):
        assert torch.equal(c.attend(q, _pos(*first), window=window), out)
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B,S,L,page", [(129, 1, 70, None), (300, 1, 400, 32), (300, 3, 1100, None), (257, 9, 300, 64)])
def test_more_sequences_than_a_cta_has_threads(fmt, dt, B, S, L, page):
    H, KV, hd = 4, 2, 64
    c = _filled(fmt, B, KV, L, hd, page)
    k, v = c.load(0, L, dtype=torch.float32)
    first = [-S if i % 7 == 3 else int((L - S) * ((i * 0.6180339887 + 0.5) % 1.0)) for i in range(B)]
    q = _rand(8, B, S, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    lse, out = torch.full((B, S, H), 7.0, device=DEV), torch.full_like(q, math.nan)
    c.attend(q, _pos(*first), out=out, lse=lse)
    want, want_lse, tol = _reference(k, v, q, first)
    _check(out, want, tol, (fmt, dt, B, S, L, page))
    _log_sums(lse, want_lse, dt, S * H // KV >= 64)
    for _ in range(20):
        assert torch.equal(c.attend(q, _pos(*first)), out)
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
def test_both_kernels_share_a_workspace(fmt):
    """16-bit queries: many rows whose parts are joined by a kernel of its own, few rows whose parts are counted, in turns on one workspace."""
    B, H, KV, hd, L = 1, 8, 2, 128, 8192
    c = _filled(fmt, B, KV, L, hd)
    k, v = c.load(0, L, dtype=torch.float32)
    calls = []
    for S in (1, 16, 70, 300, 5):
        q = _rand(S, B, S, H, hd).to(torch.bfloat16).to(DEV)
        got = c.attend(q, _pos(L - S))
        want, _, tol = _reference(k, v, q, [L - S])
        _check(got, want, tol, (fmt, S))
        calls.append((q, _pos(L - S), got))
    for i in range(60):
        for q, pos, want in calls[::1 if i % 2 else -1]:
            assert torch.equal(c.attend(q, pos), want)
            assert torch.equal(c.attend(q, pos, out=torch.empty_like(q)), want)


def _scales_to_nan(c, fmt, b, positions, keys=True, values=True):
    """The scales of these positions, in every head: a tile is 32 rows of K's codes, K's scales by row, V's codes, V's scales by pairs of rows."""
    rb, nb = c.head_dim // 2 if fmt == "q4_0" else c.head_dim, c.head_dim // 32
    tile = 32 * 2 * (rb + 2 * nb)
    words = c.pages[b].view(c.kv_heads, -1, tile)
    for j in positions:
        t, r = j // 32, j % 32
        at_k, at_v = 32 * rb + r * nb * 2, 32 * rb + 32 * nb * 2 + 32 * rb + (r // 2) * nb * 4 + (r % 2) * 2
        if keys:
            words[:, t, at_k:at_k + 2 * nb] = 0xff
        if values:
            for block in range(nb):
                words[:, t, at_v + 4 * block:at_v + 4 * block + 2] = 0xff


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt,S", [("f32", 1), ("f32", 40), ("bf16", 1), ("f16", 5), ("bf16", 70), ("f16", 300)])
@pytest.mark.parametrize("window", [0, 37])
def test_scales_that_nobody_sees_change_no_bit(fmt, dt, S, window):
    """NaN behind the last position, and below the window's lower edge, up to the very neighbours of what is seen."""
    B, KV, H, hd, L = 2, 2, 8, 128, 480
    c = _filled(fmt, B, KV, L, hd)
    q = _rand(9, B, S, H, hd).to(TYPES[dt]).to(DEV)
    first = [133, 97]
    want = c.attend(q, _pos(*first), window=window)
    k, v = c.load(0, L, dtype=torch.float32)
    ref, _, tol = _reference(k, v, q, first, window=window)
    _check(want, ref, tol, (fmt, dt, S, window))
    for b, p in enumerate(first):
        _scales_to_nan(c, fmt, b, range(p + S, L))
        if window:
            _scales_to_nan(c, fmt, b, range(0, p - window + 1))
    assert torch.equal(c.attend(q, _pos(*first), window=window), want)
    assert torch.isnan(c.load(0, L, dtype=torch.float32)[0]).any() and _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt,S", [("f32", 40), ("bf16", 7), ("f16", 70), ("bf16", 300)])
@pytest.mark.parametrize("which", ["keys", "values", "both"])
@pytest.mark.parametrize("window,bad", [(0, 140), (0, 163), (20, 150), (20, 120)])
def test_a_scale_that_is_not_finite_reaches_exactly_the_rows_that_see_it(fmt, dt, S, which, window, bad):
    B, KV, H, hd, L, first = 1, 2, 8, 64, 480, [134]
    c = _filled(fmt, B, KV, L, hd)
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(9, B, S, H, hd).to(TYPES[dt]).to(DEV)
    want, _, tol = _reference(k, v, q, first, window=window)
    _scales_to_nan(c, fmt, 0, [bad], keys=which != "values", values=which != "keys")
    got = c.attend(q, _pos(*first), window=window)
    p = first[0] + torch.arange(S)
    sees = (bad <= p) & ((p - window < bad) if window else torch.ones(S, dtype=torch.bool))
    assert torch.isnan(got[0, sees.to(DEV)]).all()
    if not sees.all():
        _check(got[:, ~sees.to(DEV)], want[:, ~sees.to(DEV)], tol, (fmt, dt, S, which, window, bad))
    assert _status() == 0


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_q8_0_blocks_are_the_oracles_but_at_ties(O, dt):
    """The scale is max|x| times the f32 nearest 1 / 127, the oracle's max|x| divided by 127. Both are max|x| / 127 to 2^-23, and a code is x times the scale's
    reciprocal, so a code can differ only where x / scale is a whole number and a half to 127 * 2^-21, and then by one."""
    n, KV, hd = 4096, 8, 128
    x = (_rand(41, 1, n, KV, hd) * torch.exp(_rand(42, 1, n, KV, 1))).to(TYPES[dt])
    c = _cache("q8_0", 1, KV, n, hd)
    c.store(x.to(DEV), x.to(DEV), _pos(0))
    got = [t.transpose(1, 2).cpu().double().numpy().reshape(-1, 32) for t in c.load(0, n, dtype=torch.float32)]
    assert np.array_equal(got[0], got[1])
    a = x.float().numpy()
    want = O.to_float(8, O.from_float(8, a), a.size).astype(np.float64).reshape(-1, 32)
    step = np.abs(a.reshape(-1, 32).astype(np.float64)).max(1, keepdims=True) / 127
    half = np.abs(np.abs(a.reshape(-1, 32) / step) % 1 - 0.5)
    codes = [np.rint(t / step) for t in (got[0], want)]
    other = codes[0] != codes[1]
    assert np.all(half[other] <= 127 * 2.0 ** -21) and np.all(np.abs(codes[0] - codes[1]) <= 1)
    assert np.mean(other) < 2e-4                               # bf16 rows, which have the most ties: 5e-5
    same = ~other
    assert np.all(np.abs(got[0] - want)[same] <= 2.0 ** -10 * np.abs(want)[same])   # the f16 scale's last bit, if that
    if dt != "f32":
        assert np.array_equal(got[0][same], want[same])


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("B,S,H,KV,hd,L", [(1, 1, 8, 2, 128, 131072), (4, 1, 4, 2, 64, 40000), (1, 5, 14, 2, 64, 16384), (1, 64, 8, 2, 128, 8192), (16, 1, 8, 2, 128, 200)])
def test_f32_queries_are_as_exact_as_f32_products(fmt, B, S, H, KV, hd, L):
    """At most one and a half times the error that products, weights and sums in f32 have on the same blocks, or 1e-6 of the result's norm."""
    c = _filled(fmt, B, KV, L, hd, v_gain=0.7)
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(9, B, S, H, hd, gain=1.5).to(DEV)
    at = torch.arange(L, device=DEV) > torch.arange(L - S, L, device=DEV)[:, None]

    def result(kind):
        rows = q.to(kind).view(B, S, KV, H // KV, hd).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, hd)
        score = (rows @ k.to(kind).transpose(-1, -2) * hd ** -0.5).view(B, KV, H // KV, S, L).masked_fill(at, -math.inf)
        weight = torch.exp(score - score.amax(-1, keepdim=True))
        out = (weight.view(B, KV, -1, L) @ v.to(kind)).view(B, KV, H // KV, S, hd) / weight.sum(-1, keepdim=True)
        return out.permute(0, 3, 1, 2, 4).reshape(B, S, H, hd).double()
    want = result(torch.float64)
    error = lambda x: float((x.double() - want).norm() / want.norm())
    assert error(c.attend(q, _pos(L - S))) <= max(1.5 * error(result(torch.float32)), 1e-6)
