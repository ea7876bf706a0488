"""The quantized KV cache: blocks against the oracle bit for bit, attention against plain 64-bit arithmetic on what the blocks stand for.

Tolerances. f32 queries: |err| <= V (4 u (hd / 16 + 16) S + 64 u), u = 2^-24, V = max |v|, S the largest sum of |scale q_i k_i| of a visible pair: a score
is off by at most its rounding, an output by twice the scores' times V, and by its own sums. 16-bit queries: the 2-norm of the error is below half a unit
of the output's type (2^-9, 2^-12) for its rounding, as much for the weights' (and, in the kernel for many queries, the keys' and values') rounding, doubled:
2^-7.5 -> 2^-8 for bf16, 2^-10 for f16."""
import ctypes
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _init():
    from xn_b200 import _lib, quantized
    quantized.init(DEV)
    _lib.check(_lib.lib().xnq_init(0))   # the status word starts at zero
    yield
    _lib.check(_lib.lib().xnq_init(0))


def _status():
    from xn_b200 import _lib
    st = ctypes.c_uint()
    _lib.check(_lib.lib().xnq_device_status(ctypes.byref(st)))
    return st.value


def _fmt(name):
    from xn_b200.dtypes import GgmlDType
    return GgmlDType.Q4_0 if name == "q4_0" else GgmlDType.Q8_0


def _cache(fmt, B, KV, L, hd, page=None, seed=0):
    """A cache, by pages in a random order where `page` says so."""
    from xn_b200.kv_cache import QuantizedKVCache
    if not page:
        return QuantizedKVCache(_fmt(fmt), B, KV, L, hd, DEV)
    per = -(-L // page)
    c = QuantizedKVCache(_fmt(fmt), B, KV, L, hd, DEV, page_size=page, num_pages=B * per + 3)
    g = torch.Generator().manual_seed(seed)
    c.page_table.copy_(torch.randperm(B * per + 3, generator=g)[:B * per].view(B, per))
    return c


def _rand(seed, *shape, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g) * gain


def _pos(*p):
    return torch.tensor(p, dtype=torch.int64, device=DEV)


def _held(O, fmt, x):
    """What the blocks of the f32 rows stand for: Q4_0 the oracle's, Q8_0 with its scale formed by a product with 1 / 127."""
    a = x.float().cpu().numpy()
    if fmt == "q8_0":
        blocks = a.reshape(-1, 32)
        d = np.abs(blocks).max(1, keepdims=True) * (np.float32(1) / np.float32(127))
        with np.errstate(divide="ignore"):
            y = blocks * np.where(d != 0, np.float32(1) / d, np.float32(0))
        code = np.sign(y) * np.floor(np.abs(y).astype(np.float64) + 0.5)
        held = (code.astype(np.float32) * d.astype(np.float16).astype(np.float32)).reshape(a.shape)
        near = O.to_float(8, O.from_float(8, a), a.size).reshape(a.shape)   # the file's quantizer: a last bit of the scale, a code at a tie
        assert np.all(np.abs(held - near) <= np.repeat(np.abs(blocks).max(1), 32).reshape(a.shape) * (1 / 127 + 2.0 ** -11))
        assert np.mean(held != near) < 0.02
        return torch.from_numpy(held).to(DEV)
    return torch.from_numpy(O.to_float(int(_fmt(fmt)), O.from_float(int(_fmt(fmt)), a), a.size).reshape(a.shape)).to(DEV)


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,KV,S,L,hd,page,start", [(1, 1, 1, 1, 64, None, 0), (1, 8, 1, 512, 128, None, 511), (2, 3, 5, 40, 128, None, 31), (3, 2, 33, 100, 64, 32, 3),
                                                    (2, 8, 64, 200, 128, 64, 64), (1, 2, 67, 70, 128, 32, 1)])
def test_stored_blocks_are_the_oracles(O, fmt, dt, B, KV, S, L, hd, page, start):
    c = _cache(fmt, B, KV, L, hd, page)
    k, v = (_rand(7 * S + i, B, S, KV, hd, gain=3.0).to(TYPES[dt]) for i in (0, 1))
    k[0, 0, 0, :32] = 0                                         # a block of zeros
    v[0, S - 1, KV - 1, 32:64] = torch.tensor([1.0, -1.0] * 16)   # equal magnitudes: the first one's sign
    k[0, S - 1, 0, 32:64] = torch.tensor([-2.0, 2.0] * 16)
    v[B - 1, 0, 0, :32] *= 1e-6
    c.store(k.to(DEV), v.to(DEV), _pos(start))
    want_k, want_v = (_held(O, fmt, x).transpose(1, 2) for x in (k, v))
    got_k, got_v = c.load(start, S, dtype=torch.float32)
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)
    for t in TYPES.values():
        a, b = c.load(start, S, dtype=t)
        assert torch.equal(a, want_k.to(t)) and torch.equal(b, want_v.to(t))
    whole = c.load(0, L, dtype=torch.float32)
    for w, want in zip(whole, (want_k, want_v)):                # nothing else was touched
        assert torch.equal(w[:, :, start:start + S], want)
        w[:, :, start:start + S] = 0
        assert not w.any()
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_of_two_equal_magnitudes_the_first_gives_the_sign(O, fmt, dt):
    """Every ordered pair of places of a block's largest values, one positive and one negative."""
    x = (_rand(21, 992, 32).clamp(-1, 1) * 0.9)
    pairs = [(i, j) for i in range(32) for j in range(32) if i != j]
    for n, (i, j) in enumerate(pairs):
        x[n, i], x[n, j] = 2.0, -2.0
    x = x.view(1, 496, 1, 64).to(TYPES[dt])
    c = _cache(fmt, 1, 1, 496, 64)
    c.store(x.to(DEV), x.flip(1).contiguous().to(DEV), _pos(0))
    got_k, got_v = c.load(0, 496, dtype=torch.float32)
    assert torch.equal(got_k, _held(O, fmt, x).transpose(1, 2)) and torch.equal(got_v, _held(O, fmt, x.flip(1)).transpose(1, 2))


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
def test_tokens_one_at_a_time_and_at_own_positions(O, fmt):
    """Positions of their own, odd and even, in any order: a pair of positions shares words of the values' codes."""
    B, KV, L, hd = 3, 2, 65, 128
    c = _cache(fmt, B, KV, L, hd, 32)
    k, v = (_rand(i, B, L, KV, hd).to(DEV) for i in (0, 1))
    for step in range(L):
        at = [(step * 7 + 11 * b) % L for b in range(B)]
        rows = torch.arange(B), torch.tensor(at)
        c.store(k[rows][:, None], v[rows][:, None], _pos(*at))
    got = c.load(0, L, dtype=torch.float32)
    assert torch.equal(got[0], _held(O, fmt, k).transpose(1, 2)) and torch.equal(got[1], _held(O, fmt, v).transpose(1, 2))
    starts = _pos(0, 13, 60)
    part = c.load(starts, 5, dtype=torch.float32)
    for b, s in enumerate((0, 13, 60)):
        assert torch.equal(part[0][b], got[0][b, :, s:s + 5]) and torch.equal(part[1][b], got[1][b, :, s:s + 5])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_strided_and_unaligned_rows(O, dt):
    B, KV, S, hd = 2, 4, 9, 64
    x = _rand(5, B, KV, S, hd).to(TYPES[dt]).to(DEV)
    fused = _rand(6, B, S, 3 * KV * hd + 8).to(TYPES[dt]).to(DEV)
    odd = torch.empty(B * S * KV * hd + 1, dtype=TYPES[dt], device=DEV)[1:].view(B, S, KV, hd).copy_(x.transpose(1, 2))   # not 16-byte aligned
    every_other = _rand(8, B, S, KV, 2 * hd).to(TYPES[dt]).to(DEV)[..., ::2]
    same = _rand(9, 1, S, 1, hd).to(TYPES[dt]).to(DEV).expand(B, S, KV, hd)
    for k, v in [(x.transpose(1, 2), fused[..., KV * hd:2 * KV * hd].unflatten(2, (KV, hd))), (odd, every_other), (same, odd)]:
        c = _cache("q8_0", B, KV, 20, hd)
        c.store(k, v, _pos(3, 10))
        got = c.load(_pos(3, 10), S, dtype=torch.float32)
        assert torch.equal(got[0], _held(O, "q8_0", k.contiguous()).transpose(1, 2)) and torch.equal(got[1], _held(O, "q8_0", v.contiguous()).transpose(1, 2))


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,S,H,KV,hd", [(1, 1, 4, 4, 128), (3, 7, 6, 2, 64), (2, 33, 8, 1, 128)])
def test_rotation_before_the_store(O, fmt, dt, B, S, H, KV, hd):
    L = 80
    c = _cache(fmt, B, KV, L, hd, 32)
    qkv = _rand(S, B, S, (H + 2 * KV) * hd).to(TYPES[dt])
    ang = torch.arange(L, dtype=torch.float32)[:, None] / 10000.0 ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd)[None]
    cos, sin = ang.cos(), ang.sin()
    first = [5 + 11 * b for b in range(B)]
    at = torch.tensor(first)[:, None] + torch.arange(S)
    x = qkv.float().unflatten(2, (-1, hd))

    def turned(t):
        a, b = t[..., :hd // 2], t[..., hd // 2:]
        cs, sn = cos[at][:, :, None], sin[at][:, :, None]
        return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)
    q = c.rope_store(qkv.to(DEV), cos.to(DEV), sin.to(DEV), _pos(*first), H)
    assert q.dtype is TYPES[dt] and torch.equal(q.cpu(), turned(x[:, :, :H]).to(TYPES[dt]))
    got = c.load(_pos(*first), S, dtype=torch.float32)
    assert torch.equal(got[0], _held(O, fmt, turned(x[:, :, H:H + KV])).transpose(1, 2))
    assert torch.equal(got[1], _held(O, fmt, x[:, :, H + KV:]).transpose(1, 2))
    q16 = c.rope_store(qkv.to(DEV), cos.to(DEV), sin.to(DEV), _pos(*first), H, out_dtype=torch.bfloat16)
    assert torch.equal(q16.cpu(), turned(x[:, :, :H]).to(torch.bfloat16))


def test_tokens_that_are_not_there():
    """Negative positions store nothing; positions past the cache and pages that are not there set their bits and touch nothing."""
    from xn_b200 import _lib
    B, KV, L, hd = 3, 2, 40, 64
    c = _cache("q4_0", B, KV, L, hd)
    k, v = (_rand(i, B, 4, KV, hd).to(DEV) for i in (0, 1))
    c.store(k, v, _pos(-4, -2, 0))                       # an idle slot, two tokens of padding, all four
    got = c.load(0, L, dtype=torch.float32)
    assert not got[0][0].any() and not got[1][0].any()
    assert got[0][1][:, :2].any() and not got[0][1][:, 2:].any() and got[0][2][:, :4].any(-1).all()
    assert _status() == 0
    before = c.pages.clone()
    c.store(k, v, _pos(-4, L + 5, L))
    assert torch.equal(c.pages, before) and _status() == 1 << 27
    _lib.check(_lib.lib().xnq_init(0))
    p = _cache("q8_0", B, KV, L, hd, 32)
    p.page_table[1, 1] = -1
    p.page_table[2, 0] = p.num_pages
    before = p.pages.clone()
    p.store(k, v, _pos(-4, 33, 7))
    assert torch.equal(p.pages, before) and _status() == 1 << 29
    a, b = p.load(_pos(0, 33, 7), 4, dtype=torch.float32)
    assert not a.any() and not b.any()
    _lib.check(_lib.lib().xnq_init(0))


def _reference(k, v, q, first, causal=True, window=0, scale=None, max_seq=None):
    """f64: (out [B, S, H, hd], lse [B, S, H], the f32 tolerance) from k, v [B, KV, L, hd] as read back in f32."""
    B, S, H, hd = q.shape
    KV, L = k.shape[1:3]
    scale = hd ** -0.5 if scale is None else scale
    kk, vv = (x.double().repeat_interleave(H // KV, 1) for x in (k, v))
    qq = q.double().transpose(1, 2)
    p = torch.tensor(first, device=DEV)[:, None] + torch.arange(S, device=DEV)
    hi = p if causal else (p[:, -1:] + torch.zeros_like(p))
    j = torch.arange(L, device=DEV)
    seen = (j <= hi[..., None]) & (p[..., None] >= 0)
    if window:
        seen &= j > p[..., None] - window
    seen = seen[:, None]
    score = (qq @ kk.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(score, -1)
    w = torch.where(seen, torch.exp(score - lse.masked_fill(lse == -math.inf, 0.0)[..., None]), 0.0)
    size = ((qq.abs() @ kk.abs().transpose(-1, -2)) * abs(scale)).masked_fill(~seen, 0.0).max()
    u = 2.0 ** -24
    tol = float(v.abs().max()) * (4 * u * (hd / 16 + 16) * float(size) + 64 * u)
    vv = torch.where(torch.isfinite(vv), vv, 0.0) if not torch.isfinite(vv).all() else vv
    return (w @ vv).transpose(1, 2), lse.transpose(1, 2), tol


def _check(got, want, tol, what):
    assert torch.isfinite(got.double()).all(), what
    err = got.double() - want
    if got.dtype is torch.float32:
        assert float(err.abs().max()) <= tol, (what, float(err.abs().max()), tol)
    else:
        bound = 2.0 ** -8 if got.dtype is torch.bfloat16 else 2.0 ** -10
        assert float(err.norm()) <= bound * float(want.norm()) + 1e-30, (what, float(err.norm() / want.norm()))


def _filled(fmt, B, KV, L, hd, page=None, seed=3, k_gain=1.0, v_gain=1.0):
    c = _cache(fmt, B, KV, L, hd, page, seed)
    gain = torch.exp(0.5 * torch.cos(torch.arange(hd) * 2.4))
    c.store((_rand(seed, B, L, KV, hd, gain=k_gain) * gain).to(DEV), _rand(seed + 1, B, L, KV, hd, gain=v_gain).to(DEV), _pos(0))
    return c


ATTEND = [  # B, S, H, KV, hd, L, page, first positions
    (1, 1, 1, 1, 128, 1, None, [0]), (1, 1, 32, 8, 128, 512, None, [511]), (1, 1, 4, 4, 64, 33, None, [32]), (2, 1, 8, 1, 128, 300, 64, [0, 299]),
    (16, 1, 32, 8, 128, 200, None, [199] * 16), (5, 1, 28, 4, 64, 1000, 32, [999, 31, 32, 500, -1]), (3, 5, 14, 2, 64, 400, None, [0, 395, 130]),
    (2, 9, 12, 12, 128, 90, 32, [-4, 81]), (2, 3, 40, 2, 128, 257, None, [100, 254]), (1, 17, 8, 8, 128, 50, None, [20]),
    (2, 64, 8, 2, 128, 200, None, [0, 101]), (1, 128, 8, 2, 64, 300, 32, [172]), (1, 200, 16, 2, 128, 200, None, [0]), (2, 131, 6, 3, 128, 450, 64, [-31, 300]),
    (4, 300, 32, 16, 128, 700, 64, [0, 400, 33, 399]), (3, 260, 64, 32, 64, 900, None, [640, 0, 7])]   # as many rows as take two tiles a CTA


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,S,H,KV,hd,L,page,first", ATTEND)
def test_attention(fmt, dt, B, S, H, KV, hd, L, page, first):
    c = _filled(fmt, B, KV, L, hd, page, seed=B + S)
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(77, B, S, H, hd, gain=1.5).to(TYPES[dt]).to(DEV)
    lse = torch.full((B, S, H), 7.0, device=DEV)
    got = c.attend(q, _pos(*first), lse=lse)
    want, want_lse, tol = _reference(k, v, q, first)
    _check(got, want, tol, (fmt, dt, B, S, H, KV, hd, L, page))
    seen = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse), seen) and bool((lse[~seen] == -math.inf).all()) and not got[~seen].any()
    near = 2e-3 if dt == "bf16" and S * H // KV >= 64 else 2e-4 if S * H // KV >= 64 and dt != "f32" else 2e-5   # keys in 16 bits: a score's error averages out
    assert float((lse - want_lse)[seen].abs().max() if seen.any() else 0.0) <= near * max(1.0, float(want_lse[seen].abs().max() if seen.any() else 0))
    assert torch.equal(c.attend(q, _pos(*first)), got)   # the order of no sum depends on who came first
    assert _status() == 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("S,H,KV", [(1, 8, 2), (6, 8, 2), (150, 8, 2), (40, 3, 3)])
@pytest.mark.parametrize("causal,window,scale", [(False, 0, None), (True, 1, None), (True, 33, 0.3), (False, 50, None), (True, 10000, -0.05), (True, 0, 0.0)])
def test_masks_and_scales(dt, S, H, KV, causal, window, scale):
    B, L, hd = 3, 333, 128
    c = _filled("q4_0", B, KV, L, hd, 64)
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(9, B, S, H, hd).to(TYPES[dt]).to(DEV)
    first = [L - S, -S // 2, 100]
    got = c.attend(q, _pos(*first), causal=causal, window=window, scale=scale)
    want, _, tol = _reference(k, v, q, first, causal, window, scale)
    _check(got, want, tol, (dt, S, causal, window))


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dt,S", [("f32", 1), ("bf16", 1), ("f16", 3), ("bf16", 70)])
def test_what_lies_past_a_sequence_is_not_seen(fmt, dt, S):
    """Rows behind the position (another request's, memory never written: infinite and NaN scales) change no bit."""
    B, KV, H, hd, L = 2, 2, 8, 128, 160
    c = _filled(fmt, B, KV, L, hd)
    q = _rand(9, B, S, H, hd).to(TYPES[dt]).to(DEV)
    first = _pos(77, 90)
    want = c.attend(q, first)
    k, v = c.load(0, L, dtype=torch.float32)
    raw = c.pages.clone()
    c.pages.fill_(0xff)                                    # every scale a NaN
    c.store(k.transpose(1, 2)[:1, :77 + S].expand(B, -1, -1, -1), v.transpose(1, 2)[:1, :77 + S].expand(B, -1, -1, -1), _pos(0, -1000))
    c.store(k.transpose(1, 2)[1:, :90 + S].expand(B, -1, -1, -1), v.transpose(1, 2)[1:, :90 + S].expand(B, -1, -1, -1), _pos(-1000, 0))
    again = c.load(0, 78, dtype=torch.float32)
    same = torch.equal(again[0][:, :, :78], k[:, :, :78]) and torch.equal(again[1][:, :, :78], v[:, :, :78])
    if same:   # (what blocks stand for need not quantize to the same blocks)
        assert torch.equal(c.attend(q, first), want)
    got = c.attend(q, first)
    kk, vv = c.load(0, L, dtype=torch.float32)
    ref, _, tol = _reference(torch.nan_to_num(kk), torch.nan_to_num(vv), q, [77, 90])
    _check(got, ref, tol, (fmt, dt, S))
    c.pages.copy_(raw)
    assert torch.equal(c.attend(q, first), want)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k_gain,v_gain,q_gain", [(1e-3, 1e-6, 1e3), (300.0, 3e4, 1e-2), (1.0, 1e-7, 1.0), (40.0, 1.0, 40.0), (1e-7, 1.0, 1.0)])
def test_scales_far_from_one(dt, k_gain, v_gain, q_gain):
    """Values far from one keep their accuracy: nothing overflows or sinks below f16's smallest numbers on the way."""
    B, KV, H, hd, L = 1, 2, 8, 128, 300
    c = _filled("q4_0", B, KV, L, hd, k_gain=k_gain, v_gain=v_gain)
    k, v = c.load(0, L, dtype=torch.float32)
    q = _rand(9, B, 1, H, hd, gain=q_gain).to(TYPES[dt]).to(DEV)
    want, _, tol = _reference(k, v, q, [L - 1])
    got = c.attend(q, _pos(L - 1))
    if dt == "f16" and v_gain < 1e-4:
        tol = None   # the results themselves sink below f16's smallest numbers
        assert float((got.double() - want).abs().max()) <= 2.0 ** -10 * float(want.abs().max()) + 2.0 ** -24
    else:
        _check(got, want, tol, (dt, k_gain, v_gain, q_gain))


def test_a_long_cache_and_offsets_past_32_bits():
    """More than 2^32 bytes of pages: the last sequence's rows lie behind them."""
    KV, H, hd, L, B = 8, 8, 128, 65536, 66
    c = _cache("q8_0", B, KV, L, hd)
    assert c.nbytes > 2 ** 33
    at = L - 3000
    k, v = (_rand(i, 1, 3000, KV, hd).to(DEV) for i in (0, 1))
    nobody = [-10 ** 9] * (B - 1)
    c.store(k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), _pos(*nobody, at))
    got_k, got_v = c.load(_pos(*([0] * (B - 1)), at), 3000, dtype=torch.float32)
    assert not got_k[:-1].any() and got_k[-1].any()
    q = _rand(3, 1, 1, H, hd).to(DEV).expand(B, -1, -1, -1)
    out = c.attend(q, _pos(*nobody, L - 1), window=3000)
    want, _, tol = _reference(got_k[-1:], got_v[-1:], q[-1:], [2999])
    assert not out[:-1].any()
    _check(out[-1:], want, tol, "long")
    whole = c.attend(q[:, :, :], _pos(*nobody, L - 1))       # and over all 65536 positions: the others are rows of zeros
    zk = torch.zeros(1, KV, L, hd, device=DEV); zv = torch.zeros_like(zk)
    zk[:, :, at:], zv[:, :, at:] = got_k[-1], got_v[-1]
    want, _, tol = _reference(zk, zv, q[-1:], [L - 1])
    _check(whole[-1:], want, tol, "longer")


def test_positions_past_the_cache_and_missing_pages_are_reported():
    from xn_b200 import _lib
    B, KV, H, hd, L = 2, 2, 4, 64, 64
    for S in (1, 80):
        c = _filled("q8_0", B, KV, L, hd, 32)
        k, v = c.load(0, L, dtype=torch.float32)
        q = _rand(S, B, S, H, hd).to(torch.bfloat16).to(DEV)
        got = c.attend(q, _pos(L + 9 - S, 3 - S))
        assert _status() == 1 << 28
        want, _, tol = _reference(k, v, q, [L + 9 - S, 3 - S])
        _check(got, want, tol, "past")
        _lib.check(_lib.lib().xnq_init(0))
        c.page_table[0, 0] = -5                               # the first half of sequence 0 has no page
        got = c.attend(q, _pos(L - S, 2 - S))
        assert _status() == 1 << 29
        _lib.check(_lib.lib().xnq_init(0))
        want, _, tol = _reference(k[:, :, 32:], v[:, :, 32:], q, [L - 32 - S, -S])
        if S == 1:
            _check(got[:1], want[:1], tol, "no page")
        else:                                                 # queries before position 32 see nothing
            _check(got[:1, S - 32:], want[:1, S - 32:], tol, "no page")
            assert not got[0, :S - 32].any()


def test_calls_of_any_shape_share_a_workspace():
    """A call with few rows writes its parts where a call with many rows must not look for its tickets."""
    B, KV, hd, L = 1, 8, 128, 4096
    c = _filled("q4_0", B, KV, L, hd)
    few, many = (_rand(S, B, S, 32, hd).to(DEV) for S in (1, 300))
    first = _pos(L - 1), _pos(L - 300)
    want = [c.attend(q, p) for q, p in zip((many, few), first[::-1])]
    for _ in range(3):
        assert torch.equal(c.attend(few, first[0]), want[1]) and torch.equal(c.attend(many, first[1]), want[0])


def test_strided_queries_results_and_graphs():
    B, S, H, KV, hd, L = 2, 3, 8, 2, 128, 104
    c = _filled("q4_0", B, KV, L, hd)
    q = _rand(1, B, H, S, hd).to(torch.bfloat16).to(DEV).transpose(1, 2)
    pos = _pos(20, 97)
    want = c.attend(q.contiguous(), pos)
    out = torch.full((B, H, S, hd + 8), 5.0, dtype=torch.bfloat16, device=DEV)
    res = c.attend(q, pos, out=out[..., :hd].transpose(1, 2))
    assert torch.equal(res, want) and bool((out[..., hd:] == 5).all())
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(B, S, H, hd).copy_(q)
    assert torch.equal(c.attend(odd, pos), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = c.attend(q, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    kn, vn = (_rand(i, B, 1, KV, hd).to(DEV) for i in (4, 5))
    at = _pos(20, 97)
    with torch.cuda.graph(graph):
        c.store(kn, vn, at)
        captured = c.attend(q, at)
        at += 1
    for step in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, c.attend(q, _pos(20 + step, 97 + step)))
    assert int(at[0]) == 22


def test_refusals():
    from xn_b200 import _lib
    from xn_b200.dtypes import GgmlDType as D
    from xn_b200.kv_cache import QuantizedKVCache
    for args in [(D.Q4K, 1, 1, 32, 64), (D.Q4_0, 1, 1, 32, 96), (D.Q4_0, 0, 1, 32, 64), (D.Q8_0, 1, 0, 32, 64), (D.Q8_0, 1, 1, 0, 64)]:
        with pytest.raises(ValueError):
            QuantizedKVCache(*args, DEV)
    with pytest.raises(ValueError):
        QuantizedKVCache(D.Q4_0, 1, 1, 64, 64, DEV, page_size=48, num_pages=2)
    with pytest.raises(ValueError):
        QuantizedKVCache(D.Q4_0, 1, 1, 64, 64, DEV, page_size=32)
    c = _cache("q4_0", 2, 2, 64, 64)
    x = torch.zeros(2, 1, 2, 64, device=DEV)
    pos = _pos(0, 0)
    for k, v, p in [(x[:1], x[:1], pos), (x[:, :, :1], x[:, :, :1], pos), (x, x[..., :32], pos), (x, x.half(), pos), (x.double(), x.double(), pos), (x.cpu(), x.cpu(), pos),
                    (x, x, pos.int()), (x, x, _pos(0, 0, 0)), (x, x, pos.cpu())]:
        with pytest.raises(ValueError):
            c.store(k, v, p)
    q = torch.zeros(2, 1, 4, 64, device=DEV)
    for kw in [dict(q=q[:, :, :3]), dict(q=q[..., :32]), dict(window=-1), dict(out=q.half()), dict(out=q[:, :, :1].expand(2, 1, 4, 64)), dict(lse=torch.zeros(2, 1, 2, device=DEV)),
               dict(q=q.double()), dict(pos=pos.int())]:
        with pytest.raises(ValueError):
            c.attend(**{"q": q, "pos": pos, **kw})
    with pytest.raises(_lib.XnqError):
        c.attend(q, pos, scale=math.nan)
    with pytest.raises(ValueError):
        c.rope_store(torch.zeros(2, 1, 7 * 64, device=DEV), torch.zeros(64, 32, device=DEV), torch.zeros(64, 32, device=DEV), pos, 4)
    with pytest.raises(ValueError):
        c.rope_store(torch.zeros(2, 1, 8 * 64, device=DEV), torch.zeros(64, 64, device=DEV), torch.zeros(64, 64, device=DEV), pos, 4)
    with pytest.raises(_lib.XnqError):
        c.load(60, 5)
    with pytest.raises(_lib.XnqError):
        c.load(-1, 2)
    assert c.attend(q[:, :0], pos).shape == (2, 0, 4, 64) and c.load(0, 0)[0].shape == (2, 2, 0, 64)
    assert _status() == 0
