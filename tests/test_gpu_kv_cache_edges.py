"""The quantized KV cache where it can go wrong between items, warps, halves and calls. Tolerances are those of test_gpu_kv_cache.py."""
import math

import pytest
import torch

from test_gpu_kv_cache import DEV, TYPES, _cache, _check, _filled, _init, _pos, _rand, _reference, _status  # noqa: F401 (_init: the module's fixture)

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
