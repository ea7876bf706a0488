"""Attention of many rows: a CTA that ends has none of its copies in flight. Nothing here needs a device.

A wait for a barrier's phase by its parity is over when the phase of that parity lies behind, so one of the two parities always reads as over: what ends a
CTA has to ask for the parity of the last copy into each slot. The expression is read from the source and tried against a model of the barriers.
"""
import os
import re

import pytest

SOURCE = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xn_b200", "csrc", "xnq_kv_prompt.cu")).read()


def _waited_for(issued, slots):
    """{slot: parity} that the loader waits for at its end."""
    loop = re.search(r"for \(int slot = 0; slot < P::SLOTS && slot < i; slot\+\+\) \{\s*const uint32_t parity = \(uint32_t\)\((.+?)\) & 1u;\s*"
                     r"for \(int k = 0; k < \d+ && !mbar_try\(raw_full \+ 8 \* slot, parity\); k\+\+\) \{\}", SOURCE)
    assert loop, "the loader's last waits"
    lap = loop.group(1).replace("P::SLOTS", "slots").replace("/", "//")
    return {slot: eval(lap, {"i": issued, "slot": slot, "slots": slots}) & 1 for slot in range(min(slots, issued))}   # noqa: S307 (an expression of three whole numbers)


@pytest.mark.parametrize("slots", [4, 7, 15, 16])
def test_the_last_copy_into_each_slot_is_waited_for(slots):
    for issued in range(0, 5 * slots + 3):
        begun = [len(range(s, issued, slots)) for s in range(slots)]          # copies into a slot: phases 0 .. begun - 1
        parity = _waited_for(issued, slots)
        assert set(parity) == {s for s in range(slots) if begun[s]}
        for s, p in parity.items():
            over = lambda done: (done - 1) & 1 == p                            # `done` phases are complete: the one behind has parity (done - 1) & 1
            assert over(begun[s]) and not over(begun[s] - 1)                   # all landed; the last one in flight


def test_what_gives_up_waits_for_its_products():
    role = SOURCE[SOURCE.index("warp >= MMA && warp < MMA + QT"):SOURCE.index("// ---- a row a thread ----")]
    assert re.search(r"if \(!alive && halves > 0\) \{[^}]*commit\(o_done \+ 8 \* q\);[^}]*mbar_try\(o_done \+ 8 \* q, 0\)", role)
