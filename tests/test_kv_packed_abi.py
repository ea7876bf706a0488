"""What the entries for page tables, packed tokens and trees refuse, before anything reaches a device."""
import ctypes

import pytest

from test_kv_cache_abi import ALIGN, DTYPE, NULL, P, SHAPE, SIZE, UNSUPPORTED, _cache, _rows
from xn_b200 import _lib
from xn_b200.kv_cache import TREE_MOST, _Plan, _Rope

b = ctypes.byref


def _plan(**kw):
    return _Plan(**{**dict(tokens=10, batch=2, longest=6, start=P, offsets=P, sequence=P, position=P, slot=P, sees=None, nodes=None), **kw})


def _tree(**kw):
    return _plan(**{**dict(sees=P, nodes=P), **kw})


@pytest.mark.parametrize("plan,code", [(None, NULL), (_plan(start=None), NULL), (_plan(offsets=None), NULL), (_plan(sequence=None), NULL), (_plan(position=None), NULL), (_plan(slot=None), NULL),
                                       (_plan(sees=P), NULL), (_plan(nodes=P), NULL), (_plan(tokens=-1), SHAPE), (_plan(tokens=1 << 31), SHAPE), (_plan(batch=0), SHAPE), (_plan(batch=1 << 20), SHAPE),
                                       (_plan(longest=0), SHAPE), (_tree(longest=TREE_MOST + 1), UNSUPPORTED)])
def test_plans_that_are_refused(plan, code):
    L, c, r = _lib.lib(), _cache(), _rows()
    p = None if plan is None else b(plan)
    assert L.xnq_kv_plan_make(b(c), P, 1, P, P if plan is not None and plan.sees else None, p, None) == code
    assert L.xnq_kv_store_packed(b(c), b(r), b(r), p, None, None) == code
    assert L.xnq_kv_keep(b(c), p, P, P, None) == code
    if plan is not None:
        assert L.xnq_kv_attend_packed(b(c), b(r), b(r), None, 0, 0, 4, None, 0, p, 0, 1.0, 1, 0, 0, P, 1 << 40, None) == code


def test_arguments_that_are_refused():
    L, c, r = _lib.lib(), _cache(), _rows()
    assert L.xnq_kv_plan_make(b(c), None, 1, P, None, b(_plan()), None) == NULL and L.xnq_kv_plan_make(b(c), P, 1, None, None, b(_plan()), None) == NULL
    assert L.xnq_kv_plan_make(b(c), P, 2, P, None, b(_plan()), None) == SHAPE
    assert L.xnq_kv_plan_make(b(c), P, 1, P, P, b(_plan()), None) == NULL and L.xnq_kv_plan_make(b(c), P, 1, P, None, b(_tree()), None) == NULL
    assert L.xnq_kv_plan_make(b(_cache(head_dim=80)), P, 1, P, None, b(_plan()), None) == UNSUPPORTED
    assert L.xnq_kv_plan_make(b(c), P, 1, P, None, b(_plan(batch=5)), None) == SIZE   # more sequences than the cache has pages
    assert L.xnq_kv_store_packed(b(c), None, b(r), b(_plan()), None, None) == NULL
    assert L.xnq_kv_store_packed(b(c), b(r), b(_rows(dtype=1)), b(_plan()), None, None) == DTYPE
    assert L.xnq_kv_store_packed(b(c), b(_rows(data=P + 4)), b(r), b(_plan()), None, None) == ALIGN
    rope = dict(cos_table=P, sin_table=P, table_rows=8, heads=4, q=_rows(), q_out=_rows())
    assert L.xnq_kv_store_packed(b(c), b(r), b(r), b(_plan()), b(_Rope(**{**rope, "cos_table": None})), None) == NULL
    assert L.xnq_kv_store_packed(b(c), b(r), b(r), b(_plan()), b(_Rope(**{**rope, "table_rows": 0})), None) == SHAPE
    assert L.xnq_kv_keep(b(c), b(_plan()), P, P, None) == NULL and L.xnq_kv_keep(b(c), b(_tree()), None, P, None) == NULL and L.xnq_kv_keep(b(c), b(_tree()), P, None, None) == NULL
    ok = [b(c), b(r), b(r), None, 2, 1, 4, P, 1, None, 0, 1.0, 1, 8, 4, P, 1 << 40, None]
    for i, value, code in [(0, None, NULL), (1, None, NULL), (2, b(_rows(dtype=1)), DTYPE), (5, -1, SHAPE), (6, 3, SHAPE), (7, None, NULL), (8, 3, SHAPE), (11, float("nan"), SHAPE), (13, -1, SHAPE),
                           (14, -1, SHAPE), (15, None, SIZE), (16, 0, SIZE), (15, P + 8, ALIGN)]:
        args = list(ok)
        args[i] = value
        assert L.xnq_kv_attend_packed(*args) == code, (i, value)
    ok[9] = b(_tree())
    ok[13] = 5   # shorter than the trees
    assert L.xnq_kv_attend_packed(*ok) == SHAPE
    ok[13], ok[16] = 6, L.xnq_kv_attend_packed_workspace_bytes(b(_tree()), 4, 2, 128) - 1
    assert L.xnq_kv_attend_packed(*ok) == SIZE


def test_page_tables_that_are_refused():
    L = _lib.lib()
    ok = dict(table=P, table_stride=4, source=P, from_stride=4, batch=2, page_size=32, num_pages=9, max_seq=128, length=P, first=None, sinks=0, room=P, free=P, workspace=P, ws=1 << 30, stream=None)
    for kw, code in [(dict(table=None), NULL), (dict(source=None), NULL), (dict(length=None), NULL), (dict(room=None), NULL), (dict(free=None), NULL), (dict(batch=-1), SHAPE), (dict(page_size=40), SHAPE),
                     (dict(page_size=0), SHAPE), (dict(num_pages=0), SHAPE), (dict(max_seq=0), SHAPE), (dict(sinks=-1), SHAPE), (dict(num_pages=(1 << 20) + 1), UNSUPPORTED), (dict(table_stride=3), SIZE),
                     (dict(from_stride=3), SIZE), (dict(batch=1 << 30), SIZE), (dict(workspace=None), SIZE), (dict(ws=0), SIZE), (dict(workspace=P + 4), ALIGN)]:
        assert L.xnq_kv_reserve(*{**ok, **kw}.values()) == code, kw
    assert L.xnq_kv_reserve_workspace_bytes(2, 32, 0, 128) == 0 and L.xnq_kv_reserve_workspace_bytes(2, 32, (1 << 20) + 1, 128) == 0
    assert L.xnq_kv_reserve_workspace_bytes(500, 64, 400000, 131072) >= 400000 / 8 + 500


def test_workspaces_of_packed_tokens():
    L = _lib.lib()
    assert L.xnq_kv_attend_packed_workspace_bytes(None, 4, 2, 128) == 0 and L.xnq_kv_attend_packed_workspace_bytes(b(_plan()), 3, 2, 128) == 0
    few, many = (L.xnq_kv_attend_packed_workspace_bytes(b(_plan(longest=n)), 8, 2, 128) for n in (15, 16))
    assert few == L.xnq_kv_attend_workspace_bytes(2, 15, 8, 2, 128) and many > few
