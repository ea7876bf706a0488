"""What the quantized KV cache's entries refuse, before anything reaches a device."""
import ctypes

import pytest

from xn_b200 import _lib
from xn_b200.dtypes import GgmlDType as D
from xn_b200.kv_cache import _Cache, _Rope, _Rows

P = 4096  # an address that is never read


def _cache(**kw):
    return _Cache(**{**dict(ggml_dtype=int(D.Q4_0), kv_heads=2, head_dim=128, page_size=64, num_pages=4, pages=P, page_table=None, table_stride=0, max_seq=64), **kw})


def _rows(**kw):
    return _Rows(**{**dict(data=P, dtype=0, stride_b=512, stride_s=256, stride_h=128), **kw})


def test_page_bytes():
    L = _lib.lib()
    for dt, hd, row in [(D.Q4_0, 64, 36), (D.Q4_0, 128, 72), (D.Q8_0, 64, 68), (D.Q8_0, 128, 136)]:   # a key's or value's codes and scales
        for kv, page in [(1, 32), (8, 64), (3, 4096)]:
            assert L.xnq_kv_page_bytes(int(dt), kv, hd, page) == 2 * row * kv * page
    for args in [(int(D.Q4K), 1, 128, 32), (int(D.Q4_0), 0, 128, 32), (int(D.Q4_0), 1, 96, 32), (int(D.Q4_0), 1, 128, 33), (int(D.Q4_0), 1, 128, 0)]:
        assert L.xnq_kv_page_bytes(*args) == 0


NULL, DTYPE, SHAPE, ALIGN, SIZE, UNSUPPORTED = -1, -2, -3, -4, -5, -8


@pytest.mark.parametrize("kw,code", [(dict(pages=None), NULL), (dict(ggml_dtype=int(D.Q4K)), DTYPE), (dict(head_dim=80), UNSUPPORTED), (dict(kv_heads=0), SHAPE),
                                     (dict(page_size=40), SHAPE), (dict(max_seq=0), SHAPE), (dict(max_seq=65), SIZE), (dict(num_pages=1), SIZE),
                                     (dict(page_table=P, table_stride=0), SIZE), (dict(pages=P + 8), ALIGN)])
def test_caches_that_are_refused(kw, code):
    L, c, r = _lib.lib(), _cache(**kw), _rows()
    b = ctypes.byref
    assert L.xnq_kv_store(b(c), b(r), b(r), 2, 1, P, 1, None, None) == code
    assert L.xnq_kv_load(b(c), 2, None, 0, 0, 1, 0, P, P, None) == code
    assert L.xnq_kv_attend(b(c), b(r), b(r), None, 2, 1, 4, P, 1, 1.0, 1, 0, P, 1 << 40, None) == code


def test_arguments_that_are_refused():
    L, c, r = _lib.lib(), _cache(), _rows()
    b = ctypes.byref
    assert L.xnq_kv_store(None, b(r), b(r), 2, 1, P, 1, None, None) == NULL
    assert L.xnq_kv_store(b(c), b(r), b(r), 2, 1, None, 1, None, None) == NULL
    assert L.xnq_kv_store(b(c), b(_rows(data=None)), b(r), 2, 1, P, 1, None, None) == NULL
    assert L.xnq_kv_store(b(c), b(_rows(dtype=2)), b(_rows(dtype=2)), 2, 1, P, 1, None, None) == DTYPE
    assert L.xnq_kv_store(b(c), b(r), b(_rows(dtype=1)), 2, 1, P, 1, None, None) == DTYPE
    assert L.xnq_kv_store(b(c), b(r), b(r), -1, 1, P, 1, None, None) == SHAPE
    assert L.xnq_kv_store(b(c), b(r), b(r), 2, -1, P, 1, None, None) == SHAPE
    assert L.xnq_kv_store(b(c), b(r), b(r), 2, 1, P, 2, None, None) == SHAPE
    assert L.xnq_kv_store(b(c), b(_rows(data=P + 4)), b(r), 2, 1, P, 1, None, None) == ALIGN
    assert L.xnq_kv_store(b(c), b(_rows(stride_s=130)), b(r), 2, 1, P, 1, None, None) == ALIGN
    rope = dict(cos_table=P, sin_table=P, table_rows=8, heads=4, q=_rows(), q_out=_rows())
    for kw, code in [(dict(cos_table=None), NULL), (dict(table_rows=0), SHAPE), (dict(heads=-1), SHAPE), (dict(sin_table=P + 4), ALIGN), (dict(q=_rows(dtype=1)), DTYPE),
                     (dict(q_out=_rows(data=None)), NULL)]:
        assert L.xnq_kv_store(b(c), b(r), b(r), 2, 1, P, 1, b(_Rope(**{**rope, **kw})), None) == code, kw
    assert L.xnq_kv_load(b(c), 2, None, 0, 60, 5, 0, P, P, None) == SHAPE
    assert L.xnq_kv_load(b(c), 2, None, 0, 0, 5, 2, P, P, None) == DTYPE
    assert L.xnq_kv_load(b(c), 2, None, 0, 0, 5, 0, P, None, None) == NULL
    ok = [b(c), b(r), b(r), None, 2, 1, 4, P, 1, 1.0, 1, 0, P, 1 << 40, None]
    for i, value, code in [(1, None, NULL), (2, b(_rows(dtype=1)), DTYPE), (5, -1, SHAPE), (6, 3, SHAPE), (7, None, NULL), (8, 3, SHAPE), (9, float("inf"), SHAPE), (11, -1, SHAPE),
                           (12, None, SIZE), (13, 0, SIZE), (12, P + 8, ALIGN)]:
        args = list(ok)
        args[i] = value
        assert L.xnq_kv_attend(*args) == code, (i, value)
    assert L.xnq_kv_attend_workspace_bytes(0, 1, 4, 2, 128) == 0 and L.xnq_kv_attend_workspace_bytes(1, 1, 3, 2, 128) == 0
    assert L.xnq_kv_attend_workspace_bytes(1, 1, 4, 2, 96) == 0 and L.xnq_kv_attend_workspace_bytes(3, 7, 4, 2, 128) >= 16
