"""Paged KV cache, host side, at the edges: strides that the C entry points
refuse, and the workspace query (no GPU is touched)."""
import ctypes

from tests import abi_ctypes as abi
from tests.test_paged_cpu import P16, _attend, _cache, _read, _write

STRIDE = 15


def test_unusable_strides_are_refused():
    # the rows of a page, and anything walked backwards
    for call in (_write, _read, _attend):
        for kw in (dict(row_stride=0), dict(row_stride=-64), dict(head_stride=-1024), dict(page_stride=-2048)):
            assert call(_cache(**kw)) == STRIDE
    # one head or page seen as several: for reading alone (total = 0: nothing more to do)
    for kw in (dict(head_stride=0), dict(page_stride=0)):
        assert _write(_cache(**kw)) == STRIDE
        assert _read(_cache(**kw), total=0) == 0
        assert _attend(_cache(**kw), total=0) == 0
    # the stride of a dimension with one entry is not used
    assert _read(_cache(kv_heads=1, head_stride=0, num_pages=1, page_stride=-8), total=0) == 0
    assert _write(_cache(kv_heads=1, head_stride=0, num_pages=1, page_stride=-8), total=0) == 0
    # scales that several entries share cannot be written
    eight = dict(dtype=2, k_scale=P16, v_scale=P16, scale_page_stride=32, scale_head_stride=16, scale_row_stride=1)
    assert _write(_cache(**eight), total=0) == 0
    for name in ("scale_page_stride", "scale_head_stride", "scale_row_stride"):
        assert _write(_cache(**{**eight, name: 0})) == STRIDE
        assert _read(_cache(**{**eight, name: 0}), total=0) == 0
    # queries
    f = abi.load().fa_fwd_paged

    def attend(qt, qh, Hq=4, total=3):
        return f(ctypes.byref(_cache()), P16, qt, qh, P16, None, P16, P16, 1, Hq, total, 3, 64, 1.0, 1, 0, P16,
                 0, None)

    assert attend(256, 0) == STRIDE and attend(0, 64) == STRIDE and attend(-256, 64) == STRIDE
    assert abi.load().fa_error_string(STRIDE) not in (b"ok", b"unknown error")


def test_workspace_query_answers_0_for_what_the_call_refuses():
    f = abi.load().fa_fwd_paged_workspace_bytes
    eight = dict(k_scale=P16, v_scale=P16)
    for kw in (dict(head_dim=0), dict(head_dim=96), dict(head_dim=8192), dict(head_dim=-64), dict(dtype=-1),
               dict(dtype=4, **eight), dict(kv_heads=3), dict(kv_heads=1 << 20)):
        for args in ((1, 4, 1, 1, 8192), (8, 4, 8, 1, 1 << 20), (1, 4, 99, 99, 64)):
            assert f(ctypes.byref(_cache(**kw)), *args) == 0, (kw, args)
    assert f(ctypes.byref(abi.PagedCache(kv_heads=1)), 1, 4, 9, 9, 64) == 0  # all else zero
    assert f(ctypes.byref(_cache()), 1 << 21, 4, 9, 9, 64) == 0
    assert f(ctypes.byref(_cache()), 1, 4, 1 << 29, 9, 64) == 0
