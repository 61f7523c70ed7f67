"""The paged cache's checks of arguments on the CPU, beside test_paged_abi.py: what the documentation allows is not refused. Every call
here ends before anything is enqueued."""
from dooms_amd import _lib
from test_paged_abi import decode, desc, prefill


def test_strides_along_one_page_or_head_are_not_checked():
    for kw in (dict(n_head_kv=1, head_stride=1, kv_stride=128, page_stride=16 * 128), dict(n_pages=1, page_stride=3),
               dict(n_head_kv=1, head_stride=0, kv_stride=128, page_stride=16 * 128)):
        d = desc(max_pages=1000, table_stride=1000, **kw)
        assert decode(d) == _lib.RESOURCE_EXHAUSTED, _lib.last_error()
        assert prefill(d) == _lib.RESOURCE_EXHAUSTED, _lib.last_error()
    assert decode(desc(kv_stride=252)) == _lib.INVALID_ARGUMENT and "kv_stride" in _lib.last_error()
