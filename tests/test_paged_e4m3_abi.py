"""The paged cache's calls in 8 bits on the CPU: layout, refusals of the C ABI and of the front end. Every call here is refused, or has
nothing to do, before anything is enqueued."""
import ctypes
import os
import subprocess
import types

import pytest
import torch

from dooms_amd import _lib
from dooms_amd import attention as A
from test_paged_abi import P, ROOT, desc, rope


def scales(**kw):
    base = dict(k=P, v=P, page_stride=32, head_stride=16, reserved=0)
    base.update(kw)
    return _lib.MxPagedScales(**base)


def store(d, s=None, r=None, qkv=P, positions=0, k=P, v=P, table=P, kv_len=P, cu_q=0, q=P):
    return _lib.paged_store_raw(d, r or rope(), qkv, positions, k, v, table, kv_len, cu_q, q, 0, s or scales())


def decode(d, s=None, q=P, k=P, v=P, table=P, kv_len=P, out=P, lse=0, ws=P, ws_bytes=0):
    return _lib.paged_decode_raw(d, q, k, v, table, kv_len, out, lse, ws, ws_bytes, 0, s or scales())


def prefill(d, s=None, q=P, k=P, v=P, table=P, kv_len=P, cu_q=P, out=P, lse=0, ws=P, ws_bytes=0):
    return _lib.paged_prefill_raw(d, q, k, v, table, kv_len, cu_q, out, lse, ws, ws_bytes, 0, s or scales())


CALLS = (store, decode, prefill)


def test_layout_matches_c(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mx_paged.h"\n'
                   'int main(void){printf("%zu %zu %zu %zu\\n", sizeof(mx_paged_scales), offsetof(mx_paged_scales, page_stride),'
                   ' offsetof(mx_paged_scales, head_stride), offsetof(mx_paged_scales, reserved)); return 0;}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    S = _lib.MxPagedScales
    assert got == [ctypes.sizeof(S), S.page_stride.offset, S.head_stride.offset, S.reserved.offset]


@pytest.mark.parametrize("code,word,kw", [
    (_lib.INVALID_ARGUMENT, "reserved", dict(reserved=1)),
    (_lib.INVALID_ARGUMENT, "scales->page_stride", dict(page_stride=-16)),
    (_lib.INVALID_ARGUMENT, "scales->page_stride", dict(page_stride=40)),
    (_lib.INVALID_ARGUMENT, "scales->head_stride", dict(head_stride=8)),
    (_lib.INVALID_ARGUMENT, "overlap", dict(page_stride=16)),
    (_lib.INVALID_ARGUMENT, "overlap", dict(head_stride=0)),
    (_lib.INVALID_ARGUMENT, "aligned", dict(k=0)),
    (_lib.INVALID_ARGUMENT, "aligned", dict(v=0)),
    (_lib.INVALID_ARGUMENT, "aligned", dict(k=P + 8)),
    (_lib.INVALID_ARGUMENT, "aligned", dict(v=P + 1)),
])
def test_scales_are_refused(code, word, kw):
    for call in CALLS:
        assert call(desc(), scales(**kw)) == code, call.__name__
        assert word in _lib.last_error(), (call.__name__, _lib.last_error())


def test_null_scales_are_refused():
    L, d, r = _lib.lib(), ctypes.byref(desc()), ctypes.byref(rope())
    assert L.mx_paged_store_e4m3(d, r, None, P, None, P, P, P, P, None, P, None) == _lib.INVALID_ARGUMENT and "scales" in _lib.last_error()
    assert L.mx_paged_decode_e4m3(d, None, P, P, P, P, P, P, None, None, 0, None) == _lib.INVALID_ARGUMENT and "scales" in _lib.last_error()
    assert L.mx_paged_prefill_e4m3(d, None, P, P, P, P, P, P, P, None, None, 0, None) == _lib.INVALID_ARGUMENT and "scales" in _lib.last_error()
    assert L.mx_paged_decode_e4m3(None, ctypes.byref(scales()), P, P, P, P, P, P, None, None, 0, None) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("code,word,kw", [
    (_lib.INVALID_ARGUMENT, "dtype", dict(dtype=_lib.DTYPE_F32)),
    (_lib.UNSUPPORTED, "head_dim 96", dict(head_dim=96)),
    (_lib.INVALID_ARGUMENT, "kv_stride", dict(kv_stride=264)),  # a multiple of 8, not of 16
    (_lib.INVALID_ARGUMENT, "head_stride", dict(head_stride=136)),
    (_lib.INVALID_ARGUMENT, "page_stride", dict(page_stride=16 * 256 + 8)),
    (_lib.INVALID_ARGUMENT, "overlap", dict(head_stride=64)),
    (_lib.UNSUPPORTED, "page_size (8)", dict(page_size=8)),
    (_lib.INVALID_ARGUMENT, "table_stride", dict(table_stride=3)),
])
def test_descriptor_is_refused(code, word, kw):
    for call in CALLS:
        assert call(desc(**kw)) == code, call.__name__
        assert word in _lib.last_error(), (call.__name__, _lib.last_error())


def test_nothing_to_do_and_workspaces():
    for call in CALLS:
        assert call(desc(n_rows=0), scales(k=0, v=0)) == _lib.OK
        assert call(desc(n_seq=0, n_rows=0), scales(k=0, v=0)) == _lib.OK
        for name in ("k", "v", "table", "kv_len"):
            assert call(desc(), **{name: 0}) == _lib.INVALID_ARGUMENT and name in _lib.last_error()
    d = desc(max_pages=1000, table_stride=1000)
    assert decode(d, ws_bytes=_lib.paged_decode_workspace_bytes(d) - 1) == _lib.RESOURCE_EXHAUSTED
    assert prefill(d, ws_bytes=_lib.paged_prefill_workspace_bytes(d) - 1) == _lib.RESOURCE_EXHAUSTED
    lone = dict(n_head_kv=1, head_stride=1, kv_stride=128, page_stride=16 * 128)  # strides along one page or head are not looked at
    assert decode(desc(max_pages=1000, table_stride=1000, **lone), scales(head_stride=1, page_stride=16)) == _lib.RESOURCE_EXHAUSTED


def test_front_end_refusals(monkeypatch):
    """On the CPU: the checks in front of the device's, with tensors that say they are on one."""
    monkeypatch.setattr(A, "_native", lambda: A._General())
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc = [torch.zeros(4, 2, 16, dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2)]
    assert A._paged_scales(None, pages.to(torch.float16)) is None
    s = A._paged_scales(sc, pages)
    assert (s.k, s.v, s.page_stride, s.head_stride) == (sc[0].data_ptr(), sc[1].data_ptr(), 32, 16)
    with pytest.raises(ValueError, match="belong"):
        A._paged_scales(sc, pages.to(torch.float16))
    wrong = torch.zeros(4, 16, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    strided = torch.zeros(8, 2, 16, dtype=torch.uint8).view(torch.float8_e8m0fnu)[::2]
    for bad, word in ((None, "need scales"), ([sc[0]], "need scales"), ([sc[0], sc[1].view(torch.uint8)], "float8_e8m0fnu"),
                      ([wrong, wrong], "kv heads"), ([sc[0], wrong.transpose(1, 2)], "unit stride"), ([sc[0], strided], "strides")):
        with pytest.raises(ValueError, match=word):
            A._paged_scales(bad, pages)
    table, kv_len = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        A.paged_decode(torch.zeros(1, 4 * 64), pages, pages, table, kv_len, n_head=4, scales=sc)
    with pytest.raises(ValueError, match="device tensor"):
        A.paged_decode(torch.zeros(1, 4 * 64).half(), pages, pages, table, kv_len, n_head=4, scales=sc)
    with pytest.raises(ValueError, match="device tensor"):
        A.paged_store(torch.zeros(1, 8 * 64), pages, pages, table, kv_len, n_head=4, rope_mode=0, scales=sc)


def test_other_extensions_are_refused(monkeypatch):
    from dooms_amd import _native as ext
    version = _lib.lib().mx_attn_abi_version()
    sizes = ctypes.sizeof(_lib.MxPagedScales), ctypes.sizeof(_lib.MxPagedPrefix)
    for v, s in ((version + 1, sizes), (version, (sizes[0] + 8, sizes[1])), (version, (sizes[0], sizes[1] + 8))):
        with pytest.raises(ImportError, match="dooms_amd.build"):
            ext.bind_paged_more(v, s, 0, 0, 0, 0)
    old = types.SimpleNamespace(bind=lambda *a: None, bind_paged=lambda *a: None)
    monkeypatch.setattr(A, "_bound", None)
    monkeypatch.setattr(A, "_ext", None)
    monkeypatch.setattr(A.importlib, "import_module", lambda *a: old)
    with pytest.raises(ImportError, match="dooms_amd.build"):
        A._native()
    assert A._bound is None
