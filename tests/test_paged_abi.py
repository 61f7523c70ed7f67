"""The paged cache's C ABI (include/mx_paged.h) on the CPU: layouts, refusals, workspace sizes. Every call here is refused, or has
nothing to do, before anything is enqueued."""
import ctypes
import os
import subprocess

import pytest
import torch

from dooms_amd import _lib
from dooms_amd import attention as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096  # an aligned fake device address, never dereferenced


def test_layouts_match_c(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mx_paged.h"\n'
                   'int main(void){printf("%zu %zu %zu %zu %zu %zu %d\\n", sizeof(mx_paged_desc), offsetof(mx_paged_desc, reserved),'
                   ' offsetof(mx_paged_desc, page_stride), offsetof(mx_paged_desc, scale), sizeof(mx_paged_rope),'
                   ' offsetof(mx_paged_rope, base), MX_PAGED_MAX_AXES); return 0;}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    D, R = _lib.MxPagedDesc, _lib.MxPagedRope
    assert got == [ctypes.sizeof(D), D.reserved.offset, D.page_stride.offset, D.scale.offset, ctypes.sizeof(R), R.base.offset,
                   _lib.PAGED_MAX_AXES]


def desc(**kw):
    base = dict(n_head=8, n_head_kv=2, head_dim=128, dtype=_lib.DTYPE_F16, row_dtype=_lib.DTYPE_F16, n_seq=3, n_rows=3, causal=1,
                page_size=16, n_pages=10, max_pages=4, max_q=0, max_kv_len=0, page_stride=16 * 256, kv_stride=256, head_stride=128,
                table_stride=4, row_stride=1536, out_stride=1024, scale=0.1)
    base.update(kw)
    return _lib.MxPagedDesc(**base)


def rope(**kw):
    base = dict(mode=1, n_axes=1, axis_pairs=(64,), axis_restart=0, base=1e4, reserved=0)
    base.update(kw)
    base["axis_pairs"] = (ctypes.c_int32 * 4)(*base["axis_pairs"])
    return _lib.MxPagedRope(**base)


def store(d, r=None, qkv=P, positions=0, k=P, v=P, table=P, kv_len=P, cu_q=0, q=P):
    return _lib.paged_store_raw(d, r or rope(), qkv, positions, k, v, table, kv_len, cu_q, q, 0)


def decode(d, q=P, k=P, v=P, table=P, kv_len=P, out=P, lse=0, ws=P, ws_bytes=0):
    return _lib.paged_decode_raw(d, q, k, v, table, kv_len, out, lse, ws, ws_bytes, 0)


def prefill(d, q=P, k=P, v=P, table=P, kv_len=P, cu_q=P, out=P, lse=0, ws=P, ws_bytes=0):
    return _lib.paged_prefill_raw(d, q, k, v, table, kv_len, cu_q, out, lse, ws, ws_bytes, 0)


@pytest.mark.parametrize("code,word,kw", [
    (_lib.INVALID_ARGUMENT, "reserved", dict(reserved=1)),
    (_lib.INVALID_ARGUMENT, "n_head", dict(n_head=0)),
    (_lib.INVALID_ARGUMENT, "multiple of n_head_kv", dict(n_head=7)),
    (_lib.UNSUPPORTED, "head_dim 32", dict(head_dim=32)),
    (_lib.UNSUPPORTED, "head_dim 96", dict(head_dim=96)),
    (_lib.INVALID_ARGUMENT, "dtype", dict(dtype=_lib.DTYPE_F32)),
    (_lib.INVALID_ARGUMENT, "row_dtype", dict(row_dtype=7)),
    (_lib.INVALID_ARGUMENT, "n_seq", dict(n_seq=-1)),
    (_lib.INVALID_ARGUMENT, "n_seq", dict(n_seq=65536, n_rows=65536)),
    (_lib.INVALID_ARGUMENT, "n_rows", dict(n_rows=-3)),
    (_lib.INVALID_ARGUMENT, "max_q", dict(max_q=-1)),
    (_lib.INVALID_ARGUMENT, "max_kv_len", dict(max_kv_len=-1)),
    (_lib.UNSUPPORTED, "page_size (8)", dict(page_size=8)),
    (_lib.UNSUPPORTED, "page_size (48)", dict(page_size=48)),
    (_lib.UNSUPPORTED, "page_size", dict(page_size=131072)),
    (_lib.INVALID_ARGUMENT, "n_pages", dict(n_pages=0)),
    (_lib.INVALID_ARGUMENT, "max_pages", dict(max_pages=0)),
    (_lib.UNSUPPORTED, "2^30", dict(page_size=65536, max_pages=1 << 15, table_stride=1 << 15, page_stride=65536 * 256)),
    (_lib.INVALID_ARGUMENT, "table_stride", dict(table_stride=3)),
    (_lib.INVALID_ARGUMENT, "page_stride", dict(page_stride=-8)),
    (_lib.INVALID_ARGUMENT, "kv_stride", dict(kv_stride=252)),
    (_lib.INVALID_ARGUMENT, "overlap", dict(kv_stride=0)),
    (_lib.INVALID_ARGUMENT, "overlap", dict(head_stride=64)),
    (_lib.INVALID_ARGUMENT, "overlap", dict(page_stride=15 * 256)),
    (_lib.UNSUPPORTED, "2^26", dict(kv_stride=1 << 27, page_stride=1 << 32)),
    (_lib.INVALID_ARGUMENT, "row_stride", dict(row_stride=1000)),
    (_lib.INVALID_ARGUMENT, "row_stride", dict(row_stride=1537)),
    (_lib.INVALID_ARGUMENT, "out_stride", dict(out_stride=1016)),
    (_lib.INVALID_ARGUMENT, "out_stride", dict(out_stride=1028)),
])
def test_descriptor_is_refused(code, word, kw):
    for call in (store, decode, prefill):
        assert call(desc(**kw)) == code, call.__name__
        assert word in _lib.last_error(), (call.__name__, _lib.last_error())


def test_attention_refusals():
    for call in (decode, prefill):
        assert call(desc(row_dtype=_lib.DTYPE_BF16)) == _lib.INVALID_ARGUMENT and "row_dtype" in _lib.last_error()
        assert call(desc(causal=2)) == _lib.INVALID_ARGUMENT and "causal" in _lib.last_error()
        for s in (float("inf"), float("nan")):
            assert call(desc(scale=s)) == _lib.INVALID_ARGUMENT and "scale" in _lib.last_error()
        for name in ("q", "out", "k", "v", "table", "kv_len"):
            assert call(desc(), **{name: 0}) == _lib.INVALID_ARGUMENT and name in _lib.last_error()
        for name in ("q", "out", "k", "v"):
            assert call(desc(), **{name: P + 8}) == _lib.INVALID_ARGUMENT and "aligned" in _lib.last_error()
        for name in ("table", "kv_len", "lse"):
            assert call(desc(), **{name: P + 2}) == _lib.INVALID_ARGUMENT and "aligned" in _lib.last_error()
        assert call(desc(n_rows=0), q=0, out=0) == _lib.OK
        assert call(desc(n_seq=0, n_rows=0), q=0, out=0, table=0, kv_len=0) == _lib.OK
    assert prefill(desc(), cu_q=0) == _lib.INVALID_ARGUMENT and "cu_q" in _lib.last_error()
    assert decode(desc(n_rows=4)) == _lib.INVALID_ARGUMENT and "multiple of n_seq" in _lib.last_error()
    assert decode(desc(n_seq=0)) == _lib.INVALID_ARGUMENT and "no sequence" in _lib.last_error()
    assert decode(desc(n_rows=3 * 20000)) == _lib.UNSUPPORTED and "mx_paged_prefill" in _lib.last_error()
    wide = dict(n_seq=65535, max_pages=1 << 20, table_stride=1 << 20, page_size=1024, page_stride=1024 * 256)
    assert decode(desc(n_rows=65535, **wide)) == _lib.UNSUPPORTED and "more than one launch" in _lib.last_error()
    assert decode(desc(n_head=4096, n_head_kv=4096, row_stride=3 * 4096 * 128, out_stride=4096 * 128, kv_stride=4096 * 128,
                       page_stride=16 * 4096 * 128)) == _lib.UNSUPPORTED and "row tile" in _lib.last_error()
    assert prefill(desc(), ws=P + 16, ws_bytes=1 << 30) == _lib.INVALID_ARGUMENT and "256-byte" in _lib.last_error()
    assert prefill(desc(), ws_bytes=1 << 20) == _lib.RESOURCE_EXHAUSTED
    assert prefill(desc(n_rows=1 << 28, **wide)) == _lib.UNSUPPORTED and "more than one launch" in _lib.last_error()
    for call in (decode, prefill):
        assert call(desc(n_rows=(1 << 30) + 3)) == _lib.INVALID_ARGUMENT and "n_rows" in _lib.last_error()


def test_decode_workspace():
    d = desc(max_pages=1000, table_stride=1000)
    need = _lib.paged_decode_workspace_bytes(d)
    assert need > 0
    assert decode(d, ws=0, ws_bytes=need) == _lib.INVALID_ARGUMENT and "workspace" in _lib.last_error()
    assert decode(d, ws=P + 16, ws_bytes=need) == _lib.INVALID_ARGUMENT and "256-byte" in _lib.last_error()
    assert decode(d, ws_bytes=need - 1) == _lib.RESOURCE_EXHAUSTED
    assert _lib.paged_decode_workspace_bytes(desc(max_pages=1000, max_kv_len=100)) == 0  # one split
    assert _lib.paged_decode_workspace_bytes(desc(head_dim=96)) == 0 and "head_dim" in _lib.last_error()
    assert _lib.lib().mx_paged_decode_workspace_bytes(None) == 0
    assert _lib.lib().mx_paged_prefill_workspace_bytes(None) == 0


@pytest.mark.parametrize("n_head,n_kv,hd", [(14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 256)])
def test_decode_workspace_sized_once(n_head, n_kv, hd):
    """A workspace for the most and longest sequences serves fewer and shorter ones."""
    for n_q in (1, 4):
        below = {}
        for n_seq in (1, 3, 16, 64, 300):
            most = 0
            for length in [1, 100, 129, 257, 300, 511, 512, 513, 1000, 2000, 4096, 8192, 30000, 131072]:
                b = A.paged_decode_workspace_bytes(n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_q=n_q, n_seq=n_seq, max_kv_len=length)
                assert b >= most and b >= below.get(length, 0), (n_seq, n_q, length)
                most = below[length] = b


@pytest.mark.parametrize("word,kw", [
    ("reserved", dict(reserved=1)), ("mode", dict(mode=3)), ("mode", dict(mode=-1)), ("n_axes", dict(n_axes=0)), ("n_axes", dict(n_axes=5)),
    ("axis_restart", dict(axis_restart=2)), ("base", dict(base=0.0)), ("base", dict(base=float("nan"))), ("base", dict(base=-2.0)),
    ("base", dict(base=0.5)),
    ("not head_dim / 2", dict(axis_pairs=(63,))), ("more than head_dim / 2", dict(axis_pairs=(65,))),
    ("axis_pairs[1]", dict(n_axes=2, axis_pairs=(64, 0))), ("axis_pairs[0]", dict(axis_pairs=(-1,))),
    ("positions", dict(n_axes=2, axis_pairs=(32, 32))),
])
def test_rope_is_refused(word, kw):
    assert store(desc(), rope(**kw)) == _lib.INVALID_ARGUMENT and word in _lib.last_error()


def test_store_refusals():
    assert _lib.lib().mx_paged_store(ctypes.byref(desc()), None, P, None, P, P, P, P, None, P, None) == _lib.INVALID_ARGUMENT
    assert "rope" in _lib.last_error()
    assert store(desc(), qkv=0) == _lib.INVALID_ARGUMENT and "qkv" in _lib.last_error()
    assert store(desc(), qkv=P + 8) == _lib.INVALID_ARGUMENT
    assert store(desc(), q=P + 2) == _lib.INVALID_ARGUMENT and "q_out" in _lib.last_error()
    assert store(desc(), positions=P + 2) == _lib.INVALID_ARGUMENT and "positions" in _lib.last_error()
    assert store(desc(n_rows=5)) == _lib.INVALID_ARGUMENT and "multiple of n_seq" in _lib.last_error()
    assert store(desc(n_rows=0), qkv=0) == _lib.OK
    for name in ("k", "v", "table", "kv_len"):
        assert store(desc(), **{name: 0}) == _lib.INVALID_ARGUMENT and name in _lib.last_error()


def test_front_end_refuses_host_tensors():
    k = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    table, kv_len, cu = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(1, 4 * 64, dtype=torch.float16)
    ws = torch.zeros(1024, dtype=torch.uint8)
    with pytest.raises(ValueError, match="device tensor"):
        A.paged_decode(q, k, k, table, kv_len, n_head=4, workspace=ws)
    with pytest.raises(ValueError, match="device tensor"):
        A.paged_prefill(q, k, k, table, kv_len, cu, n_head=4)
    with pytest.raises(ValueError, match="device tensor"):
        A.paged_store(torch.zeros(1, 8 * 64), k, k, table, kv_len, n_head=4, rope_mode=0)


def test_extension_of_other_descriptors_is_refused():
    from dooms_amd import _native as ext
    version = _lib.lib().mx_attn_abi_version()
    sizes = [ctypes.sizeof(_lib.MxPagedDesc), ctypes.sizeof(_lib.MxPagedRope)]
    for v, s in [(version + 1, sizes), (version, [sizes[0] + 8, sizes[1]]), (version, [sizes[0], sizes[1] + 8])]:
        with pytest.raises(ImportError, match="dooms_amd.build"):
            ext.bind_paged(v, tuple(s), 0, 0, 0)
