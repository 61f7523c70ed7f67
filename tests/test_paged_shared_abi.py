"""mx_paged_decode_shared on the CPU: layout, refusals, workspace sizes. Every call here is refused, or has nothing to do, before anything
is enqueued."""
import ctypes
import os
import subprocess

import pytest
import torch

from dooms_amd import _lib
from dooms_amd import attention as A
from test_paged_abi import P, ROOT, desc
from test_paged_e4m3_abi import scales


def prefix(**kw):
    base = dict(n_groups=2, reserved=0, cu_seq=P, prefix_len=P)
    base.update(kw)
    return _lib.MxPagedPrefix(**base)


def shared(d, x=None, s=None, q=P, k=P, v=P, table=P, kv_len=P, out=P, lse=0, ws=P, ws_bytes=1 << 40):
    return _lib.paged_decode_shared_raw(d, x or prefix(), q, k, v, table, kv_len, out, lse, ws, ws_bytes, 0, s)


def test_layout_matches_c(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mx_paged.h"\n'
                   'int main(void){printf("%zu %zu %zu\\n", sizeof(mx_paged_prefix), offsetof(mx_paged_prefix, cu_seq),'
                   ' offsetof(mx_paged_prefix, prefix_len)); return 0;}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    X = _lib.MxPagedPrefix
    assert got == [ctypes.sizeof(X), X.cu_seq.offset, X.prefix_len.offset]


@pytest.mark.parametrize("s", [None, "scales"])
def test_refusals(s):
    s = s and scales()
    for code, word, kw in ((_lib.INVALID_ARGUMENT, "reserved", dict(reserved=1)), (_lib.INVALID_ARGUMENT, "n_groups", dict(n_groups=-1)),
                           (_lib.INVALID_ARGUMENT, "n_groups", dict(n_groups=65536)), (_lib.INVALID_ARGUMENT, "cu_seq", dict(cu_seq=0)),
                           (_lib.INVALID_ARGUMENT, "prefix_len", dict(prefix_len=0)), (_lib.INVALID_ARGUMENT, "aligned", dict(cu_seq=P + 2))):
        assert shared(desc(), prefix(**kw), s) == code and word in _lib.last_error(), (kw, _lib.last_error())
    for code, word, kw in ((_lib.INVALID_ARGUMENT, "dtype", dict(dtype=_lib.DTYPE_F32)), (_lib.UNSUPPORTED, "head_dim 32", dict(head_dim=32)),
                           (_lib.INVALID_ARGUMENT, "multiple of n_seq", dict(n_rows=4)), (_lib.INVALID_ARGUMENT, "causal", dict(causal=2)),
                           (_lib.INVALID_ARGUMENT, "row_dtype", dict(row_dtype=_lib.DTYPE_BF16)), (_lib.INVALID_ARGUMENT, "kv_stride", dict(kv_stride=252)),
                           (_lib.INVALID_ARGUMENT, "scale", dict(scale=float("nan"))),
                           (_lib.UNSUPPORTED, "more than one launch", dict(n_head=64, n_seq=1, n_rows=1 << 21, row_stride=64 * 128, out_stride=64 * 128))):
        assert shared(desc(**kw), prefix(n_groups=1), s) == code and word in _lib.last_error(), (kw, _lib.last_error())
    for name in ("q", "out", "k", "v", "table", "kv_len"):
        assert shared(desc(), None, s, **{name: 0}) == _lib.INVALID_ARGUMENT and name in _lib.last_error()
    need = _lib.paged_decode_shared_workspace_bytes(desc(), 2)
    assert need > 0
    assert shared(desc(), None, s, ws=0) == _lib.INVALID_ARGUMENT and "workspace" in _lib.last_error()
    assert shared(desc(), None, s, ws=P + 16) == _lib.INVALID_ARGUMENT and "256-byte" in _lib.last_error()
    assert shared(desc(), None, s, ws_bytes=need - 1) == _lib.RESOURCE_EXHAUSTED
    assert shared(desc(n_rows=0), None, s, q=0, out=0) == _lib.OK
    assert shared(desc(n_seq=0, n_rows=0), None, s, q=0, out=0, table=0, kv_len=0) == _lib.OK


def test_null_structs():
    L, d = _lib.lib(), ctypes.byref(desc())
    assert L.mx_paged_decode_shared(d, None, None, P, P, P, P, P, P, None, P, 1 << 40, None) == _lib.INVALID_ARGUMENT
    assert "prefix" in _lib.last_error()
    assert L.mx_paged_decode_shared(None, None, ctypes.byref(prefix()), P, P, P, P, P, P, None, P, 1 << 40, None) == _lib.INVALID_ARGUMENT
    assert L.mx_paged_decode_shared_workspace_bytes(None, 1) == 0
    assert _lib.paged_decode_shared_workspace_bytes(desc(head_dim=96), 1) == 0 and "head_dim" in _lib.last_error()
    assert _lib.paged_decode_shared_workspace_bytes(desc(), 65536) == 0 and "n_groups" in _lib.last_error()


@pytest.mark.parametrize("n_head,n_kv,hd", [(14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 256)])
def test_workspace_sized_once(n_head, n_kv, hd):
    """A workspace for the most sequences, groups and own keys serves fewer."""
    for n_q in (1, 4):
        size = lambda n_seq, groups, own: A.paged_shared_workspace_bytes(n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_q=n_q, n_seq=n_seq,
                                                                         n_groups=groups, max_own_len=own)
        seqs, owns = (1, 2, 16, 64, 300, 3000), (1, 100, 129, 1000, 30000)
        for i, n_seq in enumerate(seqs):
            counts = (0, 1, 2, 16, 300)
            for j, own in enumerate(owns):
                for n, groups in enumerate(counts):
                    b = size(n_seq, groups, own)
                    assert b > 0 and (j == 0 or b >= size(n_seq, groups, owns[j - 1])) and (n == 0 or b >= size(n_seq, counts[n - 1], own))
                    assert i == 0 or b >= size(seqs[i - 1], groups, own)
        assert A.paged_shared_workspace_bytes(n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_q=n_q, n_seq=16, n_groups=4, max_own_len=0) >= \
            A.paged_shared_workspace_bytes(n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_q=n_q, n_seq=16, n_groups=4, max_own_len=5000)


def test_front_end_refusals(monkeypatch):
    monkeypatch.setattr(A, "_native", lambda: A._General())
    k = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    q, table, kv_len = torch.zeros(2, 4 * 64, dtype=torch.float16), torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    cu, plen = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([1], dtype=torch.int32)
    call = lambda cu=cu, plen=plen, q=q, **kw: A.paged_decode_shared(q, k, k, table, kv_len, cu, plen, n_head=4, **kw)
    with pytest.raises(ValueError, match="device tensor"):
        call()
    with pytest.raises(ValueError, match="3 rows|rows, not"):
        call(q=torch.zeros(3, 256, dtype=torch.float16))
    for bad in (cu.long(), cu[None], torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="cu_seq"):
            call(cu=bad)
    with pytest.raises(ValueError, match="prefix_len"):
        call(plen=plen.float())
    with pytest.raises(ValueError, match="one entry more"):
        call(cu=torch.zeros(3, dtype=torch.int32))
