"""One workspace for calls of different entry points: each leaves the split counters at its start at zero for the next."""
import math

import pytest
import torch

from dooms_amd import _lib
from dooms_amd import attention as A

COUNTERS = 2048 * 256  # bytes at the start of a workspace


@pytest.mark.parametrize("n_head,n_kv,hd,n_q", [(32, 8, 128, 100), (14, 2, 64, 60), (8, 8, 256, 128), (28, 4, 128, 1)])
def test_rotated_rows_of_short_prompts_lie_behind_the_counters(n_head, n_kv, hd, n_q):
    d = _lib.make_desc(n_head, n_kv, hd, n_q, (n_head + 2 * n_kv) * hd, n_kv * hd, n_head * hd, 1 / math.sqrt(hd), causal=1)
    rows = n_q * n_head * hd * 4
    assert _lib.prefill_workspace_bytes(d) >= COUNTERS + rows
    P = 4096
    call = lambda nb: _lib.prefill_rope_ws_raw(d, 0, 1e4, P, P, P, P, 0, P, nb, 0)
    assert call(COUNTERS + rows - 1) == _lib.RESOURCE_EXHAUSTED and "workspace" in _lib.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,hd,n_q", [(32, 8, 128, 100), (14, 2, 64, 60)])
def test_short_prompt_then_split_decode(device, n_head, n_kv, hd, n_q):
    """A decoder's workspace: a prompt of fewer keys than a split, then a step over a long cache."""
    g = torch.Generator().manual_seed(1)
    heads = dict(n_head=n_head, n_head_kv=n_kv, head_dim=hd)
    ws = A.new_workspace(64 << 20, device)
    qkv = torch.randn(n_q, (n_head + 2 * n_kv) * hd, generator=g).to(device)
    k, v = (torch.randn(5000, n_kv * hd, generator=g).half().to(device) for _ in range(2))
    q = torch.randn(1, n_head * hd, generator=g).half().to(device)
    want = A.decode(q, [k], [v], [5000], **heads)[0]
    short = [torch.zeros(n_q, n_kv * hd, dtype=torch.float16, device=device) for _ in range(2)]
    alone = A.prefill_rope(qkv, *short, rope_mode=0, workspace="auto", **heads)[0]
    for _ in range(2):
        out = A.prefill_rope(qkv, *short, rope_mode=0, workspace=ws, **heads)[0]
        assert torch.equal(out, alone)
        assert not ws[:COUNTERS].any()
        assert torch.equal(A.decode(q, [k], [v], [5000], workspace=ws, **heads)[0], want)


@pytest.mark.gpu
def test_every_call_that_keeps_counters(device):
    """The calls that may share a workspace, each split, in turn on one: the results of a workspace of their own, and the counters
    at zero behind each."""
    g = torch.Generator().manual_seed(2)
    n_head, n_kv, hd, L = 16, 4, 128, 3000
    heads = dict(n_head=n_head, n_head_kv=n_kv, head_dim=hd)
    rnd = lambda *s: torch.randn(*s, generator=g).to(device)
    q, qkv = rnd(40, n_head * hd).half(), rnd(40, (n_head + 2 * n_kv) * hd)
    k, v = rnd(L, n_kv * hd).half(), rnd(L, n_kv * hd).half()
    pages = [rnd(400, 16, n_kv, hd).half() for _ in range(2)]
    table = torch.randperm(400, generator=g).to(torch.int32).view(2, 200).to(device)
    lens = torch.tensor([3200, 1500], dtype=torch.int32, device=device)
    cu = torch.tensor([0, 30, 40], dtype=torch.int32, device=device)
    calls = [
        lambda ws: A.decode(q[:1], [k], [v], [L], workspace=ws, **heads)[0],
        lambda ws: A.paged_decode(q[:2], *pages, table, lens, n_head=n_head, workspace=ws)[0],
        lambda ws: A.decode(q[:1].float(), [k], [v], [L], workspace=ws, **heads)[0],
        lambda ws: A.decode_rope(qkv[:1], [k.clone()], [v.clone()], [L], rope_mode=1, workspace=ws, **heads)[0],
        lambda ws: A.paged_prefill(q, *pages, table, lens, cu, n_head=n_head, workspace=ws)[0],
        lambda ws: A.prefill(q, k, v, p0=L - 40, workspace=ws, **heads)[0],
        lambda ws: A.paged_decode(q[:16], *pages, table, lens, n_head=n_head, n_q=8, workspace=ws)[0],
        lambda ws: A.prefill_rope(qkv, k.clone(), v.clone(), p0=L - 40, rope_mode=0, workspace=ws, **heads)[0],
        lambda ws: A.prefill_rope(qkv[:9], k[:9].clone(), v[:9].clone(), rope_mode=0, workspace=ws, **heads)[0],
    ]
    want = [f(A.new_workspace(128 << 20, device)) for f in calls]
    ws = A.new_workspace(128 << 20, device)
    for _ in range(2):
        for i, f in enumerate(calls):
            assert torch.equal(f(ws), want[i]), i
            assert not ws[:COUNTERS].any(), i


def test_one_counter_region():
    """Every call's partials lie behind the same counters, which the front end zeroes."""
    paged = A.paged_decode_workspace_bytes(n_head=1, n_head_kv=1, head_dim=64, n_q=1, n_seq=1, max_kv_len=1 << 20)
    assert paged - 2 * 512 * 4 * (64 + 4) * 4 == COUNTERS  # two partials of 4 rows for each of 512 workgroups
    prompts = A.paged_prefill_workspace_bytes(n_head=1, n_head_kv=1, head_dim=64, n_rows=1, n_seq=1, max_q=1, max_kv_len=1)
    assert prompts - 2 * 512 * 4 * 64 * (32 + 2) * 4 == COUNTERS  # of 4 waves, 32 outputs, m and l a lane
    assert A.decode_workspace_bytes(n_head=1, n_head_kv=1, head_dim=64, n_q=1, batch=1, max_kv_len=256) - 2 * 4 * (64 + 4) * 4 == COUNTERS
    assert A._PAGED_COUNTERS == COUNTERS


def test_workspace_without_a_length():
    """No length and no table: room for any length, as the call that follows may be split."""
    for n_seq in (1, 3, 200, 65535):
        shape = dict(n_head=8, n_head_kv=2, head_dim=128, n_q=1, n_seq=n_seq)
        assert A.paged_decode_workspace_bytes(max_kv_len=0, **shape) == A.paged_decode_workspace_bytes(max_kv_len=100000, **shape) > 0
