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
