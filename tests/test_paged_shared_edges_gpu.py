"""Decode behind shared prefixes where its own plan can go wrong: what the first launch leaves for the join, and sizes at the ends of what
the call takes."""
import math

import pytest
import torch

from dooms_amd import attention as A
from paged_helpers import attend, close
from test_paged_gpu import BF16, F16, F32, gen
from test_paged_shared_gpu import Shared, check

pytestmark = pytest.mark.gpu


def left_for_the_join(ws, n_seq):
    """(rows of a kv head's partials, own keys of each sequence, [first row, rows of a part, parts, own row] of each) in a workspace: they lie
    behind the counters, each block in whole 256 bytes."""
    w = ws.view(torch.int32)[A._PAGED_COUNTERS // 4:].cpu()
    own = 64 + (n_seq + 63) // 64 * 64
    return int(w[0]), w[64:64 + n_seq], w[own:own + 4 * n_seq].view(n_seq, 4)


@pytest.mark.parametrize("n_groups", [200, 20000])
def test_overlapping_groups_that_have_no_room(device, n_groups):
    """Groups of all sequences over and over: more parts than the launch has workgroups for, and rows than the workspace. The join is
    given none of them, and nothing around the workspace is written."""
    n_seq, n_head, n_kv, hd, keys = 192, 32, 8, 128, 256
    g = gen(80)
    s = Shared(g, [(keys, [5 + i % 9 for i in range(n_seq)])], n_kv, hd, 16, F16)
    q = torch.randn(n_seq, n_head * hd, generator=g).to(F16).to(device)
    (k, v, table, kv_len, cu, plen), _ = s.to(device)
    nb = A.paged_shared_workspace_bytes(n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_q=1, n_seq=n_seq, n_groups=n_groups, max_own_len=16)
    room = torch.zeros(nb + (64 << 20), dtype=torch.uint8, device=device)
    ws = room[32 << 20:(32 << 20) + nb]
    many = torch.tensor([0, n_seq] * (n_groups // 2) + [0], dtype=torch.int32, device=device)
    call = lambda cu, plen: A.paged_decode_shared(q, k, v, table, kv_len, cu, plen, n_head=n_head, max_own_len=16, workspace=ws)[0]
    call(many, torch.full((n_groups,), keys, dtype=torch.int32, device=device))  # undefined, in bounds
    rows, _, info = left_for_the_join(ws, n_seq)
    assert rows == 0  # there was no room
    assert (info[:, :3] == 0).all()
    assert not room[:32 << 20].any() and not room[(32 << 20) + nb:].any()
    ref, _, tol, _ = attend(s, q.cpu(), [1] * n_seq, n_head, hd ** -0.5, True, True, F16)
    close(call(cu, plen), ref, tol, "the next call")
    rows, _, info = left_for_the_join(ws, n_seq)
    assert rows > 0 and (info[:, 2] > 0).all()


class Sample:
    """Some sequences of a cache whose sequences all have the same first keys, for `attend`."""

    def __init__(self, k, v, lens):
        self.k, self.v, self.lens, self.dtype = k.double(), v.double(), lens, k.dtype
        self.n_head_kv, self.hd = k.shape[1:]

    def keys(self, b):
        return self.k[:self.lens[b]], self.v[:self.lens[b]]


def test_more_rows_than_a_grid_holds_in_a_line(device):
    """2^24 rows of heads of 256: a row a workgroup of the join, and 2^32 threads."""
    n_seq = n_head = 4096
    n_kv, hd, page = 64, 256, 16
    g = gen(81)
    kp, vp = (torch.randn(2, page, n_kv, hd, generator=g).to(F16) for _ in range(2))
    lens = [page + 1 + b % 3 for b in range(n_seq)]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    dg = torch.Generator(device=device).manual_seed(81)
    q = torch.randn(n_seq, n_head * hd, generator=dg, dtype=F16, device=device)
    out = torch.full_like(q, math.nan)
    o, lse = A.paged_decode_shared(q, kp.to(device), vp.to(device), ints([[0, 1]] * n_seq), ints(lens), ints([0, n_seq]), ints([page]), n_head=n_head,
                                   out=out, want_lse=True, max_own_len=3)
    assert torch.isfinite(lse).all()
    for rows in o.split(256):
        assert torch.isfinite(rows).all()
    some = [0, 2047, 2048, 4095]
    c = Sample(kp.flatten(0, 1), vp.flatten(0, 1), [lens[b] for b in some])
    ref, rlse, tol, ltol = attend(c, q[some].cpu(), [1] * len(some), n_head, hd ** -0.5, True, True, F16)
    close(o[some], ref, tol, "out")
    close(lse[some], rlse, ltol, "lse")


@pytest.mark.parametrize("n_q", [1, 3])
@pytest.mark.parametrize("eight", [False, True])
def test_a_prefix_longer_than_a_sequence_alone(device, eight, n_q):
    """A row has to see the whole prefix, of a group of one sequence too."""
    g = gen(82)
    s = Shared(g, [(100, [9]), (40, [4, 5]), (300, [n_q - 1 or 1])], 2, 64, 16, F16, eight)
    q = torch.randn(4 * n_q, 4 * 64, generator=g).to(F16)
    ref, rlse, tol, ltol = attend(s, q, [n_q] * 4, 4, 0.125, True, True, F16)
    (k, v, table, kv_len, cu, plen), scales = s.to(device)
    kv_len[0] = 100 + n_q - 2  # one row sees all but a key
    o, lse = A.paged_decode_shared(q.to(device), k, v, table, kv_len, cu, plen, n_head=4, n_q=n_q, want_lse=True, scales=scales)
    assert torch.isnan(o[:n_q]).all() and torch.isnan(lse[:n_q]).all()
    close(o[n_q:], ref[n_q:], tol[n_q:], "others")
    close(lse[n_q:], rlse[n_q:], ltol[n_q:], "others' lse")


@pytest.mark.parametrize("n_q,causal", [(1, True), (3, False)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_no_keys_behind_the_prefix(device, hd, eight, n_q, causal):
    """Sequences that end with their prefix, at a page's end, a multiple of 16 and neither: what their tables say from there on places none
    of their keys, and may be no page."""
    groups = [(64, [0, 9, 0]), (48, [0, 0]), (100, [30, 0, 0, 5]), (7, [0, 3])]
    check(device, 83, 8, 2, hd, groups, 32, F16, n_q=n_q, causal=causal, eight=eight)
    g = gen(84)
    s = Shared(g, groups, 2, hd, 32, F16, eight)
    q = torch.randn(len(s.lens) * n_q, 8 * hd, generator=g).to(F16)
    ref, rlse, tol, ltol = attend(s, q, [n_q] * len(s.lens), 8, hd ** -0.5, causal, True, F16)
    for b in range(len(s.lens)):
        if s.first[b] != b and s.lens[b] == s.prefix[b]:
            s.cache.table[b] = -5
    args, scales = s.to(device)
    o, lse = A.paged_decode_shared(q.to(device), *args, n_head=8, n_q=n_q, causal=causal, want_lse=True, scales=scales)
    close(o, ref, tol, "out")
    close(lse, rlse, ltol, "lse")


@pytest.mark.parametrize("n_q", [1, 3])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 14, 2), (128, 8, 2), (256, 4, 1)])
def test_long_prefixes_of_one_sequence(device, hd, n_head, n_kv, eight, n_q):
    """The hint counts the keys behind the prefix, of a sequence alone in its group too: prefixes longer than a chunk of those are computed in
    parts, as shared ones are."""
    n = [max(i, n_q) for i in range(12)]
    groups = [(4000, [9 + n_q]), (300, [n[4], n[9], n[1]]), (1003, [n[1]]), (20, [n[7]]), (0, [n[5]]), (2048, [n[2]])]
    check(device, 85, n_head, n_kv, hd, groups, 16, BF16, n_q=n_q, eight=eight, own_hint=16)
    check(device, 86, n_head, n_kv, hd, [(5000, [n[3]])], 64, F16, n_q=n_q, eight=eight, own_hint=16)
    ws = A.new_workspace(64 << 20, device)
    check(device, 85, n_head, n_kv, hd, groups, 16, BF16, n_q=n_q, eight=eight, own_hint=16, ws=ws)
    _, own, info = left_for_the_join(ws, 8)
    alone = [0, 4, 7]
    assert (info[alone, 2] >= 8).all() and (own[alone] < 64).all()
    assert info[5, 2] == 0 and int(own[5]) == 20 + n[7] and info[6, 2] == 0


@pytest.mark.parametrize("eight", [False, True])
def test_more_groups_than_workgroups(device, eight):
    """Prefixes of which none is cut into parts, as there are more of them than a kv head has workgroups: of two sequences and of one, and
    under more kv heads than the chip has CUs."""
    many = [(60 + 13 * i % 300, [1 + (i + j) % 20 for j in range(1 + i % 2)]) for i in range(300)]
    check(device, 87, 4, 2, 64, many, 16, F16, eight=eight, own_hint=20)
    check(device, 88, 600, 300, 64, [(200, [3, 5]), (70, [2, 4, 1]), (500, [9])], 16, F16, eight=eight, own_hint=9)
