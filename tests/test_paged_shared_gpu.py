"""Decode attention of sequences that share prefixes, against the definition in 64 bits (paged_helpers.py) over each sequence's keys:
the prefix's from the pages of its group's first sequence, the rest from its own.

Tolerances. The prefix's part is computed as packed prompts are (the sum that divides is that of the rounded probabilities), the other
as decode is; `attend` with rounded_sum bounds both. The join adds a rounding of 2^-24 and an exponential's 2^-21 a part, which the
64 parts at most of its terms L 2^-24 and 2^-21 cover."""
import math

import pytest
import torch

from dooms_amd import attention as A
from e4m3_helpers import Cache8
from paged_helpers import Cache, attend, close
from test_paged_gpu import BF16, F16, F32, gen, padded

pytestmark = pytest.mark.gpu


class Shared:
    """Groups of (prefix length, own lengths of its sequences) over a cache whose tables share the prefix's pages: whole ones are the
    first sequence's, the others' own tables say nothing for them; of a page that the prefix ends in each sequence has a copy of
    its own, in which the prefix's rows are garbage but for the first's."""

    def __init__(self, g, groups, n_kv, hd, page, dtype, eight=False, gaps=(), **kw):
        self.groups = groups
        lens = [p + o for p, own in groups for o in own]
        self.cache = (Cache8 if eight else Cache)(g, lens, n_kv, hd, page, dtype, **kw)
        self.eight, self.dtype, self.hd, self.n_head_kv, self.lens, self.page = eight, dtype, hd, n_kv, lens, page
        self.first, c = [], self.cache
        b = 0
        for p, own in groups:
            self.first += [b] * len(own)
            for i in range(1, len(own)):
                c.table[b + i, :p // page] = -3
                if p % page:
                    for pool in ((c.k, c.v, c.ks, c.vs) if eight else (c.k, c.v)):
                        at = c.table[b + i, p // page].long()
                        if at < 0 or at >= pool.shape[0]:
                            continue
                        if pool.dim() == 3:
                            pool[at, :, :p % page] = 255
                        else:
                            pool[at, :p % page] = 0x7f if eight else float("nan")
            b += len(own)
        self.prefix = [p for p, own in groups for _ in own]
        self.cu = [0]
        for _, own in groups:
            self.cu.append(self.cu[-1] + len(own))

    def keys(self, b):
        c, p = self.cache, min(self.prefix[b], self.lens[b])
        first, mine = c.keys(self.first[b], p), c.keys(b, self.lens[b]) if self.first[b] == b else self._own(b)
        return tuple(torch.cat((x[:p], y[p:])) for x, y in zip(first, mine))

    def _own(self, b):
        table = self.cache.table.clone()
        self.cache.table[b, :self.prefix[b] // self.page] = self.cache.table[self.first[b], :self.prefix[b] // self.page]
        try:
            return self.cache.keys(b, self.lens[b])
        finally:
            self.cache.table = table

    def to(self, device):
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
        return (*self.cache.to(device)[:4], ints(self.cu), ints([p for p, _ in self.groups])), \
            (self.cache.to(device)[4] if self.eight else None)


def check(device, seed, n_head, n_kv, hd, groups, page, dtype, n_q=1, causal=True, scale=None, out_dtype=None, eight=False, pad=0, own_hint=None,
          ws=None, mutate=None, what="", **kw):
    g = gen(seed)
    s = Shared(g, groups, n_kv, hd, page, dtype, eight, **kw)
    if mutate:
        mutate(s)
    q = torch.randn(len(s.lens) * n_q, n_head * hd, generator=g).to(dtype)
    od = out_dtype or dtype
    dev_q, out = q.to(device), torch.full((q.shape[0], n_head * hd), 3.0, dtype=od, device=device)
    if pad:
        dev_q, out = padded(dev_q, pad), padded(out, pad)
    args, scales = s.to(device)
    o, lse = A.paged_decode_shared(dev_q, *args, n_head=n_head, n_q=n_q, causal=causal, scale=scale, out=out, want_lse=True,
                                   max_own_len=own_hint, scales=scales, workspace=ws)
    assert o.data_ptr() == out.data_ptr()
    ref, rlse, tol, ltol = attend(s, q, [n_q] * len(s.lens), n_head, 1 / math.sqrt(hd) if scale is None else scale, causal, True, od)
    close(o, ref, tol, f"{what} out")
    close(lse, rlse, ltol, f"{what} lse")


HEADS = [(64, 14, 2), (128, 28, 4), (128, 8, 8), (128, 32, 8), (256, 4, 1)]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,n_head,n_kv", HEADS)
def test_one_group(device, hd, n_head, n_kv, dtype, eight):
    """Prefixes of one key to many, in whole pages and not, own keys from one on; two sequences to more than a tile holds."""
    for p, own in ((16, [1, 5]), (1, [1, 2, 3]), (63, [9, 30, 1]), (64, [40] * 9), (700, [3, 200, 17, 64]), (1000, [1 + 7 * i % 90 for i in range(40)]),
                   (5000, [20, 600])):
        check(device, 50, n_head, n_kv, hd, [(p, own)], 16, dtype, eight=eight, what=f"{p} {len(own)}")


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd,n_head,n_kv", HEADS)
def test_groups(device, hd, n_head, n_kv, eight):
    """Groups of very different prefixes and sizes: of one sequence, without a prefix, of none."""
    groups = [(300, [10, 1, 50]), (0, [33, 70]), (2000, [5]), (40, []), (17, [400, 1]), (0, []), (900, [30, 30, 600, 2, 9])]
    for page in (16, 64):
        check(device, 51, n_head, n_kv, hd, groups, page, BF16, eight=eight, what=f"{page}")
    many = [(16 + 11 * i % 200, [1 + (i + j) % 20 for j in range(1 + i % 3)]) for i in range(80)]
    check(device, 52, n_head, n_kv, hd, many, 16, F16, eight=eight, what="many")


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_q,causal", [(2, True), (4, True), (3, False), (8, True)])
def test_rows(device, hd, n_q, causal, eight):
    """Several new rows; sequences whose own keys are the new ones alone, and (the last key that all rows see is the prefix's) all but one."""
    for groups in ([(100, [n_q, n_q + 30, n_q - 1, 2 * n_q])], [(64, [n_q - 1, n_q]), (530, [n_q + 90, n_q, n_q + 1])]):
        check(device, 53, 14, 2, hd, groups, 16, F16, n_q=n_q, causal=causal, eight=eight, what=f"{groups}")
    for scale in (0.0, -0.3):
        check(device, 54, 8, 8, hd, [(90, [n_q, 40, 300])], 32, BF16, n_q=n_q, causal=causal, scale=scale, eight=eight, what=f"{scale}")


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_layouts(device, hd):
    for page, heads_first, pad, od, eight in ((16, True, 8, F32, False), (128, False, 24, None, False), (64, True, 8, F32, True)):
        check(device, 55, 8, 2, hd, [(200, [1, 77, 30]), (450, [5, 5])], page, F16, heads_first=heads_first, pad=pad, out_dtype=od, eight=eight)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd,group", [(64, 7), (128, 1), (128, 4), (128, 8), (256, 4)])
def test_many_sequences_in_ranges(device, hd, group, eight):
    """More own keys than chunks serve: the workgroups walk ranges of them, with prefixes of different lengths from sequence to sequence,
    and no hint of their lengths."""
    own = [1 + (b * 53) % 400 for b in range(40)]
    own[17], own[39] = 2100, 900
    groups = [(333, own[:17]), (48, own[17:18]), (1029, own[18:38]), (0, own[38:])]
    check(device, 56, 8 * group, 8, hd, groups, 16, BF16, eight=eight, extra_width=380)


def test_more_rows_than_the_chip_holds(device):
    check(device, 57, 8, 8, 64, [(70, [16 + i % 3 for i in range(600)])], 16, F16, n_q=16, own_hint=18)


@pytest.mark.parametrize("hint", [1, 100, 100000])
@pytest.mark.parametrize("n_seq", [2, 30])
def test_hints_may_be_wrong(device, hint, n_seq):
    check(device, 58, 8, 2, 128, [(100, [1 + 31 * i % 700 for i in range(n_seq)])], 16, F16, own_hint=hint)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_empty_and_wrong_sequences(device, hd, eight):
    """Padding entries of 0 keys are zeros and take nothing from their group; fewer keys than the prefix, a length or prefix that is none
    and a page that is none are NaN, where they belong."""
    g = gen(59)
    groups = [(100, [5, 7, 9, 30, 2]), (50, [4, 4, 4]), (40, [6, 6]), (64, [3])]
    s = Shared(g, groups, 2, hd, 16, F16, eight)
    q = torch.randn(len(s.lens), 8 * hd, generator=g).to(F16)
    ref, rlse, tol, ltol = attend(s, q, [1] * len(s.lens), 8, hd ** -0.5, True, True, F16)
    (k, v, table, kv_len, cu, plen), scales = s.to(device)
    capacity = table.shape[1] * 16
    kv_len[1], kv_len[2], kv_len[3], kv_len[6] = 0, 99, capacity + 1, -5
    table[4, 102 // 16] = k.shape[0]  # of its own keys
    plen[2] = -1
    plen[3] = capacity + 1
    nan, zero, ok = [2, 3, 4, 6, 8, 9, 10], [1], [0, 5, 7]
    ws = A.new_workspace(256 << 20, device)
    for _ in range(2):
        o, lse = A.paged_decode_shared(q.to(device), k, v, table, kv_len, cu, plen, n_head=8, want_lse=True, scales=scales, workspace=ws)
        assert torch.isnan(o[nan]).all() and torch.isnan(lse[nan]).all()
        assert (o[zero] == 0).all() and (lse[zero] == -math.inf).all()
        close(o[ok], ref[ok], tol[ok], "others")
        close(lse[ok], rlse[ok], ltol[ok], "others' lse")
    table[0, 2] = -1  # of the prefix: all that attend it
    o, _ = A.paged_decode_shared(q.to(device), k, v, table, kv_len, cu, plen, n_head=8, scales=scales, workspace=ws)
    assert torch.isnan(o[[0, 2, 3, 4]]).all() and (o[1] == 0).all()
    close(o[[5, 7]], ref[[5, 7]], tol[[5, 7]], "others")


def test_group_bounds_that_are_none(device):
    """Out of range, backwards or overlapping: in bounds, and right for the sequences of sound groups beside them."""
    g = gen(60)
    s = Shared(g, [(48, [5, 6, 7, 8]), (0, [9, 10])], 2, 128, 16, F16)
    q = torch.randn(6, 8 * 128, generator=g).to(F16)
    ref, _, tol, _ = attend(s, q, [1] * 6, 8, 128 ** -0.5, True, True, F16)
    (k, v, table, kv_len, _, _), _ = s.to(device)
    ws = A.new_workspace(256 << 20, device)

    def call(cu, plen):
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
        return A.paged_decode_shared(q.to(device), k, v, table, kv_len, ints(cu), ints(plen), n_head=8, workspace=ws)[0]
    close(call([0, 4], [48]), ref, tol, "sequences of no group")
    close(call([-7, 4, 6, 1000], [48, 0, 5]), ref, tol, "clamped")
    close(call([0, 4, 4, 4, 6], [48, 9, 1000, 0]), ref, tol, "empty groups")
    for cu, plen in (([6, 4, 0], [48, 48]), ([0, 6, 0, 6], [48, 48, 48]), ([5, 5, 5], [1, 1]), ([0, 6, 0, 6, 0, 6, 0], [48] * 6)):
        call(cu, plen)  # undefined, in bounds
    close(call([0, 4], [48]), ref, tol, "the next call")


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_no_numbers(device, hd, eight):
    """A value that is no number or infinite: in the prefix all rows of its group have it, among own keys the rows that see it."""
    def poke(b, pos):
        def f(s):
            c = s.cache
            page, row = int(c.table[b, pos // 16]), pos % 16
            if eight:
                c.v[page, row, 1, 9] = 0x7f
            else:
                c.v[page, row, 1, 9] = math.inf
        return f
    for b, pos in ((0, 70), (1, 103)):
        check(device, 61, 6, 2, hd, [(100, [4, 6, 30]), (33, [4, 5])], 16, F16, n_q=4, eight=eight, mutate=poke(b, pos), what=f"{b} {pos}")


def test_results_do_not_depend_on_the_run(device):
    g = gen(62)
    s = Shared(g, [(3000, [1 + 37 * i % 500 for i in range(30)])], 8, 128, 16, BF16)
    q = torch.randn(30, 32 * 128, generator=g).to(BF16).to(device)
    args, _ = s.to(device)
    ws = A.new_workspace(256 << 20, device)
    want = A.paged_decode_shared(q, *args, n_head=32, workspace=ws)[0]
    for _ in range(20):
        assert torch.equal(A.paged_decode_shared(q, *args, n_head=32, workspace=ws)[0], want)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n_head,n_kv,hd", [(14, 2, 64), (32, 8, 128), (4, 2, 256)])
def test_steps_captured(device, n_head, n_kv, hd, eight):
    """A step (append, decode) of sampled answers, captured and replayed while they grow, one ends and the prefixes change, with other
    calls on the same workspace between the replays."""
    g = gen(63)
    dtype, steps = BF16, 4
    groups = [(100, [9, 1, 30]), (257, [4, 4])]
    s = Shared(g, [(p, [o + steps + 1 for o in own]) for p, own in groups], n_kv, hd, 16, dtype, eight)
    c = s.cache
    lens = [p + o for p, own in groups for o in own]
    (k, v, table, kv_len, cu, plen), scales = s.to(device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    wide = (n_head + 2 * n_kv) * hd
    with torch.cuda.stream(stream):
        ws = A.new_workspace(256 << 20, device)
        x, q = torch.zeros(5, wide, device=device), torch.zeros(5, n_head * hd, dtype=dtype, device=device)
        o = torch.zeros_like(q)

        def step():
            A.paged_store(x, k, v, table, kv_len, n_head=n_head, rope_mode=1, q=q, scales=scales)
            A.paged_decode_shared(q, k, v, table, kv_len, cu, plen, n_head=n_head, out=o, scales=scales, workspace=ws)
        kv_len.copy_(torch.tensor([n + 1 for n in lens], dtype=torch.int32))
        step()
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(steps):
            lens = [n + 1 for n in lens]
            if i == 2:
                lens[1] = 0  # ended
                plen.copy_(torch.tensor([40, 200], dtype=torch.int32))  # a shorter prefix is a prefix too ...
                table[1:3, :6], table[4, :16] = table[0, :6].clone(), table[3, :16].clone()  # ... with the rest in every table
                if eight:
                    for t in (k.view(torch.uint8), v.view(torch.uint8)):
                        t[table[2, 6].long(), :4], t[table[4, 16].long(), :1] = t[table[0, 6].long(), :4].clone(), t[table[3, 16].long(), :1].clone()
                    for t in scales:
                        t = t.view(torch.uint8)
                        t[table[2, 6].long(), :, :4], t[table[4, 16].long(), :, :1] = t[table[0, 6].long(), :, :4].clone(), t[table[3, 16].long(), :, :1].clone()
                else:
                    for t in (k, v):
                        t[table[2, 6].long(), :4], t[table[4, 16].long(), :1] = t[table[0, 6].long(), :4].clone(), t[table[3, 16].long(), :1].clone()
                c.table = table.cpu()
                s.prefix = [40] * 3 + [200] * 2
            if i > 2:
                lens[1] = 0
            kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
            x.copy_(torch.randn(5, wide, generator=g))
            graph.replay()
            stream.synchronize()
            names = ("k", "v", "ks", "vs") if eight else ("k", "v")
            for name, t in zip(names, (k, v, *(scales or ()))):
                setattr(c, name, t.view(torch.uint8).cpu() if eight else t.cpu())
            s.lens = c.lens = lens
            ref, _, tol, _ = attend(s, q.cpu(), [1] * 5, n_head, hd ** -0.5, True, True, dtype)
            close(o, ref, tol, f"step {i}")
            A.paged_decode(q, k, v, table[:1].repeat(5, 1), torch.full_like(kv_len, 60), n_head=n_head, scales=scales, workspace=ws)


def test_extension_and_general_path_agree(device, monkeypatch):
    for eight in (False, True):
        g = gen(64)
        s = Shared(g, [(100, [3, 60])], 2, 128, 16, F16, eight)
        q = torch.randn(2, 8 * 128, generator=g).to(F16).to(device)
        args, scales = s.to(device)
        ws = A.new_workspace(A.paged_shared_workspace_bytes(n_head=8, n_head_kv=2, head_dim=128, n_q=1, n_seq=2, n_groups=1, max_own_len=60), device)
        call = lambda **kw: A.paged_decode_shared(q, *args, n_head=8, want_lse=True, scales=scales, max_own_len=60, **kw)
        want = call(workspace=ws)
        with monkeypatch.context() as m:
            m.setattr(A, "_native", lambda: A._General())
            for got in (call(workspace=ws), call()):
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        none = torch.zeros(0, dtype=torch.int32, device=device)
        o, _ = A.paged_decode_shared(q[:1], *args[:2], args[2][:1].contiguous(), args[3][:1].contiguous(), none.new_zeros(1), none, n_head=8,
                                     scales=scales)  # no groups: nothing is shared
        alone, _ = A.paged_decode(q[:1], *args[:2], args[2][:1].contiguous(), args[3][:1].contiguous(), n_head=8, scales=scales)
        assert torch.equal(o, alone)


@pytest.mark.parametrize("eight", [False, True])
def test_groups_of_one_and_one_sequence(device, eight):
    """Nothing is shared then, and the results are those of a decode."""
    for groups in ([(30, [5])], [(30 + 7 * i, [1 + 40 * i]) for i in range(9)]):
        check(device, 65, 8, 2, 128, groups, 16, F16, eight=eight, what=f"{len(groups)}")


@pytest.mark.parametrize("n_groups", [64, 65, 4200])
def test_many_groups(device, n_groups):
    """A sequence's group among many, with runs of empty ones."""
    groups = [(16 + i % 40, [] if i % 7 == 3 or 20 <= i < 30 else [1 + i % 9] * (1 + i % 3 // 2)) for i in range(n_groups)]
    check(device, 66, 1, 1, 64, groups, 16, F16, own_hint=9)


def test_calls_on_two_streams(device):
    """Each with a workspace of its own."""
    g = gen(67)
    s = Shared(g, [(2000, [1 + 37 * i % 300 for i in range(20)])], 4, 128, 16, BF16)
    args, _ = s.to(device)
    qs = [torch.randn(20, 16 * 128, generator=g).to(BF16).to(device) for _ in range(2)]
    ws = [A.new_workspace(64 << 20, device) for _ in range(2)]
    want = [A.paged_decode_shared(q, *args, n_head=16, workspace=w)[0] for q, w in zip(qs, ws)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(A.paged_decode_shared(qs[i], *args, n_head=16, workspace=ws[i])[0])
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


def test_workspace_shared_with_other_calls(device):
    """The counters of the calls that keep them lie in front of what this one writes."""
    g = gen(68)
    s = Shared(g, [(2496, [1 + 37 * i % 500 for i in range(12)])], 4, 128, 16, F16)
    q = torch.randn(12, 16 * 128, generator=g).to(F16).to(device)
    args, _ = s.to(device)
    table = s.cache.table.clone()
    table[1:, :156] = table[0, :156]  # whole pages of the prefix, which a plain decode reads too
    plain = (args[0], args[1], table.to(device), args[3])
    prompt = torch.randn(300, 16 * 128, generator=g).to(F16).to(device)
    cu = torch.tensor([0] * 12 + [300], dtype=torch.int32, device=device)
    calls = [lambda w: A.paged_decode_shared(q, *args, n_head=16, workspace=w)[0], lambda w: A.paged_decode(q, *plain, n_head=16, workspace=w)[0],
             lambda w: A.paged_prefill(prompt, *plain, cu, n_head=16, workspace=w)[0]]
    want = [f(A.new_workspace(128 << 20, device)) for f in calls]
    ws = A.new_workspace(128 << 20, device)
    for _ in range(3):
        for f, w in zip(calls, want):
            assert torch.equal(f(ws), w)
            assert not ws[:A._PAGED_COUNTERS].any()


def test_calls_without_groups_need_no_more(device):
    """The workspace sized for a call serves it without groups as well."""
    for n_head, n_kv, hd, n_seq in ((8, 2, 128, 1), (14, 2, 64, 3), (4, 1, 256, 40)):
        g = gen(69)
        c = Cache(g, [900 + 7 * i for i in range(n_seq)], n_kv, hd, 16, F16)
        q = torch.randn(n_seq, n_head * hd, generator=g).to(F16).to(device)
        none = torch.zeros(1, dtype=torch.int32, device=device)
        nb = A.paged_shared_workspace_bytes(n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_q=1, n_seq=n_seq, n_groups=0, max_own_len=2000)
        ws = A.new_workspace(nb, device)
        ref, _, tol, _ = attend(c, q.cpu(), [1] * n_seq, n_head, hd ** -0.5, True, False, F16)
        close(A.paged_decode_shared(q, *c.to(device), none, none[:0], n_head=n_head, max_own_len=2000, workspace=ws)[0], ref, tol, "out")
