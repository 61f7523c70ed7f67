"""The paged cache's kernels against their definitions in 64 bits (paged_helpers.py): every type, head dim, page layout and mask
where they can go wrong."""
import math

import pytest
import torch

from dooms_amd import _lib
from dooms_amd import attention as A
from paged_helpers import TINY, U, Cache, attend, close, rotate

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN = float("nan")


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def cu_of(rows, device):
    return torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device=device)


def padded(t, pad, fill=NAN):
    """t's rows at a stride `pad` elements wider."""
    w = torch.full((t.shape[0], t.shape[1] + pad), fill, dtype=t.dtype, device=t.device)
    w[:, :t.shape[1]] = t
    return w[:, :t.shape[1]]


# ---- store ----

def store_case(device, seed, n_head, n_kv, hd, rows, lens, page, dtype, in_dtype, mode, axis_pairs=None, restart=False, positions=None,
               base=10000.0, uniform=False, heads_first=False, pad=0, tail=0, what=""):
    g = gen(seed)
    c = Cache(g, lens, n_kv, hd, page, dtype, heads_first=heads_first)
    total = sum(rows)
    x = torch.randn(total + tail, (n_head + 2 * n_kv) * hd, generator=g).to(in_dtype)
    pairs = axis_pairs or (hd // 2,)
    pos = torch.cat([torch.arange(L - n, L) for n, L in zip(rows, lens)]).to(torch.int32)
    turn_pos = pos[None] if positions is None else positions
    q0 = torch.full((total + tail, n_head * hd), 7.0, dtype=dtype, device=device)
    if pad:
        q0 = padded(q0, pad)
    k, v, table, kv_len = c.to(device)
    dev_x = padded(x.to(device), pad) if pad else x.to(device)
    dev_pos = None
    if positions is not None:
        dev_pos = torch.zeros(len(pairs), total + tail, dtype=torch.int32)
        dev_pos[:, :total] = positions
        dev_pos = dev_pos.to(device)
    got = A.paged_store(dev_x, k, v, table, kv_len, n_head=n_head, rope_mode=mode, rope_base=base, cu_q=None if uniform else cu_of(rows, device),
                        positions=dev_pos, axis_pairs=axis_pairs, axis_restart=restart, q=q0)
    assert got is q0
    xr = x[:total].double().view(total, n_head + 2 * n_kv, hd)
    ref, mag = rotate(xr[:, :n_head + n_kv], turn_pos, mode, base, pairs, restart)
    tol = U[dtype] * ref.abs() + (0.0 if mode == 2 else 2.0 ** -21) * mag + TINY[dtype]
    close(got[:total], ref[:, :n_head].flatten(1), tol[:, :n_head].flatten(1), f"{what} q")
    if tail:
        assert (got[total:] == 7.0).all()
    want_k, want_v, tol_k = c.k.double(), c.v.double(), torch.zeros(c.k.shape, dtype=torch.float64)
    at = 0
    for b, (n, L) in enumerate(zip(rows, lens)):
        p = torch.arange(L - n, L)
        where = (c.table[b, p // page].long(), p % page)
        want_k[where], tol_k[where] = ref[at:at + n, n_head:], tol[at:at + n, n_head:]
        want_v[where] = xr[at:at + n, n_head + n_kv:].to(dtype).double()  # rounded once
        at += n
    close(k, want_k, tol_k, f"{what} k")
    close(v, want_v, torch.zeros_like(want_v), f"{what} v")


@pytest.mark.parametrize("in_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 14, 2), (128, 28, 4), (256, 4, 1)])
def test_store_types(device, hd, n_head, n_kv, dtype, in_dtype):
    for mode in (0, 1, 2):
        store_case(device, 1 + mode, n_head, n_kv, hd, [3, 1, 0, 20], [40, 1, 17, 20], 16, dtype, in_dtype, mode, tail=2, what=f"mode {mode}")


@pytest.mark.parametrize("axis_pairs", [(32, 32), (16, 24, 24), (1, 1, 61, 1)])
@pytest.mark.parametrize("restart", [False, True])
@pytest.mark.parametrize("mode", [0, 1])
def test_store_axes(device, axis_pairs, restart, mode):
    g = gen(5)
    pos = torch.randint(-50, 5000, (len(axis_pairs), 37), generator=g).to(torch.int32)
    store_case(device, 6, 8, 2, 128, [30, 7], [64, 300], 64, BF16, F32, mode, axis_pairs, restart, pos, base=1e6)


@pytest.mark.parametrize("hd,heads_first,pad,uniform", [(128, True, 0, False), (64, False, 24, True), (256, True, 8, True)])
def test_store_layouts(device, hd, heads_first, pad, uniform):
    store_case(device, 9, 4, 4, hd, [2, 2, 2], [2, 33, 700], 32, F16, F32, 1, heads_first=heads_first, pad=pad, uniform=uniform)


def test_store_far_positions(device):
    """Angles in 64 bits: at 2^31 - 1 an f32 product of position and frequency would be off by many turns."""
    pos = torch.tensor([[2 ** 31 - 1, 131071, 10 ** 9 + 7, -(2 ** 31)]], dtype=torch.int32)
    store_case(device, 10, 2, 1, 128, [4], [4], 16, F16, F32, 1, positions=pos, base=5e5)


def test_store_one_sequence_of_many(device):
    """More sequences than a wave has lanes, most of them without new rows."""
    rows = [1 if b % 3 == 0 else 0 for b in range(200)]
    store_case(device, 11, 4, 2, 64, rows, [1 + b % 40 for b in range(200)], 16, F16, F32, 0)


@pytest.mark.parametrize("n_seq", [64, 65, 129, 4097])
def test_store_many_sequences(device, n_seq):
    """The sequence of a row among many, runs of empty ones at the start, in between and at the end."""
    rows = [0 if b < 5 or 30 <= b < 50 or b > n_seq - 7 else b % 3 for b in range(n_seq)]
    store_case(device, 12, 2, 1, 64, rows, [n + b % 20 for b, n in enumerate(rows)], 16, BF16, F16, 1, tail=2)


def test_store_many_rows(device):
    """More rows than a grid has workgroups along one dimension, and offsets past 2^32 bytes."""
    n = (1 << 22) + 5
    x = torch.randn(n, 1, device=device).to(F16) * torch.arange(1, 193, device=device).to(F16)[None] / 64
    table = torch.arange(n // 4096 + 1, dtype=torch.int32, device=device)[None].contiguous()
    k = torch.zeros(table.shape[1], 4096, 1, 64, dtype=F16, device=device)
    wide = torch.zeros(2, table.shape[1], 4096, 10, 64, dtype=F16, device=device)[:, :, :, 9:]
    v = torch.zeros_like(k)
    lens = torch.tensor([n], dtype=torch.int32, device=device)
    q = A.paged_store(x, k, v, table, lens, n_head=1, rope_mode=2)
    assert torch.equal(q, x[:, :64]) and torch.equal(k.view(-1, 64)[:n], x[:, 64:128]) and torch.equal(v.view(-1, 64)[:n], x[:, 128:])
    assert (k.view(-1, 64)[n:] == 0).all()
    A.paged_store(x, wide[0], wide[1], table, lens, n_head=1, rope_mode=2, want_q=False)
    assert torch.equal(wide[0, -1, (n - 1) % 4096, 0], x[-1, 64:128])


def test_store_leaves_out_what_has_no_place(device):
    """Rows whose page is none, whose length passes the table or whose position is below 0 are not stored; their queries are."""
    g = gen(12)
    c = Cache(g, [20, 20, 20, 20], 2, 64, 16, F16, garbage=0.0)
    c.table[0, 1] = c.k.shape[0]  # one past the pool
    c.table[1, 1] = -1
    lens = torch.tensor([20, 20, 49, 2], dtype=torch.int32, device=device)  # the table holds 3 pages; 4 new rows of 2 keys
    k, v, table, _ = c.to(device)
    k0, v0 = k.clone(), v.clone()
    x = torch.randn(16, (4 + 4) * 64, generator=g)
    q = A.paged_store(x.to(device), k, v, table, lens, n_head=4, rope_mode=2)
    close(q, x[:, :256].double(), U[F16] * x[:, :256].double().abs() + TINY[F16], "q")
    for got, was, col in ((k, k0, 256), (v, v0, 384)):
        want = was.clone()
        new = x[:, col:col + 128].view(16, 2, 64).to(F16).to(device)
        for t in (14, 15):  # the last two rows of sequence 3 are its keys 0 and 1
            want[table[3, 0].long(), t - 14] = new[t]
        assert torch.equal(got, want)


# ---- decode ----

def decode_case(device, seed, n_head, n_kv, hd, lens, page, dtype, n_q=1, causal=True, scale=None, out_dtype=None, heads_first=False,
                pad=0, max_kv_len=None, ws=None, mutate=None, q_std=1.0, what=""):
    g = gen(seed)
    c = Cache(g, lens, n_kv, hd, page, dtype, heads_first=heads_first)
    if mutate:
        mutate(c)
    q = (torch.randn(len(lens) * n_q, n_head * hd, generator=g) * q_std).to(dtype)
    od = out_dtype or dtype
    dev_q, out = q.to(device), torch.full((q.shape[0], n_head * hd), 3.0, dtype=od, device=device)
    if pad:
        dev_q, out = padded(dev_q, pad), padded(out, pad)
    k, v, table, kv_len = c.to(device)
    o, lse = A.paged_decode(dev_q, k, v, table, kv_len, n_head=n_head, n_q=n_q, causal=causal, scale=scale, out=out, want_lse=True,
                            max_kv_len=max_kv_len, workspace=ws)
    sc = 1 / math.sqrt(hd) if scale is None else scale
    ref, rlse, tol, ltol = attend(c, q, [n_q] * len(lens), n_head, sc, causal, False, od)
    close(o, ref, tol, f"{what} out")
    close(lse, rlse, ltol, f"{what} lse")
    return o


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 14, 2), (64, 3, 3), (128, 28, 4), (128, 32, 8), (256, 8, 1)])
@pytest.mark.parametrize("n_q", [1, 3])
def test_decode_types(device, hd, n_head, n_kv, n_q, dtype):
    decode_case(device, 20, n_head, n_kv, hd, [3, 16, 129, 700, 33], 16, dtype, n_q=n_q)
    decode_case(device, 21, n_head, n_kv, hd, [1500], 64, dtype, n_q=n_q, out_dtype=F32)


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("heads_first", [False, True])
def test_decode_pages(device, page, heads_first):
    """Lengths either side of pages, blocks of 32 keys and splits."""
    decode_case(device, 22, 8, 2, 128, [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 511, 513], page, F16, heads_first=heads_first)


@pytest.mark.parametrize("lens", [[0], [0, 0, 5], [1], [2, 0, 1, 300, 0]])
@pytest.mark.parametrize("n_q,causal", [(1, True), (4, True), (4, False)])
def test_decode_empty_rows(device, lens, n_q, causal):
    """Sequences without keys, and causal rows at positions below 0: zeros and -inf."""
    decode_case(device, 23, 4, 2, 64, lens, 16, F16, n_q=n_q, causal=causal)


@pytest.mark.parametrize("n_q", [1, 2, 8, 40])
@pytest.mark.parametrize("causal", [True, False])
def test_decode_rows(device, n_q, causal):
    """One to many row tiles a kv head, at groups that do not divide them."""
    decode_case(device, 24, 7, 1, 128, [50, 800], 32, BF16, n_q=n_q, causal=causal)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_decode_scale(device, scale):
    decode_case(device, 25, 4, 2, 128, [40, 300], 16, F16, n_q=2, scale=scale)


def test_decode_strides(device):
    decode_case(device, 26, 4, 2, 128, [40, 300], 16, F16, n_q=2, pad=40)
    decode_case(device, 26, 4, 2, 64, [40, 300], 16, BF16, out_dtype=F32, pad=8)


@pytest.mark.parametrize("max_kv_len", [None, 1, 4000])
def test_decode_long(device, max_kv_len):
    """Many splits, whatever the hint says of the length."""
    decode_case(device, 27, 8, 8, 128, [4000], 16, F16, max_kv_len=max_kv_len)
    decode_case(device, 28, 14, 2, 64, [9000, 100], 64, BF16, max_kv_len=max_kv_len)


@pytest.mark.parametrize("longest", [100, 400])
def test_decode_thousands_of_sequences(device, longest):
    lens = [(b * 37) % 90 for b in range(4500)]
    lens[7], lens[4499] = longest, longest - 3
    decode_case(device, 36, 4, 2, 64, lens, 16, F16)


@pytest.mark.parametrize("n_seq,n_q", [(65, 1), (130, 2), (700, 1)])
def test_decode_many_sequences(device, n_seq, n_q):
    """More sequences than lanes, some empty, one long one among them."""
    lens = [(b * 37) % 90 for b in range(n_seq)]
    lens[n_seq // 2] = 3000
    decode_case(device, 29, 4, 2, 64, lens, 16, F16, n_q=n_q)


@pytest.mark.parametrize("max_kv_len", [None, 100, 600, 3000, 1 << 20])
@pytest.mark.parametrize("hd,n_head,n_kv,n_q", [(64, 4, 2, 1), (64, 14, 2, 1), (64, 14, 2, 2), (64, 14, 2, 7), (128, 8, 2, 1), (128, 7, 1, 1),
                                                (128, 16, 1, 1), (128, 28, 4, 4), (256, 4, 2, 1), (256, 16, 2, 3)])
def test_decode_plans(device, hd, n_head, n_kv, n_q, max_kv_len):
    """Every way of cutting a launch (whole sequences, chunks planned by the host or from the lengths, ranges) at every tile of rows:
    the hint chooses it and may not change the result, however wrong."""
    decode_case(device, 34, n_head, n_kv, hd, [1300, 40, 0, 513, 257, 1, 700], 32, F16, n_q=n_q, max_kv_len=max_kv_len)


@pytest.mark.parametrize("hd,n_head,n_kv,n_q", [(64, 14, 2, 1), (64, 14, 2, 3), (64, 8, 1, 4), (128, 32, 8, 1), (128, 7, 1, 2), (128, 28, 4, 5),
                                                (256, 8, 2, 1), (256, 16, 1, 2)])
def test_decode_ranges(device, hd, n_head, n_kv, n_q):
    """Batches cut into ranges of all sequences' keys, more sequences than lanes, with empty ones and a length that is none."""
    lens = [(b * 53) % 400 for b in range(150)]
    lens[10], lens[70], lens[149] = 2100, 0, 1500
    decode_case(device, 35, n_head, n_kv, hd, lens, 16, BF16, n_q=n_q)


def test_decode_shared_pages(device):
    """Sequences that share a prefix's pages."""
    def share(c):
        c.table[1, :4] = c.table[0, :4]
    decode_case(device, 30, 4, 2, 128, [100, 90, 70], 16, F16, mutate=share)


def poke(b, pos, g, d, value, which="v"):
    def f(c):
        getattr(c, which)[c.table[b, pos // c.page].long(), pos % c.page, g, d] = value
    return f


@pytest.mark.parametrize("value", [math.inf, -math.inf, NAN])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_odd_values_in_masked_places(device, value, dtype):
    """A value (or key) that later rows see is an infinity or NaN: earlier rows do not know of it."""
    for hd in (64, 128):
        for L in (70, 64, 500):
            decode_case(device, 31, 4, 2, hd, [L, 40], 16, dtype, n_q=4, mutate=poke(0, L - 2, 1, 17, value), what=f"{hd} {L}")
            if math.isnan(value):
                decode_case(device, 31, 4, 2, hd, [L, 40], 16, dtype, n_q=4, mutate=poke(0, L - 1, 1, 17, value, "k"))


def test_decode_wide_scores(device):
    """Scores hundreds apart, of either sign: the running maximum carries them."""
    decode_case(device, 32, 4, 2, 128, [700, 90], 16, BF16, q_std=30.0)


@pytest.mark.parametrize("kind", ["past", "negative", "length", "negative length"])
def test_decode_bad_metadata(device, kind):
    """A page or length that is none makes the sequence's outputs NaN, in every split, and nothing else."""
    g = gen(33)
    c = Cache(g, [600, 600, 50], 2, 128, 16, F16)
    k, v, table, kv_len = c.to(device)
    q = torch.randn(3, 4 * 128, generator=g).to(F16).to(device)
    good, _ = A.paged_decode(q, k, v, table, kv_len, n_head=4)
    if kind == "past":
        table[1, 30] = k.shape[0]
    elif kind == "negative":
        table[1, 3] = -5
    else:
        kv_len[1] = table.shape[1] * 16 + 1 if kind == "length" else -1
    out, lse = A.paged_decode(q, k, v, table, kv_len, n_head=4, want_lse=True)
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    ref, rlse, tol, ltol = attend(c, q.cpu(), [1, 1, 1], 4, 128 ** -0.5, True, False, F16)
    for b in (0, 2):
        close(out[b:b + 1], ref[b:b + 1], tol[b:b + 1], f"sequence {b}")
    close(good, ref, tol, "good")


def test_decode_workspace_of_other_shapes(device):
    """One workspace for calls of every shape, and for the contiguous caches' calls: each leaves it ready for the next."""
    ws = A.new_workspace(64 << 20, device)
    for i in range(3):
        decode_case(device, 40 + i, 8, 8, 128, [3000], 16, F16, ws=ws)
        decode_case(device, 50 + i, 28, 4, 128, [2000, 300, 9], 32, BF16, n_q=5, ws=ws)
        decode_case(device, 60 + i, 14, 2, 64, [1000] * 9, 64, F16, ws=ws)
        kc = torch.randn(2000, 8 * 128, device=device).to(F16)
        q = torch.randn(1, 32 * 128, device=device).to(F16)
        a, _ = A.decode(q, [kc], [kc], [2000], n_head=32, n_head_kv=8, head_dim=128, workspace=ws)
        b, _ = A.decode(q, [kc], [kc], [2000], n_head=32, n_head_kv=8, head_dim=128)
        assert torch.equal(a, b)


def test_decode_same_bits(device):
    """The order in which splits finish does not reach the result."""
    g = gen(70)
    c = Cache(g, [5000, 1234], 8, 128, 16, BF16)
    k, v, table, kv_len = c.to(device)
    q = torch.randn(2, 32 * 128, generator=g).to(BF16).to(device)
    ws = A.new_workspace(64 << 20, device)
    first = A.paged_decode(q, k, v, table, kv_len, n_head=32, workspace=ws)[0]
    for _ in range(20):
        assert torch.equal(first, A.paged_decode(q, k, v, table, kv_len, n_head=32, workspace=ws)[0])


# ---- prefill ----

def prefill_case(device, seed, n_head, n_kv, hd, rows, lens, page, dtype, causal=True, scale=None, out_dtype=None, heads_first=False, pad=0,
                 tail=0, mutate=None, max_q=None, max_kv_len=None, q_std=1.0, ws=None, what=""):
    g = gen(seed)
    c = Cache(g, lens, n_kv, hd, page, dtype, heads_first=heads_first)
    if mutate:
        mutate(c)
    total = sum(rows)
    q = (torch.randn(total + tail, n_head * hd, generator=g) * q_std).to(dtype)
    od = out_dtype or dtype
    dev_q, out = q.to(device), torch.full((total + tail, n_head * hd), 3.0, dtype=od, device=device)
    lse = torch.full((total + tail, n_head), 5.0, device=device)
    if pad:
        dev_q, out = padded(dev_q, pad), padded(out, pad)
    k, v, table, kv_len = c.to(device)
    A.paged_prefill(dev_q, k, v, table, kv_len, cu_of(rows, device), n_head=n_head, causal=causal, scale=scale, out=out, lse=lse,
                    max_q=max_q, max_kv_len=max_kv_len, workspace=ws)
    sc = 1 / math.sqrt(hd) if scale is None else scale
    ref, rlse, tol, ltol = attend(c, q, rows, n_head, sc, causal, True, od)
    close(out[:total], ref, tol, f"{what} out")
    close(lse[:total], rlse, ltol, f"{what} lse")
    if tail:
        assert (out[total:] == 3.0).all() and (lse[total:] == 5.0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 14, 2), (64, 3, 3), (128, 7, 1), (128, 8, 8), (256, 4, 2)])
def test_prefill_types(device, hd, n_head, n_kv, dtype):
    prefill_case(device, 80, n_head, n_kv, hd, [5, 70, 1, 0, 300], [5, 200, 40, 9, 300], 16, dtype, tail=3)
    prefill_case(device, 81, n_head, n_kv, hd, [100, 33], [100, 400], 64, dtype, out_dtype=F32)


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_pages(device, page, heads_first, hd):
    rows = [1, 15, 17, 31, 33, 63, 65, 127, 129, 257]
    prefill_case(device, 82, 4, 2, hd, rows, [r + 16 * (i % 3) for i, r in enumerate(rows)], page, F16, heads_first=heads_first)


@pytest.mark.parametrize("max_q", [None, 1, 4096])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 8, 2), (64, 64, 8), (128, 8, 2), (128, 48, 4)])
def test_prefill_plans(device, hd, n_head, n_kv, max_q):
    """Few and many workgroups, whatever the hint says of the rows: every workgroup shape and both tile orders."""
    prefill_case(device, 83, n_head, n_kv, hd, [600, 130, 20, 1], [650, 130, 900, 77], 32, F16, max_q=max_q)


@pytest.mark.parametrize("hd,n_head,n_kv,dtype", [(128, 8, 2, F16), (64, 7, 1, BF16), (128, 4, 4, BF16), (256, 2, 1, F16)])
def test_prefill_split_tiles(device, hd, n_head, n_kv, dtype):
    """A few rows behind many keys: every tile is cut over many workgroups; with a workspace and without one."""
    for ws in (None, torch.empty(0, dtype=torch.uint8, device=device)):
        prefill_case(device, 93, n_head, n_kv, hd, [70, 3, 200], [5000, 9000, 2000], 64, dtype, ws=ws, what=f"ws {ws is not None}")


@pytest.mark.parametrize("n_head,n_kv,hd", [(32, 8, 128), (28, 4, 128), (14, 2, 64), (16, 16, 64)])
def test_prefill_ranges(device, n_head, n_kv, hd):
    """More tiles than workgroups: ranges that begin and end within tiles, sequences and kv heads."""
    prefill_case(device, 94, n_head, n_kv, hd, [700, 33, 0, 512, 1, 900], [1000, 33, 7, 512, 800, 900], 16, BF16)


def test_prefill_same_bits(device):
    """Split tiles are joined in order, whichever workgroup is last; the workspace serves call after call, of any shape."""
    g = gen(95)
    ws = A.new_workspace(A.paged_prefill_workspace_bytes(n_head=28, n_head_kv=4, head_dim=128, n_rows=1, n_seq=1, max_q=1, max_kv_len=1), device)
    cases = []
    for rows, lens, n_head, n_kv in (([300, 100], [6000, 3000], 28, 4), ([800, 10], [800, 4000], 32, 8)):
        c = Cache(g, lens, n_kv, 128, 32, BF16)
        q = torch.randn(sum(rows), n_head * 128, generator=g).to(BF16).to(device)
        cases.append((q, *c.to(device), cu_of(rows, device), n_head))
    first = [A.paged_prefill(*c[:-1], n_head=c[-1], workspace=ws)[0] for c in cases]
    for _ in range(10):
        for c, f in zip(cases, first):
            assert torch.equal(f, A.paged_prefill(*c[:-1], n_head=c[-1], workspace=ws)[0])


def test_prefill_many_sequences(device):
    rows = [(b * 7) % 40 for b in range(150)]
    prefill_case(device, 84, 4, 2, 64, rows, [r + (b % 5) * 11 for b, r in enumerate(rows)], 16, BF16)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefill_rows_without_keys(device, hd):
    """More rows than keys (the first ones are at positions below 0), and sequences without keys."""
    prefill_case(device, 85, 4, 2, hd, [40, 70, 33, 5], [3, 0, 33, 70], 16, F16)


def test_prefill_not_causal(device):
    for hd in (64, 128, 256):
        prefill_case(device, 86, 4, 2, hd, [40, 70, 3, 200], [100, 20, 0, 200], 16, F16, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_prefill_scale(device, scale):
    prefill_case(device, 87, 4, 2, 128, [40, 150], [40, 300], 16, F16, scale=scale)


def test_prefill_strides(device):
    prefill_case(device, 88, 4, 2, 128, [40, 150], [40, 300], 16, F16, pad=40)
    prefill_case(device, 88, 4, 2, 64, [40, 150], [40, 300], 16, BF16, pad=8, out_dtype=F32)


@pytest.mark.parametrize("value", [math.inf, -math.inf, NAN])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefill_odd_values_in_masked_places(device, value, dtype, hd):
    """Rows before an infinity or NaN do not know of it, in the same tile or another."""
    prefill_case(device, 89, 4, 2, hd, [100, 40], [130, 40], 16, dtype, mutate=poke(0, 101, 1, 17, value))
    prefill_case(device, 89, 4, 2, hd, [100, 40], [130, 40], 16, dtype, mutate=poke(0, 129, 0, 63, value))
    if math.isnan(value):
        prefill_case(device, 89, 4, 2, hd, [100, 40], [130, 40], 16, dtype, mutate=poke(0, 101, 1, 17, value, "k"))


def test_prefill_wide_scores(device):
    prefill_case(device, 90, 4, 2, 128, [300, 90], [300, 500], 16, BF16, q_std=30.0)
    prefill_case(device, 90, 4, 2, 64, [300, 90], [300, 500], 16, F16, q_std=30.0)


@pytest.mark.parametrize("kind", ["past", "negative", "length", "negative length"])
def test_prefill_bad_metadata(device, kind):
    g = gen(91)
    c = Cache(g, [300, 300, 50], 2, 128, 16, F16)
    k, v, table, kv_len = c.to(device)
    rows = [200, 200, 50]
    q = torch.randn(450, 4 * 128, generator=g).to(F16).to(device)
    if kind == "past":
        table[1, 2] = k.shape[0]
    elif kind == "negative":
        table[1, 0] = -1
    else:
        kv_len[1] = table.shape[1] * 16 + 1 if kind == "length" else -1
    out, lse = A.paged_prefill(q, k, v, table, kv_len, cu_of(rows, device), n_head=4, want_lse=True)
    assert torch.isnan(out[200:400]).all() and torch.isnan(lse[200:400]).all()
    ref, rlse, tol, ltol = attend(c, q.cpu(), rows, 4, 128 ** -0.5, True, True, F16)
    for s in (slice(0, 200), slice(400, 450)):
        close(out[s], ref[s], tol[s], "others")


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [0, 40, 61])
def test_prefill_bad_page_and_odd_values(device, hd, bad):
    """A page that is none in one part of a split tile, and an infinity among the values that only the last rows see."""
    g = gen(95)
    c = Cache(g, [4000, 90], 1, hd, 64, F16)
    c.v[c.table[0, 3995 // 64].long(), 3995 % 64, 0, 5] = float("inf")
    k, v, table, kv_len = c.to(device)
    table[0, bad] = -7
    q = torch.randn(60, 2 * hd, generator=g).to(F16).to(device)
    out, lse = A.paged_prefill(q, k, v, table, kv_len, cu_of([30, 30], device), n_head=2, want_lse=True)
    assert torch.isnan(out[:30]).all() and torch.isnan(lse[:30]).all()
    ref, _, tol, _ = attend(c, q.cpu(), [30, 30], 2, hd ** -0.5, True, True, F16)
    close(out[30:], ref[30:], tol[30:], "the other sequence")


@pytest.mark.parametrize("cu", [[0, 999, 999], [0, -5, 30], [20, 10, 30], [0, 60, 2 ** 31 - 1]])
def test_prefill_odd_ranges_stay_inside(device, cu):
    """Ranges of rows that pass the rows or run backwards: the call reads and writes its own rows only."""
    g = gen(92)
    c = Cache(g, [60, 60], 2, 64, 16, F16)
    k, v, table, kv_len = c.to(device)
    q = torch.randn(60, 4 * 64, generator=g).to(F16).to(device)
    room = torch.full((100, 4 * 64), 3.0, dtype=F16, device=device)
    A.paged_prefill(q, k, v, table, kv_len, torch.tensor(cu, dtype=torch.int32, device=device), n_head=4, out=room[20:80])
    assert (room[:20] == 3.0).all() and (room[80:] == 3.0).all()


# ---- together ----

def chain(device, steps, prompts, hd=128, n_head=8, n_kv=2, page=16, seed=100):
    """Prompts and decode steps through projection, store and attention; the outputs, and those of the contiguous caches."""
    g = gen(seed)
    width = n_head * hd
    w = (torch.randn((n_head + 2 * n_kv) * hd, width, generator=g) * width ** -0.5).to(F16).to(device)
    x = [torch.randn(n + steps, width, generator=g).to(device) for n in prompts]
    total = [n + steps for n in prompts]
    used = [-(-n // page) for n in total]
    k = torch.full((sum(used), page, n_kv, hd), NAN, dtype=F16, device=device)
    v = torch.full_like(k, NAN)
    ids = torch.randperm(sum(used), generator=g).to(torch.int32)
    table = torch.zeros(len(prompts), max(used), dtype=torch.int32)
    for b, n in enumerate(used):
        table[b, :n] = ids[sum(used[:b]):sum(used[:b]) + n]
    table = table.to(device)
    lens = torch.tensor(prompts, dtype=torch.int32, device=device)
    out = []
    packed = torch.cat([t[:n] for t, n in zip(x, prompts)])
    cu = cu_of(prompts, device)
    rope = dict(n_head=n_head, rope_mode=1, rope_base=1e6)
    q = A.paged_store(A.linear(packed, w), k, v, table, lens, cu_q=cu, **rope)
    out.append(A.paged_prefill(q, k, v, table, lens, cu, n_head=n_head, out_dtype=F32)[0])
    for s in range(steps):
        lens += 1
        q = A.paged_store(A.linear(torch.stack([t[n + s] for t, n in zip(x, prompts)]), w), k, v, table, lens, **rope)
        out.append(A.paged_decode(q, k, v, table, lens, n_head=n_head, out_dtype=F32)[0])
    ref_prompt, ref_steps = [], [[] for _ in range(steps)]
    heads = dict(n_head=n_head, n_head_kv=n_kv, head_dim=hd, rope_mode=1, rope_base=1e6)
    for t, n in zip(x, prompts):
        kc = torch.zeros(n + steps, n_kv * hd, dtype=F16, device=device)
        vc = torch.zeros_like(kc)
        ref_prompt.append(A.prefill_rope(A.linear(t[:n], w), kc[:n], vc[:n], **heads)[0])
        for s in range(steps):
            ref_steps[s].append(A.decode_rope(A.linear(t[n + s:n + s + 1], w), [kc], [vc], [n + s + 1], **heads)[0])
    return out, [torch.cat(ref_prompt)] + [torch.cat(r) for r in ref_steps]


def test_chain_against_the_contiguous_caches(device):
    """A run as a decoder makes it: the packed prompts and three steps, against the same through the contiguous caches. Both
    round the query, keys and probabilities to half (angles in 64 and 32 bits apart), so they agree to a few half steps of the
    values."""
    got, ref = chain(device, 3, [37, 200, 5, 130])
    for a, b in zip(got, ref):
        assert float((a - b).abs().max()) <= 2e-3 + 1e-2 * float(b.abs().max())  # the contiguous calls' own tolerance


def test_graph_replays_as_lengths_grow(device):
    """A captured step (append and attention) replayed while the sequences grow, one of them to more splits, with eager work
    between the replays: each replay against the eager calls."""
    g = gen(110)
    n_head, n_kv, hd, page = 8, 2, 128, 16
    lens = [250, 3, 0, 1020]
    c = Cache(g, lens, n_kv, hd, page, BF16, spare=40, extra_width=8)
    for b in range(4):
        used = -(-lens[b] // page)
        c.table[b, used:used + 8] = c.free[8 * b:8 * b + 8]
    k, v, table, kv_len = c.to(device)
    x = torch.zeros(4, (n_head + 2 * n_kv) * hd, device=device)
    q = torch.empty(4, n_head * hd, dtype=BF16, device=device)
    out = torch.empty(4, n_head * hd, dtype=BF16, device=device)
    ws = A.new_workspace(A.paged_decode_workspace_bytes(n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_q=1, n_seq=4, max_kv_len=2048), device)

    def step(k, v, q, out, ws):
        A.paged_store(x, k, v, table, kv_len, n_head=n_head, rope_mode=0, q=q)
        A.paged_decode(q, k, v, table, kv_len, n_head=n_head, max_kv_len=2048, out=out, workspace=ws)

    ws2 = ws.clone()
    k2, v2 = k.clone(), v.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(k2.clone(), v2.clone(), q, out, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(k, v, q, out, ws)
    for i in range(12):
        x.copy_(torch.randn(x.shape, generator=g))
        kv_len += torch.tensor([1, 1, 1 if i > 3 else 0, 5], dtype=torch.int32, device=device)
        if i > 2:
            kv_len[1] = 0 if i == 6 else i + 4
        graph.replay()
        torch.cuda.synchronize()
        q2, out2 = torch.empty_like(q), torch.empty_like(out)
        step(k2, v2, q2, out2, ws2)
        torch.cuda.synchronize()
        assert torch.equal(q, q2) and torch.equal(out.nan_to_num(9.0), out2.nan_to_num(9.0)), i
        assert torch.equal(k.nan_to_num(9.0), k2.nan_to_num(9.0))


def test_prefill_graph_replays(device):
    g = gen(111)
    c = Cache(g, [300, 90, 40], 2, 128, 16, F16)
    k, v, table, kv_len = c.to(device)
    q = torch.randn(200, 8 * 128, generator=g).to(F16).to(device)
    cu = cu_of([100, 90, 10], device)
    need = A.paged_prefill_workspace_bytes(n_head=8, n_head_kv=2, head_dim=128, n_rows=200, n_seq=3, max_q=0, max_kv_len=0)
    ws, ws2 = A.new_workspace(max(need, 1 << 20), device), A.new_workspace(max(need, 1 << 20), device)
    out = torch.zeros(200, 8 * 128, dtype=F16, device=device)
    A.paged_prefill(q, k, v, table, kv_len, cu, n_head=8, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.paged_prefill(q, k, v, table, kv_len, cu, n_head=8, out=out, workspace=ws)
    for rows, lens in (([100, 90, 10], [300, 90, 40]), ([1, 60, 7], [300, 70, 8]), ([0, 200, 0], [10, 200, 0])):
        cu.copy_(cu_of(rows, device))
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        if lens[1] == 200:
            table[1, :13] = table[0, :13]
        for _ in range(3):
            out.fill_(3.0)
            graph.replay()
            ref = torch.full_like(out, 3.0)
            A.paged_prefill(q, k, v, table, kv_len, cu, n_head=8, out=ref, workspace=ws2)
            torch.cuda.synchronize()
            assert torch.equal(out, ref)


class _General:
    """An extension that takes no call: the general path runs."""

    def __getattr__(self, name):
        return lambda *a: None


def test_extension_and_general_path(device, monkeypatch):
    """The torch extension takes ordinary calls itself, and gives the bits of the general path."""
    g = gen(114)
    ext, taken = A._native(), []

    class Counted:
        def __getattr__(self, name):
            def call(*a):
                r = getattr(ext, name)(*a)
                taken.append(r is not None)
                return r
            return call

    lens, rows, n_head, n_kv, hd = [300, 20, 77], [100, 20, 1], 8, 2, 64
    cu = cu_of(rows, device)
    pos = torch.randint(0, 500, (2, 121), generator=g).to(torch.int32).to(device)
    x = torch.randn(121, (n_head + 2 * n_kv) * hd, generator=g).to(device)
    ws = A.new_workspace(A.paged_prefill_workspace_bytes(n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_rows=121, n_seq=3, max_q=100,
                                                         max_kv_len=400), device)
    results = []
    for native in (Counted(), _General()):
        monkeypatch.setattr(A, "_native", lambda n=native: n)
        c = Cache(gen(115), lens, n_kv, hd, 16, BF16)
        k, v, table, kv_len = c.to(device)
        where = (k, v, table, kv_len)
        q = A.paged_store(x, *where, n_head=n_head, rope_mode=1, cu_q=cu, positions=pos, axis_pairs=(20, 12), axis_restart=True)
        o, lse = A.paged_prefill(q, *where, cu, n_head=n_head, want_lse=True, max_q=100, workspace=ws)
        o32, _ = A.paged_prefill(q, *where, cu, n_head=n_head, out_dtype=F32, causal=False, scale=0.3, workspace=ws)
        d, dl = A.paged_decode(q[:6], *where, n_head=n_head, n_q=2, want_lse=True, max_kv_len=400, workspace=ws)
        into = torch.zeros(6, n_head * hd + 8, dtype=BF16, device=device)
        assert A.paged_decode(q[:6], *where, n_head=n_head, n_q=2, out=into, workspace=ws)[0] is into
        results.append([q, k, v, o, lse, o32, d, dl, into])
    assert taken == [True] * 5
    for a, b in zip(*results):
        assert a.dtype == b.dtype and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_front_end_refusals(device):
    c = Cache(gen(116), [40, 40], 2, 64, 16, F16)
    k, v, table, kv_len = c.to(device)
    q = torch.zeros(2, 256, dtype=F16, device=device)
    x = torch.zeros(2, 512, device=device)
    cu = cu_of([1, 1], device)
    ws = A.new_workspace(64 << 20, device)
    bad = [dict(q=q.to(BF16)), dict(q=q.float()), dict(q=q[:, :128]), dict(q=q.cpu()), dict(q=q.t()), dict(v=v.to(BF16)), dict(v=v[:1]),
           dict(k=k.cpu()), dict(k=k.transpose(2, 3)), dict(table=table.long()), dict(table=table[0]), dict(table=table.cpu()), dict(table=table[:1].expand(2, -1)), dict(kv_len=kv_len[:1]),
           dict(kv_len=kv_len.long()), dict(kv_len=kv_len.cpu())]
    for wrong in bad:
        a = dict(dict(q=q, k=k, v=v, table=table, kv_len=kv_len), **wrong)
        for w in (None, ws):
            with pytest.raises(ValueError):
                A.paged_decode(a["q"], a["k"], a["v"], a["table"], a["kv_len"], n_head=4, workspace=w)
            with pytest.raises(ValueError):
                A.paged_prefill(a["q"], a["k"], a["v"], a["table"], a["kv_len"], cu, n_head=4, workspace=w)
        if "q" not in wrong:
            with pytest.raises(ValueError):
                A.paged_store(x, a["k"], a["v"], a["table"], a["kv_len"], n_head=4, rope_mode=0)
    for w in (None, ws):
        with pytest.raises(ValueError, match="cu_q"):
            A.paged_prefill(q, k, v, table, kv_len, cu.long(), n_head=4, workspace=w)
        with pytest.raises(ValueError, match="cu_q"):
            A.paged_prefill(q, k, v, table, kv_len, None, n_head=4, workspace=w)
        with pytest.raises(ValueError, match="out"):
            A.paged_decode(q, k, v, table, kv_len, n_head=4, out=q.to(BF16), workspace=w)
        with pytest.raises(ValueError, match="lse"):
            A.paged_decode(q, k, v, table, kv_len, n_head=4, lse=torch.zeros(2, 3, device=device), workspace=w)
        with pytest.raises(ValueError, match="rows"):
            A.paged_decode(q, k, v, table, kv_len, n_head=4, n_q=2, workspace=w)
    with pytest.raises(_lib.MxAttnError):
        wide = torch.cat([table, table.new_zeros(2, 200)], dim=1)  # room for sequences that are split, which needs a workspace
        A.paged_decode(q, k, v, wide, kv_len, n_head=4, workspace=ws[:1 << 19])
    for wrong in (dict(positions=torch.zeros(2, 2, dtype=torch.int32, device=device)), dict(positions=torch.zeros(2, device=device)),
                  dict(axis_pairs=(16, 8)), dict(axis_pairs=(16, 16)), dict(q=q.to(BF16)), dict(rope_mode=3), dict(rope_base=0.5)):
        with pytest.raises((ValueError, _lib.MxAttnError)):
            A.paged_store(x, k, v, table, kv_len, **dict(dict(n_head=4, rope_mode=0), **wrong))
    with pytest.raises(ValueError, match="qkv"):
        A.paged_store(x[:, :448], k, v, table, kv_len, n_head=4, rope_mode=0)


def test_two_streams(device):
    """Calls on two streams, each with its own workspace and outputs, over one pool."""
    g = gen(112)
    c = Cache(g, [4000, 900], 8, 128, 16, F16)
    k, v, table, kv_len = c.to(device)
    qs = [torch.randn(2, 32 * 128, generator=g).to(F16).to(device) for _ in range(2)]
    ref = [A.paged_decode(q, k, v, table, kv_len, n_head=32)[0] for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    spaces = [A.new_workspace(64 << 20, device) for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(A.paged_decode(qs[i], k, v, table, kv_len, n_head=32, workspace=spaces[i])[0])
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, ref[i])


def test_far_pages(device):
    """A pool beyond 2^32 bytes: offsets of its last pages pass 32 bits."""
    hd, page, n_pages = 128, 256, 9000
    k = torch.empty(n_pages, page, 8, hd, dtype=F16, device=device)
    v = torch.empty_like(k)
    g = gen(113)
    small = Cache(g, [400], 8, hd, page, F16)
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device=device)
    for i in range(2):
        k[n_pages - 1 - i] = small.k[small.table[0, i].long()].to(device)
        v[n_pages - 1 - i] = small.v[small.table[0, i].long()].to(device)
    kv_len = torch.tensor([400], dtype=torch.int32, device=device)
    q = torch.randn(64, 8 * hd, generator=g).to(F16)
    o, _ = A.paged_prefill(q.to(device), k, v, table, kv_len, cu_of([64], device), n_head=8)
    ref, _, tol, _ = attend(small, q, [64], 8, hd ** -0.5, True, True, F16)
    close(o, ref, tol, "prefill")
    o, _ = A.paged_decode(q[63:].to(device), k, v, table, kv_len, n_head=8)
    ref, _, tol, _ = attend(small, q[63:], [1], 8, hd ** -0.5, True, False, F16)
    close(o, ref, tol, "decode")
    x = torch.randn(1, 24 * hd, generator=g)
    kv_len += 1
    A.paged_store(x.to(device), k, v, table, kv_len, n_head=8, rope_mode=2, want_q=False)
    assert torch.equal(v[n_pages - 2, 400 - page].cpu().flatten(), x[0, 16 * hd:].to(F16))
