"""The paged cache in 8 bits: its kernels against their definitions in 64 bits (e4m3_helpers.py, paged_helpers.py).

The append's codes and scales are held to the definition itself: a key x that the kernel rotates in 64 bits is off by at most d of its
two products (none without rotation), and rounding is monotone, so the scale lies between those of the largest magnitude less and plus
d, and the code between the roundings of x - d and x + d by that scale. d: a frequency is within 10 steps of 2^-53 of the power (the
ladder's 7 products, the power itself, the angle), here and below alike, so the angle of position p within p 2^-48, and the cosine and
the products within 2^-50."""
import math

import pytest
import torch

from dooms_amd import attention as A
from e4m3_helpers import E4M3, E8M0, Cache8, power, round_e4m3, scale_byte
from paged_helpers import TINY, U, attend, close, rotate
from test_paged_gpu import BF16, F16, F32, cu_of, gen, padded

pytestmark = pytest.mark.gpu


# ---- store ----

def check_rows(codes, scales, x, d, what):
    """codes [n][heads][hd] and scale bytes [n][heads] against values x off by at most d."""
    top, far = x.abs().amax(-1), d.amax(-1)
    lo, hi = scale_byte((top - far).clamp(min=0)), scale_byte(top + far)
    assert ((scales >= lo) & (scales <= hi)).all(), f"{what}: scales off"
    unit = power(scales)[..., None]
    got = codes.view(E4M3).double()
    a, b = round_e4m3((x - d) / unit), round_e4m3((x + d) / unit)
    bad = ~((got >= a) & (got <= b))
    assert not bad.any(), f"{what}: {int(bad.sum())} codes off, the first at {torch.nonzero(bad)[0].tolist()}"


def store_case(device, seed, n_head, n_kv, hd, rows, lens, page, dtype, in_dtype, mode, heads_first=False, scale_pad=0, pad=0, tail=0,
               uniform=False, x=None, base=1e4, positions=None, axis_pairs=None, restart=False, what=""):
    g = gen(seed)
    c = Cache8(g, lens, n_kv, hd, page, dtype, heads_first=heads_first, scale_pad=scale_pad)
    total = sum(rows)
    if x is None:
        x = torch.randn(total + tail, (n_head + 2 * n_kv) * hd, generator=g).to(in_dtype)
    q0 = torch.full((total + tail, n_head * hd), 7.0, dtype=dtype, device=device)
    dev_x = x.to(device)
    if pad:
        q0, dev_x = padded(q0, pad), padded(dev_x, pad)
    k, v, table, kv_len, scales = c.to(device)
    got = A.paged_store(dev_x, k, v, table, kv_len, n_head=n_head, rope_mode=mode, rope_base=base, cu_q=None if uniform else cu_of(rows, device),
                        q=q0, scales=scales, positions=None if positions is None else positions.to(device), axis_pairs=axis_pairs,
                        axis_restart=restart)
    assert got is q0
    pos = torch.cat([torch.arange(L - n, L) for n, L in zip(rows, lens)])[None] if positions is None else positions
    xr = x[:total].double().view(total, n_head + 2 * n_kv, hd)
    ref, mag = rotate(xr[:, :n_head + n_kv], pos, mode, base, axis_pairs or (hd // 2,), restart)
    far = pos.abs().double().amax(0)[:, None, None]
    off = (0.0 if mode == 2 else 2.0 ** -48 * (2 + far)) * mag
    tol = U[dtype] * ref.abs() + (0.0 if mode == 2 else 2.0 ** -21) * mag + TINY[dtype]
    close(got[:total], ref[:, :n_head].flatten(1), tol[:, :n_head].flatten(1), f"{what} q")
    if tail:
        assert (got[total:] == 7.0).all()
    at, touched = 0, torch.zeros(c.k.shape[:2], dtype=torch.bool)
    k8, v8, ks, vs = (t.view(torch.uint8).cpu() for t in (k, v, *scales))
    for b, (n, L) in enumerate(zip(rows, lens)):
        p = torch.arange(L - n, L)
        page_, row = c.table[b, p // page].long(), p % page
        touched[page_, row] = True
        check_rows(k8[page_, row].contiguous(), ks[page_, :, row], ref[at:at + n, n_head:], off[at:at + n, n_head:], f"{what} k {b}")
        check_rows(v8[page_, row].contiguous(), vs[page_, :, row], xr[at:at + n, n_head + n_kv:], torch.zeros(n, n_kv, hd, dtype=torch.float64), f"{what} v {b}")
        at += n
    for got8, was, s8, swas in ((k8, c.k, ks, c.ks), (v8, c.v, vs, c.vs)):
        assert torch.equal(got8[~touched], was[~touched]) and torch.equal(s8.transpose(1, 2)[~touched], swas.transpose(1, 2)[~touched])
    for s in scales:  # the bytes between the pages' rows
        if scale_pad:
            wide = s.view(torch.uint8).as_strided((*s.shape[:2], page + scale_pad), s.stride())
            assert (wide[..., page:] == 255).all()


@pytest.mark.parametrize("in_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 14, 2), (128, 28, 4), (256, 4, 1)])
def test_store_types(device, hd, n_head, n_kv, dtype, in_dtype):
    for mode in (0, 1, 2):
        store_case(device, 1 + mode, n_head, n_kv, hd, [3, 1, 0, 20], [40, 1, 17, 20], 16, dtype, in_dtype, mode, tail=2, what=f"mode {mode}")


@pytest.mark.parametrize("in_dtype", [F32, BF16])
@pytest.mark.parametrize("hd,heads_first,pad,uniform,scale_pad", [(128, True, 0, False, 0), (64, False, 24, True, 16), (256, True, 8, True, 48)])
def test_store_layouts(device, hd, heads_first, pad, uniform, scale_pad, in_dtype):
    store_case(device, 9, 4, 4, hd, [2, 2, 2], [2, 33, 700], 32, F16, in_dtype, 1, heads_first=heads_first, pad=pad, uniform=uniform,
               scale_pad=scale_pad)


def test_store_axes_and_many_sequences(device):
    g = gen(5)
    pos = torch.randint(-50, 5000, (3, 37), generator=g).to(torch.int32)
    store_case(device, 6, 8, 2, 128, [30, 7], [64, 300], 64, BF16, F32, 1, positions=pos, axis_pairs=(16, 24, 24), restart=True, base=1e6)
    store_case(device, 12, 2, 1, 64, [b % 3 for b in range(129)], [b % 3 + b % 20 for b in range(129)], 16, BF16, F16, 1, tail=2)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_store_magnitudes(device, hd):
    """Rows from the smallest numbers of f32 to the largest, of one sign, at and next to the borders of a scale, and all zeros."""
    g = gen(13)
    tops = [2.0 ** -149, 2.0 ** -130, 1e-30, 3.3e38, 448.0, 448.0000305, 449.0, 1.75, 0.875, 2.0 ** -119 * 1.75, 1e-3, 65504.0]
    n = len(tops) + 2
    x = torch.rand(n, 1 + 2, hd, generator=g) * 2 - 1
    for i, t in enumerate(tops):
        x[i] *= t / 2
        x[i, :, (5 * i) % hd] = t if i % 2 else -t
    x[-2] = 0
    x[-1] = 2.0 ** -149
    store_case(device, 14, 1, 1, hd, [n], [n], 16, BF16, F32, 2, x=x.flatten(1).float(), what="magnitudes")


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("in_dtype", [F32, F16, BF16])
def test_store_ties(device, hd, in_dtype):
    """Numbers half way between two codes go to the even one, over all of them."""
    codes = torch.arange(0, 0x7e, dtype=torch.uint8).view(E4M3).double()
    half = (codes[1:] + codes[:-1]) / 2
    x = torch.zeros(4, 3, hd, dtype=torch.float64)
    for i in range(4):
        pick = half[torch.arange(hd) * 4 % len(half)] if i % 2 else half[(torch.arange(hd) * 7 + 50 * i) % len(half)]
        x[i] = pick * torch.where(torch.arange(hd) % 2 == 0, 1.0, -1.0)
        x[i, :, i] = 448.0
    if in_dtype != F32:
        x = x.to(in_dtype).double()
    k, v = (torch.zeros(1, 16, 1, hd, dtype=E4M3, device=device) for _ in range(2))
    s = [torch.zeros(1, 1, 16, dtype=torch.uint8, device=device).view(E8M0) for _ in range(2)]
    A.paged_store(x.to(in_dtype).flatten(1).to(device), k, v, torch.zeros(1, 1, dtype=torch.int32, device=device),
                  torch.tensor([4], dtype=torch.int32, device=device), n_head=1, rope_mode=2, scales=s)
    for pool, scale, at in ((k, s[0], 1), (v, s[1], 2)):
        assert (scale.view(torch.uint8)[0, 0, :4] == 127).all()
        assert torch.equal(pool[0, :4, 0].double().cpu(), round_e4m3(x[:, at]))


@pytest.mark.parametrize("in_dtype", [F32, F16, BF16])
def test_store_infinities_and_nan(device, in_dtype):
    """They become NaN codes and leave the scale to the rest of the row; a row of them alone has the scale of zeros."""
    hd = 128
    x = torch.randn(3, 3, hd, generator=gen(15)).to(in_dtype)
    clean = x.clone()
    bad = torch.zeros(hd, dtype=torch.bool)
    bad[[0, 17, 64, 127]] = True
    x[0, 1:, bad] = torch.tensor([math.inf, -math.inf, math.nan, math.inf]).to(in_dtype)
    x[2] = math.inf
    k, v = (torch.zeros(1, 16, 1, hd, dtype=E4M3, device=device) for _ in range(2))
    s = [torch.zeros(1, 1, 16, dtype=torch.uint8, device=device).view(E8M0) for _ in range(2)]
    A.paged_store(x.flatten(1).to(device), k, v, torch.zeros(1, 1, dtype=torch.int32, device=device),
                  torch.tensor([3], dtype=torch.int32, device=device), n_head=1, rope_mode=2, scales=s)
    for pool, scale, at in ((k, s[0], 1), (v, s[1], 2)):
        byte, got = scale.view(torch.uint8)[0, 0, :3].cpu(), pool[0, :3, 0].double().cpu()
        want = torch.where(bad, 0.0, clean[0, at].double())
        assert byte.tolist() == [int(scale_byte(want.abs().amax())), int(scale_byte(clean[1, at].double().abs().amax())), 0]
        assert torch.isnan(got[0, bad]).all() and torch.isnan(got[2]).all()
        assert torch.equal(got[0, ~bad], round_e4m3(want / power(byte[0]))[~bad])


def test_store_leaves_out_what_has_no_place(device):
    g = gen(12)
    c = Cache8(g, [20, 20, 20, 20], 2, 64, 16, F16)
    c.table[0, 1] = c.k.shape[0]  # one past the pool
    c.table[1, 1] = -1
    lens = torch.tensor([20, 20, 49, 2], dtype=torch.int32, device=device)  # the table holds 3 pages; 4 new rows of 2 keys
    k, v, table, _, scales = c.to(device)
    x = torch.randn(16, (4 + 4) * 64, generator=g)
    q = A.paged_store(x.to(device), k, v, table, lens, n_head=4, rope_mode=2, scales=scales)
    assert q.dtype == F16
    close(q, x[:, :256].double(), U[F16] * x[:, :256].double().abs() + TINY[F16], "q")
    k8, v8, ks, vs = (t.view(torch.uint8).cpu() for t in (k, v, *scales))
    zero = torch.zeros(2, 64, dtype=torch.float64)
    for got, was, s8, swas, col in ((k8, c.k, ks, c.ks, 256), (v8, c.v, vs, c.vs, 384)):
        page = c.table[3, 0].long()
        for t in (14, 15):  # the last two rows of sequence 3 are its keys 0 and 1
            check_rows(got[page, t - 14][None], s8[page, :, t - 14][None], x[t, col:col + 128].double().view(1, 2, 64), zero[None], f"row {t}")
        got[page, :2], s8[page, :, :2] = was[page, :2], swas[page, :, :2]
        assert torch.equal(got, was) and torch.equal(s8, swas)


def test_store_without_queries_and_their_types(device):
    g = gen(16)
    c = Cache8(g, [9], 1, 64, 16, BF16)
    for in_dtype in (F32, F16, BF16):
        x = torch.randn(9, 4 * 64, generator=g).to(in_dtype).to(device)
        k, v, table, kv_len, scales = c.to(device)
        assert A.paged_store(x, k, v, table, kv_len, n_head=2, rope_mode=2, scales=scales, want_q=False) is None
        want = [t.clone() for t in (k.view(torch.uint8), v.view(torch.uint8))]
        for q_dtype in (None, F16, BF16):
            q = A.paged_store(x, k, v, table, kv_len, n_head=2, rope_mode=2, scales=scales, q_dtype=q_dtype)
            assert q.dtype == (q_dtype or (F16 if in_dtype == F32 else in_dtype))
            assert torch.equal(q, x[:, :128].to(q.dtype))
            assert torch.equal(k.view(torch.uint8), want[0]) and torch.equal(v.view(torch.uint8), want[1])


# ---- attention ----

def decode_case(device, seed, n_head, n_kv, hd, lens, page, dtype, n_q=1, causal=True, scale=None, out_dtype=None, heads_first=False,
                scale_pad=0, pad=0, max_kv_len=None, ws=None, mutate=None, width=0, what=""):
    g = gen(seed)
    c = Cache8(g, lens, n_kv, hd, page, dtype, heads_first=heads_first, scale_pad=scale_pad, extra_width=1 + width)
    if mutate:
        mutate(c)
    q = torch.randn(len(lens) * n_q, n_head * hd, generator=g).to(dtype)
    od = out_dtype or dtype
    dev_q, out = q.to(device), torch.full((q.shape[0], n_head * hd), 3.0, dtype=od, device=device)
    if pad:
        dev_q, out = padded(dev_q, pad), padded(out, pad)
    k, v, table, kv_len, scales = c.to(device)
    o, lse = A.paged_decode(dev_q, k, v, table, kv_len, n_head=n_head, n_q=n_q, causal=causal, scale=scale, out=out, want_lse=True,
                            max_kv_len=max_kv_len, scales=scales, workspace=ws)
    ref, rlse, tol, ltol = attend(c, q, [n_q] * len(lens), n_head, 1 / math.sqrt(hd) if scale is None else scale, causal, False, od)
    close(o, ref, tol, f"{what} out")
    close(lse, rlse, ltol, f"{what} lse")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 14, 2), (128, 28, 4), (128, 4, 4), (128, 8, 1), (256, 4, 1)])
def test_decode_lengths(device, hd, n_head, n_kv, dtype):
    """One key to many, a page that ends within a block, one sequence and ragged ones."""
    for lens in ([1], [2, 17, 31], [0, 33, 64, 100], [513], [1000, 5, 2047], [4096, 4095], [16385]):
        decode_case(device, 20, n_head, n_kv, hd, lens, 16, dtype, what=f"{lens}")


@pytest.mark.parametrize("page,heads_first,scale_pad,pad", [(16, True, 0, 8), (64, False, 16, 0), (256, True, 32, 24)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_decode_layouts(device, hd, page, heads_first, scale_pad, pad):
    for lens in ([300, 77], [5000]):
        decode_case(device, 21, 8, 2, hd, lens, page, F16, heads_first=heads_first, scale_pad=scale_pad, pad=pad, out_dtype=F32, what=f"{lens}")


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_q,causal", [(2, True), (4, True), (7, False), (5, True)])
def test_decode_rows(device, hd, n_q, causal):
    for lens in ([n_q, 90], [3, 40, 0], [2500, 600]):
        decode_case(device, 22, 14, 2, hd, lens, 16, BF16, n_q=n_q, causal=causal, what=f"{lens}")
    for scale in (0.0, -0.3):
        decode_case(device, 23, 8, 8, hd, [70, 900], 32, F16, n_q=n_q, causal=causal, scale=scale, what=f"scale {scale}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,group,n_q", [(64, 4, 1), (64, 7, 4), (128, 1, 1), (128, 8, 1), (128, 4, 4), (128, 7, 4), (256, 4, 1), (256, 7, 4)])
def test_decode_ranges(device, hd, group, n_q, dtype):
    """Many sequences of very different lengths, whose keys the workgroups share out in ranges."""
    lens = [(b * 53) % 400 for b in range(40)]
    lens[3], lens[4], lens[5], lens[17], lens[39] = 0, 1, 0, 2100, 900
    decode_case(device, 24, 8 * group, 8, hd, lens, 16, dtype, n_q=n_q, width=380)


def poke8(b, pos, head, d, code=None, byte=None, which="v"):
    def f(c):
        page, row = int(c.table[b, pos // c.page]), pos % c.page
        pool, scale = (c.k, c.ks) if which == "k" else (c.v, c.vs)
        if code is not None:
            pool[page, row, head, d] = code
        if byte is not None:
            scale[page, head, row] = byte
    return f


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("what", ["nan code", "nan scale", "infinite in f16"])
def test_decode_no_numbers_behind_the_mask(device, hd, what):
    """A NaN code, a NaN scale, and a scale that f16 cannot hold, at a key that only later rows see: the rows before do not know of it."""
    n_q = 4
    kw = {"nan code": dict(code=0xff), "nan scale": dict(byte=255), "infinite in f16": dict(code=0x70, byte=150)}[what]
    for L in (40, 100, 700, 3000):
        decode_case(device, 25, 6, 2, hd, [L, 50], 16, F16, n_q=n_q, mutate=poke8(0, L - 2, 1, 9, **kw), what=f"{what} {L}")


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_small_and_large_scales(device, hd):
    """Scales at the ends of the range: bf16 holds their products, down to its smallest numbers."""
    def shift(by):
        def f(c):
            for s in (c.vs,):
                s[s != 255] = (s[s != 255].int() + by).to(torch.uint8)
        return f
    for by in (-60, 60):
        decode_case(device, 26, 4, 2, hd, [100, 700], 16, BF16, out_dtype=F32, mutate=shift(by), what=f"{by}")


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_decode_bad_metadata(device, hd):
    g = gen(27)
    lens = [700, 900, 50, 400, 30]
    c = Cache8(g, lens, 2, hd, 16, F16)
    q = torch.randn(len(lens), 8 * hd, generator=g).to(F16)
    ref, rlse, tol, ltol = attend(c, q, [1] * len(lens), 8, hd ** -0.5, True, False, F16)
    k, v, table, kv_len, scales = c.to(device)
    table[1, 20], kv_len[3] = k.shape[0], table.shape[1] * 16 + 1
    ws = A.new_workspace(64 << 20, device)
    for _ in range(2):
        o, lse = A.paged_decode(q.to(device), k, v, table, kv_len, n_head=8, want_lse=True, scales=scales, workspace=ws)
        assert torch.isnan(o[[1, 3]]).all() and torch.isnan(lse[[1, 3]]).all()
        ok = [0, 2, 4]
        close(o[ok], ref[ok], tol[ok], "others")
        close(lse[ok], rlse[ok], ltol[ok], "others' lse")


def prefill_case(device, seed, n_head, n_kv, hd, rows, lens, page, dtype, causal=True, scale=None, out_dtype=None, heads_first=False,
                 scale_pad=0, pad=0, tail=0, ws=None, mutate=None, width=0, what=""):
    g = gen(seed)
    c = Cache8(g, lens, n_kv, hd, page, dtype, heads_first=heads_first, scale_pad=scale_pad, extra_width=1 + width)
    if mutate:
        mutate(c)
    total = sum(rows)
    q = torch.randn(total + tail, n_head * hd, generator=g).to(dtype)
    od = out_dtype or dtype
    dev_q, out = q.to(device), torch.full((total + tail, n_head * hd), 3.0, dtype=od, device=device)
    if pad:
        dev_q, out = padded(dev_q, pad), padded(out, pad)
    k, v, table, kv_len, scales = c.to(device)
    o, lse = A.paged_prefill(dev_q, k, v, table, kv_len, cu_of(rows, device), n_head=n_head, causal=causal, scale=scale, out=out,
                             want_lse=True, scales=scales, workspace=ws)
    ref, rlse, tol, ltol = attend(c, q, rows, n_head, 1 / math.sqrt(hd) if scale is None else scale, causal, True, od)
    close(o[:total], ref, tol, f"{what} out")
    close(lse[:total], rlse, ltol, f"{what} lse")
    if tail:
        assert (o[total:] == 3.0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 14, 2), (128, 28, 4), (128, 8, 2), (256, 4, 1)])
def test_prefill_lengths(device, hd, n_head, n_kv, dtype):
    for rows, lens in (([1], [1]), ([5, 1, 63], [5, 90, 64]), ([130, 0, 33], [130, 7, 500]), ([200], [1500]), ([90, 40], [0, 15])):
        prefill_case(device, 30, n_head, n_kv, hd, rows, lens, 16, dtype, what=f"{rows} {lens}")


@pytest.mark.parametrize("n_head,n_kv,rows", [(3, 3, 200), (4, 2, 200), (8, 2, 200), (7, 1, 700)])
def test_prefill_eight_waves(device, n_head, n_kv, rows):
    """The workgroups of eight waves, of every number of heads (head dim 128, a table of many keys)."""
    for causal in (True, False):
        prefill_case(device, 31, n_head, n_kv, 128, [rows], [rows + 90], 16, F16, causal=causal, width=200, what=f"{causal}")
    prefill_case(device, 32, n_head, n_kv, 128, [rows, 3], [rows + 2000 - rows % 64, 3], 16, BF16, width=200, pad=8, tail=2, out_dtype=F32)
    prefill_case(device, 32, n_head, n_kv, 128, [rows], [rows + 700], 64, BF16, width=80, heads_first=True, scale_pad=16,
                 ws=torch.empty(0, dtype=torch.uint8, device=device))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefill_options(device, hd):
    for page, heads_first, scale_pad in ((16, True, 16), (128, False, 0)):
        prefill_case(device, 33, 6, 2, hd, [100, 20], [400, 20], page, F16, heads_first=heads_first, scale_pad=scale_pad, pad=8, tail=3, out_dtype=F32)
    prefill_case(device, 34, 6, 2, hd, [70, 5], [300, 5], 32, BF16, causal=False)
    for scale in (0.0, -0.2):
        prefill_case(device, 35, 6, 2, hd, [70, 5], [300, 5], 32, F16, scale=scale)


@pytest.mark.parametrize("hd,width", [(64, 0), (128, 0), (128, 200), (256, 0)])
@pytest.mark.parametrize("what", ["nan code", "nan scale", "infinite in f16"])
def test_prefill_no_numbers_behind_the_mask(device, hd, width, what):
    kw = {"nan code": dict(code=0x7f), "nan scale": dict(byte=255), "infinite in f16": dict(code=0xf0, byte=150)}[what]
    for at, L in ((101, 130), (129, 130), (1990, 2000)):
        prefill_case(device, 36, 4, 2, hd, [120, 40], [L, 40], 16, F16, mutate=poke8(0, at, 1, 17, **kw), width=width, what=f"{what} {at} {L}")


@pytest.mark.parametrize("hd,width", [(64, 0), (128, 200), (256, 0)])
def test_prefill_bad_metadata(device, hd, width):
    g = gen(37)
    lens, rows = [1500, 1800, 50, 400], [200, 200, 50, 100]
    c = Cache8(g, lens, 2, hd, 16, F16, extra_width=1 + width)
    q = torch.randn(sum(rows), 4 * hd, generator=g).to(F16)
    ref, _, tol, _ = attend(c, q, rows, 4, hd ** -0.5, True, True, F16)
    k, v, table, kv_len, scales = c.to(device)
    table[1, 70], kv_len[3] = k.shape[0], table.shape[1] * 16 + 1
    out, lse = A.paged_prefill(q.to(device), k, v, table, kv_len, cu_of(rows, device), n_head=4, want_lse=True, scales=scales)
    for s, what in ((slice(200, 400), "page"), (slice(450, 550), "length")):
        assert torch.isnan(out[s]).all() and torch.isnan(lse[s]).all(), what
    for s in (slice(0, 200), slice(400, 450)):
        close(out[s], ref[s], tol[s], "others")


# ---- together ----

@pytest.mark.parametrize("n_head,n_kv,hd,dtype", [(14, 2, 64, F16), (32, 8, 128, BF16), (4, 2, 256, F16)])
def test_prompt_then_steps_captured(device, n_head, n_kv, hd, dtype):
    """A layer as a server runs it, on a stream of its own: prompts appended and attended, then a captured step (append, decode) that
    replays while the sequences grow. Each replay equals the definition over what the cache holds."""
    g = gen(40)
    rows, page, steps = [70, 1, 200], 16, 4
    lens = list(rows)
    c = Cache8(g, [n + steps + 1 for n in lens], n_kv, hd, page, dtype)
    k, v, table, _, scales = c.to(device)
    wide = (n_head + 2 * n_kv) * hd
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ws = A.new_workspace(128 << 20, device)
    torch.cuda.synchronize()

    def stored(lens):
        c.k, c.v, c.ks, c.vs = (t.view(torch.uint8).cpu() for t in (k, v, *scales))
        c.lens = lens
        return c

    with torch.cuda.stream(stream):
        x = torch.randn(sum(rows), wide, generator=g).to(device)
        kv_len = torch.tensor(lens, dtype=torch.int32, device=device)
        q = A.paged_store(x, k, v, table, kv_len, n_head=n_head, rope_mode=1, cu_q=cu_of(rows, device), scales=scales, q_dtype=dtype)
        o, _ = A.paged_prefill(q, k, v, table, kv_len, cu_of(rows, device), n_head=n_head, scales=scales, workspace=ws)
        stream.synchronize()
        ref, _, tol, _ = attend(stored(lens), q.cpu(), rows, n_head, hd ** -0.5, True, True, dtype)
        close(o, ref, tol, "prompts")
        step_x, step_q = torch.zeros(3, wide, device=device), torch.zeros(3, n_head * hd, dtype=dtype, device=device)
        step_o = torch.zeros_like(step_q)

        def step():
            A.paged_store(step_x, k, v, table, kv_len, n_head=n_head, rope_mode=1, q=step_q, scales=scales)
            A.paged_decode(step_q, k, v, table, kv_len, n_head=n_head, out=step_o, scales=scales, workspace=ws)
        lens = [n + 1 for n in lens]
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        step()
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(steps):
            if i:
                lens = [n + 1 for n in lens]
                kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
            step_x.copy_(torch.randn(3, wide, generator=g))
            graph.replay()
            stream.synchronize()
            ref, _, tol, _ = attend(stored(lens), step_q.cpu(), [1] * 3, n_head, hd ** -0.5, True, False, dtype)
            close(step_o, ref, tol, f"step {i}")


def test_extension_and_general_path_agree(device, monkeypatch):
    g = gen(41)
    c = Cache8(g, [40, 300], 2, 128, 16, BF16)
    k, v, table, kv_len, scales = c.to(device)
    q = torch.randn(2, 8 * 128, generator=g).to(BF16).to(device)
    x = torch.randn(2, 12 * 128, generator=g).to(device)
    ws = A.new_workspace(128 << 20, device)
    cu = cu_of([1, 1], device)

    def calls():
        return [A.paged_store(x, k, v, table, kv_len, n_head=8, rope_mode=0, scales=scales, q_dtype=BF16),
                *[t.view(torch.uint8).clone() for t in (k, v, *scales)],
                A.paged_decode(q, k, v, table, kv_len, n_head=8, scales=scales, workspace=ws)[0],
                A.paged_prefill(q, k, v, table, kv_len, cu, n_head=8, scales=scales, workspace=ws)[0]]
    want = calls()
    monkeypatch.setattr(A, "_native", lambda: A._General())
    for a, b in zip(want, calls()):
        assert torch.equal(a, b)


def test_pages_four_gigabytes_apart(device):
    """Codes and scales whose offsets pass 32 bits, for the append, a decode and a prompt."""
    g = gen(42)
    c = Cache8(g, [40, 33], 2, 128, 16, F16)
    total, apart = c.k.shape[0], (1 << 32) // 3 // 16 * 16 + 4096  # the pool spans more than 2^32 bytes from its fourth page on

    def far(t, shape, strides):
        wide = torch.empty(apart * total, dtype=torch.uint8, device=device).as_strided(shape, (apart, *strides))
        wide.copy_(t)
        return wide
    k, v = (far(t, t.shape, (256, 128, 1)).view(E4M3) for t in (c.k, c.v))
    scales = [far(t, t.shape, (16, 1)).view(E8M0) for t in (c.ks, c.vs)]
    _, _, table, kv_len, _ = c.to(device)
    q = torch.randn(2, 8 * 128, generator=g).to(F16)
    ref, _, tol, _ = attend(c, q, [1, 1], 8, 128 ** -0.5, True, False, F16)
    close(A.paged_decode(q.to(device), k, v, table, kv_len, n_head=8, scales=scales)[0], ref, tol, "decode")
    ref, _, tol, _ = attend(c, q, [1, 1], 8, 128 ** -0.5, True, True, F16)
    close(A.paged_prefill(q.to(device), k, v, table, kv_len, cu_of([1, 1], device), n_head=8, scales=scales)[0], ref, tol, "prompt")
    x = torch.randn(2, 12 * 128, generator=g)
    A.paged_store(x.to(device), k, v, table, kv_len, n_head=8, rope_mode=2, scales=scales)
    for b, L in enumerate(c.lens):
        page, row = int(c.table[b, (L - 1) // 16]), (L - 1) % 16
        for pool, scale, at in ((k, scales[0], 1024), (v, scales[1], 1280)):
            check_rows(pool.view(torch.uint8)[page, row][None].cpu(), scale.view(torch.uint8)[page, :, row][None].cpu(),
                       x[b, at:at + 256].double().view(1, 2, 128), torch.zeros(1, 2, 128, dtype=torch.float64), f"row {b}")


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_results_do_not_depend_on_the_run(device, hd):
    g = gen(43)
    lens = [2100, 7, 900, 0, 333]
    c = Cache8(g, lens, 4, hd, 16, BF16)
    k, v, table, kv_len, scales = c.to(device)
    q = torch.randn(5, 16 * hd, generator=g).to(BF16).to(device)
    rows = [200, 7, 90, 0, 333]
    p = torch.randn(sum(rows), 16 * hd, generator=g).to(BF16).to(device)
    ws = A.new_workspace(128 << 20, device)
    call = lambda: (A.paged_decode(q, k, v, table, kv_len, n_head=16, scales=scales, workspace=ws)[0],
                    A.paged_prefill(p, k, v, table, kv_len, cu_of(rows, device), n_head=16, scales=scales, workspace=ws)[0])
    want = call()
    for _ in range(10):
        for a, b in zip(call(), want):
            assert torch.equal(a, b)
