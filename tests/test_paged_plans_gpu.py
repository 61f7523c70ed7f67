"""Every kernel that the paged calls' plans choose, on the cases where its own bookkeeping matters; the plan of each case is asked from
the diagnostic variant of the library, so that a bound that moves cannot take the cases with it."""
import ctypes
import math

import pytest
import torch

from dooms_amd import _lib
from dooms_amd import attention as A
from dooms_amd import build as B
from paged_helpers import Cache, attend, close
from test_paged_edges_gpu import wide
from test_paged_gpu import BF16, F16, F32, cu_of, gen, poke, prefill_case

PAGE = 16
CHUNKS, FIXED, RANGES = 0, 1, 2


def plan_of(prefill, n_head, n_kv, hd, n_seq, n_rows, keys, max_q=0):
    """[rows of a tile, waves, how the call is cut or heads of a tile] with a table of so many keys."""
    L = ctypes.CDLL(B.LIB_TRACE)
    L.mx_paged_trace_plan.argtypes = [ctypes.POINTER(_lib.MxPagedDesc), ctypes.c_int32, ctypes.POINTER(ctypes.c_int32)]
    d = _lib.MxPagedDesc(n_head=n_head, n_head_kv=n_kv, head_dim=hd, dtype=_lib.DTYPE_F16, n_seq=n_seq, n_rows=n_rows, page_size=PAGE,
                         max_pages=keys // PAGE, max_q=max_q)
    plan = (ctypes.c_int32 * 3)()
    assert L.mx_paged_trace_plan(ctypes.byref(d), prefill, plan) == _lib.OK
    return list(plan)


# ---- decode in ranges of all sequences' keys ----

# head dim, group, rows a sequence, rows of a tile
RANGED = [(64, 4, 1, 4), (64, 4, 2, 8), (64, 4, 3, 16), (64, 7, 4, 32), (64, 8, 6, 32),
          (128, 1, 1, 4), (128, 8, 1, 8), (128, 4, 4, 16), (128, 7, 4, 32), (128, 8, 6, 32),
          (256, 4, 1, 4), (256, 2, 4, 8), (256, 4, 3, 16), (256, 7, 4, 16)]
N_KV, TABLE = 8, 8192
LENS = [(b * 53) % 400 for b in range(40)]
LENS[3], LENS[4], LENS[5], LENS[17], LENS[39] = 0, 1, 0, 2100, 900  # several ranges, and parts of one


@pytest.mark.parametrize("hd,group,n_q,rt", RANGED)
def test_decode_range_plans(hd, group, n_q, rt):
    assert plan_of(0, N_KV * group, N_KV, hd, len(LENS), len(LENS) * n_q, TABLE) == [rt, 4, RANGES]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,group,n_q,rt", RANGED)
def test_decode_ranges_of_every_tile(device, hd, group, n_q, rt, dtype):
    """Several sequences in a range and several ranges in a sequence, empty ones between; then with lengths and pages that are none
    in the middle of ranges, whose sequences are NaN and whose neighbours are not."""
    g = gen(130 + rt)
    n_head = N_KV * group
    c = Cache(g, LENS, N_KV, hd, PAGE, dtype)
    wide(width=TABLE // PAGE - c.table.shape[1])(c)
    k, v, table, kv_len = c.to(device)
    q = torch.randn(len(LENS) * n_q, n_head * hd, generator=g).to(dtype)
    ref, rlse, tol, ltol = attend(c, q, [n_q] * len(LENS), n_head, hd ** -0.5, True, False, dtype)
    q = q.to(device)
    ws = A.new_workspace(A.paged_decode_workspace_bytes(n_head=n_head, n_head_kv=N_KV, head_dim=hd, n_q=n_q, n_seq=len(LENS),
                                                        max_kv_len=TABLE), device)
    call = lambda: A.paged_decode(q, k, v, table, kv_len, n_head=n_head, n_q=n_q, want_lse=True, workspace=ws)
    out, lse = call()
    close(out, ref, tol, "out")
    close(lse, rlse, ltol, "lse")
    table[10, 0], table[17, 60], table[17, 131] = -1, table.shape[1] * 100, -7  # the first page; of other parts of a long one
    kv_len[21], kv_len[30] = TABLE + 1, -3
    bad = torch.zeros(len(LENS), dtype=torch.bool)
    bad[[10, 17, 21, 30]] = True
    bad = bad.repeat_interleave(n_q)
    for _ in range(2):  # the counters are left at zero
        out, lse = call()
        assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
        close(out[~bad], ref[~bad], tol[~bad], "others")
        close(lse[~bad], rlse[~bad], ltol[~bad], "others' lse")


@pytest.mark.gpu
@pytest.mark.parametrize("hd,group,n_q,rt", [r for r in RANGED if r[2] > 1])
def test_decode_ranges_with_odd_values(device, hd, group, n_q, rt):
    """An infinity and a NaN among the keys that only later rows see, of sequences within a range and at its ends."""
    g = gen(140)
    n_head = N_KV * group
    c = Cache(g, LENS, N_KV, hd, PAGE, F16)
    for b, value in ((8, math.inf), (17, -math.inf), (18, math.nan), (39, math.inf)):
        poke(b, LENS[b] - 1, b % N_KV, 17, value)(c)
    wide(width=TABLE // PAGE - c.table.shape[1])(c)
    q = torch.randn(len(LENS) * n_q, n_head * hd, generator=g).to(F16)
    ref, _, tol, _ = attend(c, q, [n_q] * len(LENS), n_head, hd ** -0.5, True, False, F16)
    close(A.paged_decode(q.to(device), *c.to(device), n_head=n_head, n_q=n_q)[0], ref, tol, "out")


# ---- prompts on 8 waves ----

# heads, kv heads, rows, heads of a tile
EIGHT = [(3, 3, 200, 1), (4, 2, 200, 2), (6, 1, 200, 2), (8, 2, 200, 4), (7, 1, 200, 4), (7, 1, 700, 2), (7, 1, 1100, 1)]


@pytest.mark.parametrize("n_head,n_kv,rows,heads", EIGHT)
def test_prefill_shapes(n_head, n_kv, rows, heads):
    assert plan_of(1, n_head, n_kv, 128, 1, rows, 3200) == [256 // heads, 8, heads]
    for hd in (64, 128, 256):
        assert plan_of(1, n_head, n_kv, hd, 1, rows, 1024 if hd == 128 else 3200) == [128, 4, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,rows,heads", EIGHT)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prefill_options_on_eight_waves(device, n_head, n_kv, rows, heads, dtype):
    """What the 4-wave kernels are tested for: both masks, scales, strides, f32 outputs, heads first, rows without keys and behind the
    last sequence, with a workspace and without."""
    def case(seed, n, L, **kw):
        what = f"{n} {L} {sorted(kw)}"
        prefill_case(device, seed, n_head, n_kv, 128, n, L, PAGE, dtype, mutate=wide(width=200), what=what, **kw)
    case(150, [rows], [rows + 90])
    case(151, [rows], [rows + 33], causal=False)
    for scale in (0.0, -0.2):
        case(152, [rows], [rows], scale=scale)
    case(153, [rows], [rows + 7], pad=40, tail=3)
    case(154, [rows], [rows + 1], pad=8, out_dtype=F32, heads_first=True)
    case(155, [rows], [rows // 3])
    case(156, [rows], [0])
    case(157, [rows], [rows + 2000 - rows % 64], ws=torch.empty(0, dtype=torch.uint8, device=device))
    if rows == 200:
        case(158, [150, 3, 0, 200, 1], [900, 3, 5, 200, 1500], tail=2)
        case(159, [150, 3, 0, 200, 1], [900, 0, 5, 20, 1500], causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,rows,heads", EIGHT[:5])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_prefill_odd_values_on_eight_waves(device, n_head, n_kv, rows, heads, value):
    """Rows before an infinity or NaN do not know of it, in the same tile, another tile, or a part of a split one."""
    for at, L in ((101, 130), (129, 130), (1990, 2000), (1810, 2000)):
        prefill_case(device, 160, n_head, n_kv, 128, [120, 40], [L, 40], PAGE, F16, mutate=wide(poke(0, at, n_kv - 1, 17, value), width=200),
                     what=f"{at} {L}")
        if math.isnan(value):
            prefill_case(device, 160, n_head, n_kv, 128, [120, 40], [L, 40], PAGE, BF16,
                         mutate=wide(poke(0, at, n_kv - 1, 17, value, "k"), width=200), what=f"key {at} {L}")


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,rows,heads", EIGHT[:5])
def test_prefill_bad_metadata_on_eight_waves(device, n_head, n_kv, rows, heads):
    g = gen(161)
    lens, rows = [1500, 1800, 50, 400], [200, 200, 50, 100]
    c = Cache(g, lens, n_kv, 128, PAGE, F16)
    q = torch.randn(sum(rows), n_head * 128, generator=g).to(F16)
    ref, _, tol, _ = attend(c, q, rows, n_head, 128 ** -0.5, True, True, F16)
    k, v, table, kv_len = c.to(device)
    table[1, 70] = k.shape[0]
    kv_len[3] = table.shape[1] * PAGE + 1
    out, lse = A.paged_prefill(q.to(device), k, v, table, kv_len, cu_of(rows, device), n_head=n_head, want_lse=True)
    for s, what in ((slice(200, 400), "page"), (slice(450, 550), "length")):
        assert torch.isnan(out[s]).all() and torch.isnan(lse[s]).all(), what
    for s in (slice(0, 200), slice(400, 450)):
        close(out[s], ref[s], tol[s], "others")
