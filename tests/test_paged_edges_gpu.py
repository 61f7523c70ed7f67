"""The paged cache's kernels where a sequence, a mask or a plan ends, against the definitions in 64 bits (paged_helpers.py)."""
import math

import pytest
import torch

from dooms_amd import attention as A
from paged_helpers import Cache, attend, close
from test_paged_gpu import BF16, F16, F32, cu_of, gen, poke, prefill_case

pytestmark = pytest.mark.gpu


def wide(*mutations, width=100):
    """A page table with room for more keys than the sequences have, so that plans for long sequences are taken; then the others."""
    def f(c):
        c.table = torch.cat([c.table, torch.full((c.table.shape[0], width), c.k.shape[0] + 7, dtype=torch.int32)], dim=1)
        for m in mutations:
            m(c)
    return f


# ---- infinities that every row of a wave sees, among the last keys of a sequence ----

@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("hd,n_head,n_kv,long", [(64, 4, 2, False), (128, 4, 2, False), (128, 8, 2, True), (128, 4, 2, True), (128, 3, 3, True),
                                                 (256, 4, 2, False)])
def test_prefill_infinity_among_the_last_keys(device, hd, n_head, n_kv, long, value):
    """The rows see the key, so the definition gives an infinity; lengths that end within a step of 64 keys, within 16 of them and
    at either, of one row, four rows and one row past a wave's 32."""
    for rows, L, at in ((1, 70, 66), (1, 70, 69), (4, 70, 66), (33, 97, 96), (33, 97, 81), (4, 80, 70), (1, 64, 63), (1, 65, 64), (7, 16, 3),
                        (200, 213, 212)):
        m = poke(0, at, n_kv - 1, 17, value)
        prefill_case(device, 120, n_head, n_kv, hd, [rows, 20], [L, 40], 16, F16, mutate=wide(m) if long else m, what=f"{rows} {L} {at}")
        prefill_case(device, 120, n_head, n_kv, hd, [rows, 20], [L, 40], 32, BF16, causal=False, mutate=wide(m) if long else m,
                     what=f"not causal {rows} {L} {at}")


@pytest.mark.parametrize("hd,long", [(64, False), (128, False), (128, True), (256, False)])
def test_prefill_scores_of_minus_infinity_first(device, hd, long):
    """The first keys' scores are -inf, so they weigh nothing, and rows before an infinity among the values are computed by
    themselves: the weights start at the first finite score. The definition is evaluated with finite keys whose weight is
    below 10^-100 instead, as its tolerance knows no infinities."""
    g = gen(121)
    c = Cache(g, [75, 50], 1, hd, 16, F16)
    (wide(poke(0, 74, 0, 5, math.inf)) if long else poke(0, 74, 0, 5, math.inf))(c)
    q = torch.randn(80, 2 * hd, generator=g)
    q[:, 3] = q[:, 3].abs().clamp_min(0.5)
    q[:, hd + 3] = q[:, hd + 3].abs().clamp_min(0.5)
    q = q.to(F16)
    for pos in (0, 1, 2):
        poke(0, pos, 0, 3, -math.inf, "k")(c)
    k, v, table, kv_len = c.to(device)
    out, lse = A.paged_prefill(q.to(device), k, v, table, kv_len, cu_of([60, 20], device), n_head=2, scale=0.125, want_lse=True)
    for pos in (0, 1, 2):
        poke(0, pos, 0, 3, -30000.0, "k")(c)
    ref, rlse, tol, ltol = attend(c, q, [60, 20], 2, 0.125, True, True, F16)
    close(out, ref, tol, "out")
    close(lse, rlse, ltol, "lse")


@pytest.mark.parametrize("hd,n_head,n_kv,dtype,long", [(64, 4, 2, F16, False), (128, 2, 2, BF16, True), (128, 8, 2, F16, True), (128, 4, 1, F16, False),
                                                       (256, 2, 1, BF16, False)])
def test_prefill_tiles_of_one_step_before_longer_ones(device, hd, n_head, n_kv, dtype, long):
    """Ranges whose tiles of one step leave the next tile's page numbers to be requested between two tiles: every step attends
    the keys of its own pages."""
    lens = [(60, 33, 200, 64, 500, 1)[b % 6] for b in range(330)]
    prefill_case(device, 122, n_head, n_kv, hd, [min(L, 1 + b % 3) for b, L in enumerate(lens)], lens, 16, dtype,
                 mutate=wide() if long else None)


# ---- layouts ----

def test_one_page_and_one_head_have_no_stride(device):
    """A pool with one kv head or one page, whose strides along them may be anything, each pool's its own."""
    g = gen(123)
    c = Cache(g, [30, 12], 1, 64, 16, F16)
    k, v, table, kv_len = c.to(device)
    last = k.squeeze(2).contiguous().unsqueeze(3).transpose(2, 3)  # stride 1 along the heads
    assert last.stride(2) == 1 and v.stride(2) == 64
    q = torch.randn(2, 4 * 64, generator=g).to(F16)
    ref, _, tol, _ = attend(c, q, [1, 1], 4, 0.125, True, True, F16)
    ws = A.new_workspace(64 << 20, device)
    for w in (None, ws):
        close(A.paged_decode(q.to(device), last, v, table, kv_len, n_head=4, workspace=w)[0], ref, tol, "decode")
        close(A.paged_prefill(q.to(device), last, v, table, kv_len, cu_of([1, 1], device), n_head=4, workspace=w)[0], ref, tol, "prefill")
    x = torch.randn(2, 6 * 64, generator=g).to(device)
    for pools in ((k.clone(), v.clone()), (last.clone(memory_format=torch.preserve_format), v.clone())):
        A.paged_store(x, *pools, table, kv_len, n_head=4, rope_mode=2)
        assert torch.equal(pools[0][table[1, 0].long(), 11, 0], x[1, 256:320].to(F16))
    one = Cache(g, [9], 2, 128, 16, BF16, spare=0)
    k, v, table, kv_len = one.to(device)
    k = torch.as_strided(k, k.shape, (3, *k.stride()[1:]))
    q = torch.randn(1, 4 * 128, generator=g).to(BF16)
    ref, _, tol, _ = attend(one, q, [1], 4, 128 ** -0.5, True, False, BF16)
    close(A.paged_decode(q.to(device), k, v, table, kv_len, n_head=4)[0], ref, tol, "one page")
