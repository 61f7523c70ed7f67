"""The paged cache's kernels where a sequence, a mask or a plan ends, against the definitions in 64 bits (paged_helpers.py)."""
import math

import pytest
import torch

from test_paged_gpu import BF16, F16, F32, poke, prefill_case

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
