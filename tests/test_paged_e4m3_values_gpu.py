"""Every code with every scale: the value that the attention calls read for it, against the definition in 64 bits.

One key and one row: the only probability is 1, so the output is the value itself, and the lse the score. All products and sums of these
have one term that is not 0: the only roundings are the expansion's to the queries' type, and for the lse that of its scale and logarithm."""
import math

import pytest
import torch

from dooms_amd import attention as A
from e4m3_helpers import E4M3, E8M0, power
from test_paged_gpu import BF16, F16, F32

pytestmark = pytest.mark.gpu

PAGE, HD = 16, 256


def pools(device):
    """Sequence b, one key in page b: all 256 codes, with scale byte b; and the values that they stand for."""
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 1, HD).expand(256, PAGE, 1, HD).contiguous()
    byte = torch.arange(256, dtype=torch.uint8).view(256, 1, 1).expand(256, 1, PAGE).contiguous()
    other = torch.full_like(byte, 127)
    table = torch.arange(256, dtype=torch.int32).view(256, 1)
    ints = torch.ones(256, dtype=torch.int32)
    value = codes[:, 0, 0].view(E4M3).double() * power(byte[:, 0, 0])[:, None]
    return codes.view(E4M3).to(device), byte.view(E8M0).to(device), other.view(E8M0).to(device), table.to(device), ints.to(device), value


def call(kind, q, k, v, table, kv_len, scales, n_head, scale):
    """Attention of one row of each sequence over its one key, which for `shared` pairs of sequences have in common."""
    device = q.device
    if kind == "decode":
        return A.paged_decode(q, k, v, table, kv_len, n_head=n_head, out_dtype=F32, want_lse=True, scales=scales, scale=scale)
    if kind == "prompts":
        cu = torch.arange(table.shape[0] + 1, dtype=torch.int32, device=device)
        return A.paged_prefill(q, k, v, table, kv_len, cu, n_head=n_head, out_dtype=F32, want_lse=True, scales=scales, scale=scale)
    n = table.shape[0]
    cu = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=device)
    twice = lambda t: t.repeat_interleave(2, 0)
    o, lse = A.paged_decode_shared(twice(q), k, v, twice(table), twice(kv_len), cu, torch.ones(n, dtype=torch.int32, device=device), n_head=n_head,
                                   out_dtype=F32, want_lse=True, scales=scales, scale=scale)
    assert torch.equal(o[::2].nan_to_num(), o[1::2].nan_to_num()) and torch.equal(lse[::2].nan_to_num(), lse[1::2].nan_to_num())
    return o[::2], lse[::2]


@pytest.mark.parametrize("kind", ["decode", "prompts", "shared"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values(device, kind, dtype):
    codes, byte, other, table, kv_len, value = pools(device)
    o, _ = call(kind, torch.zeros(256, HD, dtype=dtype, device=device), torch.zeros_like(codes.view(torch.uint8)).view(E4M3), codes, table, kv_len,
                (other, byte), 1, 1.0)
    want = value.to(dtype).double()
    got = o.double().cpu()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert same.all(), [(int(b), int(c), float(got[b, c]), float(want[b, c])) for b, c in torch.nonzero(~same)[:8]]


@pytest.mark.parametrize("kind", ["decode", "prompts", "shared"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_keys(device, kind, dtype):
    """Head h's query is dim h alone: its score is the key's value there."""
    codes, byte, other, table, kv_len, value = pools(device)
    q = torch.eye(HD, dtype=dtype, device=device).flatten()[None].expand(256, HD * HD).contiguous()
    ok = torch.isfinite(value[0])
    codes = torch.where(ok.to(device), codes.view(torch.uint8), torch.zeros_like(codes.view(torch.uint8))).view(E4M3)  # NaN spoils all dims
    want = torch.where(ok, value, 0.0).to(dtype).double()
    _, lse = call(kind, q, codes, codes, table, kv_len, (byte, other), HD, 1.0)
    got = lse.double().cpu()
    # A score times log2 e stays in f32. Prompts, and prefixes as they do, take scores below 2^27: they fuse its product with the maximum's
    # difference, so that the largest probability is 2 to the power of what the product's rounding lost, at most 2^8 there.
    fine = torch.isfinite(want).all(1) & (want.abs().amax(1) < (2.0 ** 126 if kind == "decode" else 2.0 ** 27))
    err = (got - want).abs()
    tol = 2.0 ** -21 * want.abs() + 2.0 ** -126
    bad = ~(err <= tol) & fine[:, None]
    assert not bad.any(), [(int(b), int(c), float(got[b, c]), float(want[b, c])) for b, c in torch.nonzero(bad)[:8]]
    assert torch.isnan(got[255]).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype,power_of_two", [(F16, 30), (BF16, 100)])
def test_decode_of_large_scores(device, dtype, power_of_two, eight):
    """Scores apart by more than any weight: the output is the value of the largest one, in the first block of keys, a later one and the
    last. The dims of a row of keys are one number, those
    of the query 2 to half the power."""
    top = 2.0 ** (power_of_two - power_of_two // 2)
    g = torch.Generator().manual_seed(90)
    for at in (3, 41, 69):
        k = torch.zeros(5, PAGE, 1, 64, dtype=torch.float64)
        k.view(80, 64)[:] = (-top * (1 + torch.arange(80) % 7) / 64)[:, None]
        k.view(80, 64)[at] = top * 7 / 8
        v = torch.randint(1, 9, (5, PAGE, 1, 64), generator=g).double()
        table = torch.arange(5, dtype=torch.int32, device=device)[None]
        kv_len = torch.tensor([70], dtype=torch.int32, device=device)
        q = torch.full((1, 64), 2.0 ** (power_of_two // 2) * 0.75, dtype=dtype, device=device)
        scales = None
        if eight:
            e = int(math.log2(top)) + 1  # codes of a row below 1
            scales = [torch.full((5, 1, PAGE), b, dtype=torch.uint8, device=device).view(E8M0) for b in (127 + e, 127)]
            pages = [(k / 2.0 ** e).to(E4M3), v.to(E4M3)]
        else:
            pages = [k.to(dtype), v.to(dtype)]
        o, _ = A.paged_decode(q, *(t.to(device) for t in pages), table, kv_len, n_head=1, scale=1.0, scales=scales)
        assert torch.equal(o[0].double().cpu(), v.view(80, 64)[at]), at
