"""The paged cache's definitions in 64 bits on the CPU, its inputs, and how far the kernels may be from them.

Tolerances. u is half a step of a type relative to the value (f16 2^-11, bf16 2^-8). The attention kernels round
  * each probability to the pages' type before the product with the values (u each, at most u sum p|v| / sum p in the output),
    the prompts' kernel also in the sum l that divides (another u);
  * in f16, probabilities below 2^-14 by at most 2^-25 each;
  * scores, exponentials and sums in f32: a score is off by at most (head_dim + 4) 2^-24 sum_d |q_d k_d| |scale|, which moves p by
    that factor, the exponential by 2^-21 (the hardware's own error and its argument's rounding at up to 2^2), sums by 2^-24
    a term;
  * the output once, to its type (u, or 2^-24).
"""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # half a step of the smallest values


class Cache:
    """A pool of pages dealt to sequences of the given lengths in random order; rows that hold no key are `garbage`."""

    def __init__(self, g, lens, n_head_kv, hd, page, dtype, *, heads_first=False, garbage=float("nan"), spare=2, extra_width=1):
        self.lens, self.page, self.hd, self.n_head_kv, self.dtype = list(lens), page, hd, n_head_kv, dtype
        used = [-(-n // page) for n in lens]
        total = sum(used) + spare
        ids = torch.randperm(total, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max([1] + used) + extra_width), total + 7, dtype=torch.int32)  # unused entries are no page
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.free = ids[at:]
        shape = (total, n_head_kv, page, hd) if heads_first else (total, page, n_head_kv, hd)
        self.k, self.v = (torch.full(shape, garbage, dtype=dtype) for _ in range(2))
        if heads_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        for b, n in enumerate(lens):
            for p in (self.k, self.v):
                new = torch.randn(n, n_head_kv, hd, generator=g).to(dtype)
                pos = torch.arange(n)
                p[self.table[b, pos // page].long(), pos % page] = new

    def keys(self, b, n=None):
        pos = torch.arange(self.lens[b] if n is None else n)
        at = (self.table[b, pos // self.page].long(), pos % self.page)
        return self.k[at].double(), self.v[at].double()

    def to(self, device):
        def strided(t):
            if t.is_contiguous():
                return t.to(device)
            return t.transpose(1, 2).to(device).transpose(1, 2)
        return strided(self.k), strided(self.v), self.table.to(device), torch.tensor(self.lens, dtype=torch.int32, device=device)


def attend(cache, q, rows, n_head, scale, causal, rounded_sum, out_dtype):
    """The definition for packed rows (rows[b] of sequence b): (out, lse, tolerance of out, tolerance of lse), f64. A row without
    a key is zeros and -inf."""
    hd, group, u = cache.hd, n_head // cache.n_head_kv, U[cache.dtype]
    total = sum(rows)
    out = torch.zeros(total, n_head, hd, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full((total, n_head), -math.inf, dtype=torch.float64)
    ltol = torch.zeros(total, n_head, dtype=torch.float64)
    at = 0
    for b, n in enumerate(rows):
        L = cache.lens[b]
        if n == 0 or L == 0:
            at += n
            continue
        k, v = cache.keys(b)
        qs = q[at:at + n, :n_head * hd].double().view(n, n_head, hd)
        seen = torch.ones(n, L, dtype=torch.bool)
        if causal:
            seen = torch.arange(L)[None] <= (torch.arange(n) + L - n)[:, None]
        for h in range(n_head):
            kh, vh = k[:, h // group], v[:, h // group]
            s = (qs[:, h] @ kh.T) * scale
            s = torch.where(seen, s, torch.tensor(-math.inf, dtype=torch.float64))
            live = seen.any(1)
            top = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(live[:, None], top, 0.0))
            l = p.sum(1, keepdim=True)
            wv = torch.where(seen[:, :, None], p[:, :, None], 0.0) * torch.where(seen[:, :, None], vh[None], 0.0) if \
                not torch.isfinite(vh).all() else None
            o = (wv.sum(1) if wv is not None else p @ vh) / l
            off = (hd + 4) * 2.0 ** -24 * abs(scale) * (qs[:, h].abs() @ kh.abs().T)  # of each score
            rel = u * (2 if rounded_sum else 1) + 2 * (off + 2.0 ** -21) + L * 2.0 ** -24
            vabs = torch.where(torch.isfinite(vh), vh, 0.0).abs()
            spread = ((p * rel) @ vabs + (p * (2 * (off + 2.0 ** -21) + (u if rounded_sum else 0))).sum(1, keepdim=True) * (p @ vabs) / l) / l
            floor = 2.0 ** -24 if cache.dtype == torch.float16 else 0.0
            spread = spread + floor * (seen.double() @ vabs) / l
            rs = slice(at, at + n)
            out[rs, h] = torch.where(live[:, None], o, 0.0)
            lse[rs, h] = torch.where(live, (top + torch.log(l))[:, 0], torch.tensor(-math.inf, dtype=torch.float64))
            tol[rs, h] = torch.where(live[:, None], spread, 0.0)
            mean = (p * (2 * off + 2.0 ** -20 + (u if rounded_sum else 0.0))).sum(1) / l[:, 0]
            ltol[rs, h] = torch.where(live, mean + L * 2.0 ** -24 + floor * L + (top.abs()[:, 0] + 16) * 2.0 ** -22, 0.0)
        at += n
    tol += U[out_dtype] * (out.abs() + tol) + TINY[out_dtype]
    return out.flatten(1), lse, tol.flatten(1), ltol


def close(got, ref, tol, what):
    got = got.double().cpu()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), f"{what}: infinities differ"
    err = torch.where(fine, (got - ref).abs(), 0.0)
    bad = err > torch.where(fine, tol, 0.0)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by {float((err / tol.clamp_min(1e-300)).max()):.2f} "
                           f"tolerances, at {[int(x) for x in torch.nonzero(bad)[0]]}")


def rotate(x, pos, mode, base, axis_pairs, restart):
    """x [rows][heads][hd] f64 turned for positions [axes][rows]: (rotated, sum of magnitudes of each result's two products)."""
    hd = x.shape[-1]
    out, mag = x.clone(), x.abs().clone()
    if mode == 2:
        return out, mag
    i = 0
    for a, n in enumerate(axis_pairs):
        for j in range(n):
            f = float(base) ** (-j / n if restart else -2.0 * i / hd)
            th = (pos[a].double() * f)[:, None]
            lo, hi = (2 * i, 2 * i + 1) if mode == 0 else (i, i + hd // 2)
            c, s = torch.cos(th), torch.sin(th)
            out[..., lo], out[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., lo] * s + x[..., hi] * c
            mag[..., lo] = mag[..., hi] = x[..., lo].abs() + x[..., hi].abs()
            i += 1
    return out, mag
