"""The paged key-value cache in 8 bits, and sequences that share a prefix, as a serving program calls them: the append that
quantises (paged_store), attention of new tokens (paged_decode) and of packed prompts (paged_prefill) over pages in 8 bits, and
attention of new tokens of sequences whose first keys are the same (paged_decode_shared), over pages in 16 or 8 bits.

A row of a kv head in 8 bits is head_dim codes (float8 e4m3) and one scale, the smallest power of two with which the largest
magnitude of the row is at most 448; it stands for code x scale.

A case is a dict of plain values. `kind` names the operator, `model` the head shape, `dtype` the type of the queries and outputs
(and of the pages where quant is false), `page` the keys per page; the sequences' lengths follow from `seqs`, `kv_min`,
`kv_max` (keys with the new ones) and, for the store and the prompts, `q_min`, `q_max` (new rows). Shared prefixes: `seqs`
sequences in `groups` groups, of `p_min` to `p_max` keys in common and `own_min` to `own_max` of each sequence's own.
Pages are dealt to the sequences in a random order, and rows of the pool that hold no key are NaN, codes and scales too, where
an operator only reads it, as memory that nobody wrote may be.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"

# The head shapes of this repository's decoders: query heads, kv heads, head dim, rotary mode (0 adjacent pairs, 1 split
# halves) and rotary base.
MODELS = {
    "qwen2.5-0.5b": dict(n_head=14, n_head_kv=2, head_dim=64, rope=1, base=1e6),
    "qwen2.5-7b": dict(n_head=28, n_head_kv=4, head_dim=128, rope=1, base=1e6),
    "llama-3-8b": dict(n_head=32, n_head_kv=8, head_dim=128, rope=0, base=5e5),
}
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def listed():
    return [
        # one user's decode step of a small model: one row into its page; all latency
        dict(name="quant_store_step", kind="store", model="qwen2.5-0.5b", dtype="f16", quant=True, rows="f32", page=16, seqs=1, kv_min=514, kv_max=514, q_min=1, q_max=1),
        # the packed batch of prompts that a scheduler forms each step, some behind a cached prefix
        dict(name="quant_store_prompts", kind="store", model="llama-3-8b", dtype="bf16", quant=True, rows="f32", page=64, seqs=7, kv_min=90, kv_max=1801, q_min=90, q_max=1300),
        # one user's step of a small model at chat length: latency and launch bound
        dict(name="quant_decode_chat", kind="decode", model="qwen2.5-0.5b", dtype="f16", quant=True, page=16, seqs=1, kv_min=513, kv_max=513, n_q=1),
        # one user's long document: every CU on one sequence
        dict(name="quant_decode_long", kind="decode", model="llama-3-8b", dtype="bf16", quant=True, page=64, seqs=1, kv_min=32768, kv_max=32768, n_q=1),
        # a serving step of 64 sequences of very different lengths: bound by the memory
        dict(name="quant_decode_batch", kind="decode", model="llama-3-8b", dtype="f16", quant=True, page=16, seqs=64, kv_min=111, kv_max=8191, n_q=1),
        # a few short prompts of a small model, whole: time to first token
        dict(name="quant_prompt_short", kind="prefill", model="qwen2.5-0.5b", dtype="f16", quant=True, page=16, seqs=5, kv_min=37, kv_max=420, q_min=37, q_max=420),
        # a scheduler's packed chunk of whole prompts
        dict(name="quant_prompt_packed", kind="prefill", model="llama-3-8b", dtype="bf16", quant=True, page=64, seqs=12, kv_min=65, kv_max=1711, q_min=65, q_max=1711),
        # the next chunk of long prompts, behind what the cache holds of them already: the largest prompts
        dict(name="quant_prompt_chunk", kind="prefill", model="qwen2.5-7b", dtype="f16", quant=True, page=128, seqs=2, kv_min=14001, kv_max=16384, q_min=1500, q_max=2048),
        # eight answers sampled for one question to a small model
        dict(name="shared_samples", kind="shared", model="qwen2.5-0.5b", dtype="f16", quant=False, page=16, groups=1, seqs=8, p_min=700, p_max=700, own_min=5, own_max=120, n_q=1),
        # a serving step of 64 users behind one system prompt
        dict(name="shared_system", kind="shared", model="llama-3-8b", dtype="bf16", quant=False, page=16, groups=1, seqs=64, p_min=4096, p_max=4096, own_min=40, own_max=900, n_q=1),
        # users of several applications, two drafted tokens each, over a cache in 8 bits
        dict(name="shared_drafts", kind="shared", model="qwen2.5-7b", dtype="bf16", quant=True, page=32, groups=5, seqs=40, p_min=1000, p_max=6000, own_min=10, own_max=500, n_q=2),
        # many questions about one long document: the largest call
        dict(name="shared_document", kind="shared", model="llama-3-8b", dtype="f16", quant=False, page=64, groups=1, seqs=192, p_min=16384, p_max=16384, own_min=100, own_max=1500, n_q=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed kinds: any head shape, type and page, lengths over their whole range."""
    bytes_, flops = {"store": 0.5e9, "decode": 0.55e9, "prefill": 1e9, "shared": 1e9}, {"prefill": 0.7e12, "shared": 7e10}
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= bytes_[c["kind"]] and w["flops"] <= flops.get(c["kind"], 1e12):
            return c


def _draw(rng):
    kind = rng.choice(["store", "decode", "decode", "prefill", "shared", "shared", "shared"])
    c = dict(kind=kind, model=rng.choice(sorted(MODELS)), dtype=rng.choice(["f16", "bf16"]), quant=True, page=rng.choice([16, 16, 32, 64, 128, 256]),
             seqs=_log(rng, 1, {"decode": 96, "shared": 200}.get(kind, 24)))
    if kind == "decode":
        hi = _log(rng, 16, 32768)
        n_q = rng.choice([1, 1, 1, 2, 3, 5, 8])
        return dict(c, kv_min=rng.randint(max(n_q, hi // 16), hi), kv_max=hi, n_q=n_q)
    if kind == "shared":
        c["seqs"] = max(2, c["seqs"])
        p_hi, own_hi, n_q = _log(rng, 32, 16384), _log(rng, 8, 2000), rng.choice([1, 1, 1, 2, 4])
        p_lo = rng.randint(max(1, p_hi // 8), p_hi)
        if rng.random() < 0.6:  # prefixes are mostly kept in whole pages
            p_lo, p_hi = (-(-x // c["page"]) * c["page"] for x in (p_lo, p_hi))
        return dict(c, quant=rng.random() < 0.5, groups=rng.choice([1, 1, rng.randint(1, max(1, min(8, c["seqs"] // 2)))]), p_min=p_lo, p_max=p_hi,
                    own_min=rng.randint(max(n_q, own_hi // 16), max(n_q, own_hi)), own_max=max(n_q, own_hi), n_q=n_q)
    q_hi = _log(rng, 1 if kind == "store" else 16, 4096)
    q_lo = rng.randint(max(1, q_hi // 16), q_hi)
    prefix = rng.choice([0, 0, 0, _log(rng, 16, 16384)])
    c = dict(c, q_min=q_lo, q_max=q_hi, kv_min=q_lo + prefix // 3, kv_max=q_hi + prefix)
    return dict(c, rows=rng.choice(["f32", "f32", "f16", "bf16"])) if kind == "store" else c


def _spread(n, lo, hi):
    """n lengths from the longest down to the shortest, evenly."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _shape(c):
    """(keys, new rows) of each sequence, and for shared prefixes (sequences, keys in common) of each group."""
    if c["kind"] != "shared":
        kv = _spread(c["seqs"], c["kv_min"], c["kv_max"])
        if c["kind"] == "decode":
            return kv, [c["n_q"]] * len(kv), []
        return kv, [min(q, k) for q, k in zip(_spread(c["seqs"], c["q_min"], c["q_max"]), kv)], []
    n, g = c["seqs"], c["groups"]
    sizes = [n // g + (i < n % g) for i in range(g)]
    if g > 1 and sizes[0] > 1:  # groups are not alike
        move = sizes[-1] // 2
        sizes[0] += move
        sizes[-1] -= move
    groups = list(zip(sizes, _spread(g, c["p_min"], c["p_max"])))
    mine = _spread(n, c["own_min"], c["own_max"])
    prefix = [p for size, p in groups for _ in range(size)]
    order = [(i * 7 + 3) % n if n % 7 else i for i in range(n)]  # long and short ones in every group
    return [p + mine[i] for p, i in zip(prefix, order)], [c["n_q"]] * n, groups


def work(case):
    m = MODELS[case["model"]]
    kv, nq, groups = _shape(case)
    d, rows = m["head_dim"], sum(nq)
    wide = m["n_head"] * d
    row = m["n_head_kv"] * (d + 1 if case["quant"] else 2 * d)  # bytes of a token's keys, or values
    if case["kind"] == "store":
        n = rows * (m["n_head"] + 2 * m["n_head_kv"]) * d
        return {"bytes": n * (4 if case["rows"] == "f32" else 2) + 2 * rows * wide + 2 * rows * row, "flops": 4 * n}
    pairs = sum(n * k - n * (n - 1) // 2 if k >= n else k * (k + 1) // 2 for n, k in zip(nq, kv))
    keys = sum(kv) - sum((size - 1) * p for size, p in groups)
    return {"bytes": 2 * keys * row + 4 * rows * wide, "flops": 4 * pairs * wide}


def _power(k):
    """2^k in 32 bits for whole k from -126 to 127."""
    return ((k + 127).to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """Rows of x (32 bits) in 8 bits: (codes, scales as exponents + 127 in a byte)."""
    top = x.abs().amax(-1)
    frac, e = torch.frexp(top)
    k = torch.where(top == 0, -127, (e - 9 + (frac > 0.875)).clamp(min=-127))  # 448 = 0.875 x 2^9
    return (x * _power(-k)[..., None]).to(E4M3), (k + 127).to(torch.uint8)


def _inputs(c, seed):
    """The tensors a serving program holds before the call, from the seed alone."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    pick = random.Random(seed)
    m, page, dt = MODELS[c["model"]], c["page"], TYPES[c["dtype"]]
    kv, nq, groups = _shape(c)
    if not groups:
        order = list(range(len(kv)))
        pick.shuffle(order)
        kv, nq = [kv[i] for i in order], [nq[i] for i in order]
    used = [-(-n // page) for n in kv]
    first = np.concatenate([[0], np.cumsum([size for size, _ in groups])]).astype(np.int32)
    shared = [p // page for size, p in groups for _ in range(size)] or [0] * len(kv)  # whole pages in common
    new = [n - (s if groups and b not in first else 0) for b, (n, s) in enumerate(zip(used, shared))]
    total = sum(new) + 3
    ids = torch.randperm(total, generator=g, device=DEV).to(torch.int32).cpu()
    table = torch.zeros(len(kv), max(used), dtype=torch.int32)
    at = 0
    for b, (n, fresh) in enumerate(zip(used, new)):
        table[b, n - fresh:n] = ids[at:at + fresh]
        if fresh < n:
            table[b, :n - fresh] = table[b - 1, :n - fresh]
        at += fresh
    shape = (total, page, m["n_head_kv"], m["head_dim"])
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32)
    loud = 1.0 + 5.0 * (torch.arange(m["head_dim"], device=DEV) % 29 == 3)  # keys have a few channels that stand out
    pools, scales = [], []
    for i in range(2):
        x = rnd(*shape) * loud if i == 0 else rnd(*shape) * torch.exp(0.5 * rnd(total, page, m["n_head_kv"], 1))
        if c["quant"]:
            codes, e = _quantise(x)
            pools.append(codes)
            scales.append(e.permute(0, 2, 1).contiguous())
        else:
            pools.append(x.to(dt))
        del x
    if c["kind"] != "store":
        for b, n in enumerate(kv):  # rows behind a sequence's end hold whatever was there
            if n % page:
                last = int(table[b, used[b] - 1])
                for p in pools:
                    (p.view(torch.uint8)[last, n % page:].fill_(127) if c["quant"] else p[last, n % page:].fill_(float("nan")))
                for e in scales:
                    e[last, :, n % page:] = 255
    s = dict(case=c, kv=kv, nq=nq, groups=groups, table=table.to(DEV), k=pools[0], v=pools[1], scales=[e.view(E8M0) for e in scales],
             kv_len=torch.tensor(kv, dtype=torch.int32, device=DEV))
    starts = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
    s["starts"] = [int(x) for x in starts]
    s["cu_q"] = torch.from_numpy(starts).to(DEV)
    rows = int(starts[-1])
    if groups:
        s["first"] = [int(x) for x in first]
        s["cu_seq"] = torch.from_numpy(first).to(DEV)
        s["prefix_len"] = torch.tensor([p for _, p in groups], dtype=torch.int32, device=DEV)
    if c["kind"] == "store":
        s["qkv"] = rnd(rows, (m["n_head"] + 2 * m["n_head_kv"]) * m["head_dim"]).to(TYPES[c["rows"]])
    else:
        s["q"] = (1.5 * rnd(rows, m["n_head"] * m["head_dim"])).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from dooms_amd import attention as A
        m = MODELS[case["model"]]
        shape = dict(n_head=m["n_head"], n_head_kv=m["n_head_kv"], head_dim=m["head_dim"], n_seq=len(s["kv"]))
        if case["kind"] == "decode":  # the workspace a program allocates once
            s["ws"] = A.new_workspace(A.paged_decode_workspace_bytes(n_q=case["n_q"], max_kv_len=max(s["kv"]), **shape), DEV)
        elif case["kind"] == "prefill":
            s["ws"] = A.new_workspace(A.paged_prefill_workspace_bytes(n_rows=s["starts"][-1], max_q=max(s["nq"]), max_kv_len=max(s["kv"]), **shape), DEV)
        elif case["kind"] == "shared":
            s["ws"] = A.new_workspace(A.paged_shared_workspace_bytes(n_q=case["n_q"], n_groups=len(s["groups"]), max_own_len=case["own_max"], **shape), DEV)
    torch.cuda.synchronize()
    return s


def run(state):
    """One call of the operator (own), or its plain form in 32 bits."""
    c = state["case"]
    m = MODELS[c["model"]]
    if own:
        from dooms_amd import attention as A
        where = (state["k"], state["v"], state["table"], state["kv_len"])
        scales = state["scales"] or None
        if c["kind"] == "store":
            q = A.paged_store(state["qkv"], *where, n_head=m["n_head"], cu_q=state["cu_q"], rope_mode=m["rope"], rope_base=m["base"],
                              scales=scales, q_dtype=TYPES[c["dtype"]])
            return [q, state["k"], state["v"], *state["scales"]]
        if c["kind"] == "decode":
            return A.paged_decode(state["q"], *where, n_head=m["n_head"], n_q=c["n_q"], max_kv_len=max(state["kv"]), scales=scales, workspace=state["ws"])[0]
        if c["kind"] == "prefill":
            return A.paged_prefill(state["q"], *where, state["cu_q"], n_head=m["n_head"], max_q=max(state["nq"]), max_kv_len=max(state["kv"]),
                                   scales=scales, workspace=state["ws"])[0]
        return A.paged_decode_shared(state["q"], *where, state["cu_seq"], state["prefix_len"], n_head=m["n_head"], n_q=c["n_q"], max_own_len=c["own_max"],
                                     scales=scales, workspace=state["ws"])[0]
    return {"store": _store_plain, "decode": _decode_plain, "prefill": _prefill_plain, "shared": _shared_plain}[c["kind"]](state, m)


def _store_plain(s, m):
    c, d = s["case"], m["head_dim"]
    half, nh, nkv = d // 2, m["n_head"], m["n_head_kv"]
    rows, device = s["qkv"].shape[0], s["qkv"].device
    seq = torch.repeat_interleave(torch.arange(len(s["nq"]), device=device), torch.diff(s["cu_q"]).long(), output_size=rows)
    n_new = torch.diff(s["cu_q"])[seq]
    where = (s["kv_len"][seq] - n_new + torch.arange(rows, device=device, dtype=torch.int32) - s["cu_q"][seq]).long()
    freq = m["base"] ** -(torch.arange(half, device=device, dtype=torch.float64) / half)
    angle = where.double()[:, None] * freq  # 64 bits: the angles of far positions
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x):
        a, b = (x[..., 0::2], x[..., 1::2]) if m["rope"] == 0 else (x[..., :half], x[..., half:])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.stack((a, b), -1).flatten(-2) if m["rope"] == 0 else torch.cat((a, b), -1)

    x = s["qkv"].float().view(rows, nh + 2 * nkv, d)
    page, row = s["table"][seq, where // c["page"]].long(), where % c["page"]
    for pool, scale, new in ((s["k"], s["scales"][0], turn(x[:, nh:nh + nkv])), (s["v"], s["scales"][1], x[:, nh + nkv:])):
        codes, e = _quantise(new)
        pool.view(torch.uint8)[page, row] = codes.view(torch.uint8)
        scale.view(torch.uint8)[page, :, row] = e
    return [turn(x[:, :nh]).flatten(1).to(TYPES[c["dtype"]]), s["k"], s["v"], *s["scales"]]


def _keys(s, pool, at, page, row):
    """The rows (page, row) of a pool (0 keys, 1 values) in 32 bits, [...][kv heads][head dim]."""
    x = s[pool]
    if not s["case"]["quant"]:
        return x[page, row].float()
    codes = x.view(torch.uint8)[page, row].view(E4M3).float()
    return codes * s["scales"][at].view(torch.uint8)[page, :, row].view(E8M0).float()[..., None]


def _padded(s, seqs, start, lens):
    """Keys and values of some sequences from key `start` on, padded to the longest with zeros: [sequence][kv head][dim][key] and
    [sequence][kv head][key][dim], and which of them there are."""
    pos = start + torch.arange(max(1, max(lens)), device=DEV)
    n = torch.tensor(lens, device=DEV)
    live = pos[None] < start + n[:, None]
    page = s["table"][seqs][:, (pos // s["case"]["page"]).clamp(max=s["table"].shape[1] - 1)].long()
    row = (pos % s["case"]["page"]).expand_as(page)
    k, v = (torch.where(live[:, :, None, None], _keys(s, p, i, page, row), 0.0) for i, p in enumerate("kv"))
    return k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous(), live


def _hide(live, lens, n, group):
    """Which keys the rows [group][n] of a sequence may not see: none behind its end, nor later ones of the new."""
    pos = torch.arange(live.shape[1], device=DEV)
    last = torch.tensor(lens, device=DEV)[:, None] - n + torch.arange(n, device=DEV)
    return (pos[None, None] > last[:, :, None])[:, None, None].expand(-1, 1, group, -1, -1).reshape(len(lens), 1, group * n, -1)


def _rows(q, n_seq, n, nkv, group, d):
    return q.float().view(n_seq, n, nkv, group, d).permute(0, 2, 3, 1, 4).reshape(n_seq, nkv, group * n, d)


def _decode_plain(s, m):
    d, nkv, n = m["head_dim"], m["n_head_kv"], s["case"]["n_q"]
    group, seqs = m["n_head"] // nkv, len(s["kv"])
    k, v, live = _padded(s, torch.arange(seqs, device=DEV), 0, s["kv"])
    q = _rows(s["q"], seqs, n, nkv, group, d)
    score = (torch.matmul(q, k) * d ** -0.5).masked_fill_(_hide(live, s["kv"], n, group), float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(seqs, nkv, group, n, d).permute(0, 3, 1, 2, 4).reshape(seqs * n, -1).to(s["q"].dtype)


def _prefill_plain(s, m):
    d, nkv = m["head_dim"], m["n_head_kv"]
    group = m["n_head"] // nkv
    out = torch.empty_like(s["q"])
    for b, (n, L) in enumerate(zip(s["nq"], s["kv"])):
        k, v, live = _padded(s, torch.tensor([b], device=DEV), 0, [L])
        r0 = s["starts"][b]
        q = _rows(s["q"][r0:r0 + n], 1, n, nkv, group, d)[0]
        hide = _hide(live, [L], n, 1)[0, 0]
        step = max(1, int(2e9 // (group * n * L)))  # kv heads at a time: the scores fit the memory
        for h in range(0, nkv, step):
            score = torch.bmm(q[h:h + step], k[0, h:h + step]) * d ** -0.5
            score.view(-1, group, n, L).masked_fill_(hide, float("-inf"))
            score = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.bmm(score, v[0, h:h + step]) / score.sum(-1, keepdim=True)
            heads = o.shape[0] * group
            out[r0:r0 + n, h * group * d:(h * group + heads) * d] = o.view(heads, n, d).transpose(0, 1).reshape(n, heads * d).to(out.dtype)
    return out


def _shared_plain(s, m):
    d, nkv, n = m["head_dim"], m["n_head_kv"], s["case"]["n_q"]
    group = m["n_head"] // nkv
    out = torch.empty_like(s["q"])
    for (size, prefix), b0 in zip(s["groups"], s["first"]):
        kp, vp, _ = _padded(s, torch.tensor([b0], device=DEV), 0, [prefix])
        lens = [L - prefix for L in s["kv"][b0:b0 + size]]
        ko, vo, live = _padded(s, torch.arange(b0, b0 + size, device=DEV), prefix, lens)
        q = _rows(s["q"][b0 * n:(b0 + size) * n], size, n, nkv, group, d)
        # the keys in common, once for all rows of the group
        sp = torch.matmul(q.transpose(0, 1).reshape(nkv, -1, d), kp[0]) * d ** -0.5
        so = (torch.matmul(q, ko) * d ** -0.5).masked_fill_(_hide(live, lens, n, group), float("-inf"))
        sp = sp.view(nkv, size, group * n, -1).transpose(0, 1)
        top = torch.maximum(sp.amax(-1), so.amax(-1))[..., None]
        sp, so = torch.exp(sp - top), torch.exp(so - top)
        o = torch.matmul(sp.transpose(0, 1).reshape(nkv, size * group * n, -1), vp[0]).view(nkv, size, group * n, d).transpose(0, 1)
        o = (o + torch.matmul(so, vo)) / (sp.sum(-1) + so.sum(-1))[..., None]
        out[b0 * n:(b0 + size) * n] = o.view(size, nkv, group, n, d).permute(0, 3, 1, 2, 4).reshape(size * n, -1).to(out.dtype)
    return out


def exact(case, seed):
    """The operators' definitions in 64 bits, sequence by sequence and head by head."""
    s = _inputs(case, seed)
    m = MODELS[case["model"]]
    d, page, nh, nkv = m["head_dim"], case["page"], m["n_head"], m["n_head_kv"]
    slots = [(s["table"][b].long()[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:L] for b, L in enumerate(s["kv"])]
    for (size, prefix), b0 in zip(s["groups"], s.get("first", [])):  # the first sequence's pages place the keys in common
        for b in range(b0, b0 + size):
            slots[b][:prefix] = slots[b0][:prefix]
    if case["kind"] == "store":
        return _store_exact(s, m, slots)
    flat = [t.view(torch.uint8 if case["quant"] else t.dtype).reshape(-1, nkv, d) for t in (s["k"], s["v"])]
    if case["quant"]:
        e = [x.view(torch.uint8).transpose(1, 2).reshape(-1, nkv) for x in s["scales"]]
    q = s["q"].double().view(-1, nh, d)
    out = torch.empty_like(q)
    for b, (n, L) in enumerate(zip(s["nq"], s["kv"])):
        kv = [t[slots[b]] for t in flat]
        if case["quant"]:
            kv = [t.view(E4M3).double() * torch.pow(2.0, x[slots[b]].double() - 127)[..., None] for t, x in zip(kv, e)]
        k, v = (t.double().permute(1, 0, 2).contiguous() for t in kv)
        rows = slice(s["starts"][b], s["starts"][b + 1])
        for h in range(nh):
            logits = (q[rows, h].contiguous() @ k[h * nkv // nh].T.contiguous()) / math.sqrt(d)
            logits += torch.full_like(logits, float("-inf")).triu_(L - n + 1)
            out[rows, h] = torch.softmax(logits, -1) @ v[h * nkv // nh]
    return out.flatten(1)


def _store_exact(s, m, slots):
    d, nh, nkv = m["head_dim"], m["n_head"], m["n_head_kv"]
    x = s["qkv"].double().view(-1, nh + 2 * nkv, d)
    turned = x.clone()
    codes = [t.double() for t in (s["k"], s["v"])]
    scales = [e.double() for e in s["scales"]]
    page = s["case"]["page"]
    for b, (n, L) in enumerate(zip(s["nq"], s["kv"])):
        rows = slice(s["starts"][b], s["starts"][b + 1])
        pos = torch.arange(L - n, L, device=DEV).double()
        for i in range(d // 2):
            z = torch.polar(torch.ones_like(pos), pos * math.exp(-math.log(m["base"]) * 2 * i / d))[:, None]
            lo, hi = (2 * i, 2 * i + 1) if m["rope"] == 0 else (i, i + d // 2)
            w = torch.complex(x[rows, :nh + nkv, lo], x[rows, :nh + nkv, hi]) * z
            turned[rows, :nh + nkv, lo], turned[rows, :nh + nkv, hi] = w.real, w.imag
        at = slots[b][L - n:]
        for pool, scale, new in zip(codes, scales, (turned[rows, nh:nh + nkv], x[rows, nh + nkv:])):
            unit = torch.pow(2.0, torch.ceil(torch.log2(new.abs().amax(-1, keepdim=True) / 448)))
            y = new / unit
            step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)  # of the type at y
            pool.view(-1, nkv, d)[at] = torch.round(y / step) * step
            scale[at // page, :, at % page] = unit[..., 0]
    return [turned[:, :nh].flatten(1), *codes, *scales]
