"""The paged key-value cache's operators, as a serving program calls them: the rotated append (paged_store), attention of
new tokens over the pages (paged_decode) and of packed prompts (paged_prefill).

A case is a dict of plain values. `kind` names the operator, `model` the head shape, `dtype` the pages' type, `page` the
keys per page; the sequences' lengths follow from `seqs`, `kv_min`, `kv_max` (keys with the new ones) and, for the store and
the prompts, `q_min`, `q_max` (new rows). Pages are dealt to the sequences in a random order, and rows of the pool that hold
no key are NaN where an operator only reads it, as memory that nobody wrote may be.
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


def listed():
    return [
        # one user's decode step of a small model: one row into its page; all latency
        dict(name="store_step", kind="store", model="qwen2.5-0.5b", dtype="f16", rows="f32", page=16, seqs=1, kv_min=514, kv_max=514, q_min=1, q_max=1, axes=1, restart=False),
        # a packed batch of prompts, some behind a cached prefix: the chunk that a scheduler forms each step
        dict(name="store_prompts", kind="store", model="llama-3-8b", dtype="bf16", rows="f32", page=64, seqs=7, kv_min=90, kv_max=1801, q_min=90, q_max=1300, axes=1, restart=False),
        # a prompt of text and images: time, height and width positions, from a bf16 projection
        dict(name="store_images", kind="store", model="qwen2.5-7b", dtype="bf16", rows="bf16", page=128, seqs=3, kv_min=2200, kv_max=3500, q_min=2200, q_max=3500, axes=3, restart=False),
        # one user's step of a small model at chat length: latency and launch bound
        dict(name="decode_chat", kind="decode", model="qwen2.5-0.5b", dtype="f16", page=16, seqs=1, kv_min=513, kv_max=513, n_q=1, heads_first=False),
        # one user's long context: every CU on one sequence
        dict(name="decode_long", kind="decode", model="llama-3-8b", dtype="bf16", page=64, seqs=1, kv_min=8192, kv_max=8192, n_q=1, heads_first=False),
        # four drafted tokens of each of nine sequences, verified in one call; pages with the heads outermost
        dict(name="decode_draft", kind="decode", model="qwen2.5-7b", dtype="bf16", page=32, seqs=9, kv_min=201, kv_max=5999, n_q=4, heads_first=True),
        # a serving step of 64 sequences of very different lengths: bound by the memory
        dict(name="decode_batch", kind="decode", model="llama-3-8b", dtype="f16", page=16, seqs=64, kv_min=111, kv_max=8191, n_q=1, heads_first=False),
        # a few short prompts of a small model, whole: time to first token
        dict(name="prompt_short", kind="prefill", model="qwen2.5-0.5b", dtype="f16", page=16, seqs=5, kv_min=37, kv_max=420, q_min=37, q_max=420),
        # a scheduler's packed chunk of whole prompts
        dict(name="prompt_packed", kind="prefill", model="llama-3-8b", dtype="bf16", page=64, seqs=12, kv_min=65, kv_max=1711, q_min=65, q_max=1711),
        # the next chunk of long prompts, behind what the cache holds of them already: the largest call
        dict(name="prompt_chunk", kind="prefill", model="qwen2.5-7b", dtype="f16", page=128, seqs=2, kv_min=14001, kv_max=16384, q_min=1500, q_max=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed kinds: any head shape, type and page, lengths over their whole range."""
    most = {"store": 0.6e9, "decode": 1.1e9, "prefill": 0.9e12}
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops" if c["kind"] == "prefill" else "bytes"] <= most[c["kind"]]:
            return c


def _draw(rng):
    kind = rng.choice(["store", "decode", "decode", "prefill", "prefill"])
    c = dict(kind=kind, model=rng.choice(sorted(MODELS)), dtype=rng.choice(["f16", "bf16"]), page=rng.choice([16, 16, 32, 64, 128, 256]),
             seqs=_log(rng, 1, 96 if kind == "decode" else 24))
    if kind == "decode":
        hi = _log(rng, 16, 32768)
        n_q = rng.choice([1, 1, 1, 2, 3, 5, 8])
        return dict(c, kv_min=rng.randint(max(n_q, hi // 16), hi), kv_max=hi, n_q=n_q, heads_first=rng.random() < 0.3)
    q_hi = _log(rng, 1 if kind == "store" else 16, 4096)
    q_lo = rng.randint(max(1, q_hi // 16), q_hi)
    prefix = rng.choice([0, 0, 0, _log(rng, 16, 16384)])
    c = dict(c, q_min=q_lo, q_max=q_hi, kv_min=q_lo + prefix // 3, kv_max=q_hi + prefix)
    if kind == "store":
        axes = rng.choice([1, 1, 2, 3])
        c = dict(c, rows=rng.choice(["f32", "f32", "f16", "bf16"]), axes=axes, restart=axes > 1 and rng.random() < 0.4)
    return c


def _spread(n, lo, hi):
    """n lengths from the longest down to the shortest, evenly."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lens(c):
    """(keys, new rows) of each sequence."""
    kv = _spread(c["seqs"], c["kv_min"], c["kv_max"])
    if c["kind"] == "decode":
        return kv, [c["n_q"]] * len(kv)
    return kv, [min(q, k) for q, k in zip(_spread(c["seqs"], c["q_min"], c["q_max"]), kv)]


def _axis_pairs(c):
    """Rotary pairs of each position axis: all of them, height and width in equal parts, or a quarter for the time."""
    half = MODELS[c["model"]]["head_dim"] // 2
    return {1: (half,), 2: (half // 2, half // 2), 3: (half // 4, 3 * half // 8, 3 * half // 8)}[c["axes"]]


def work(case):
    m = MODELS[case["model"]]
    kv, nq = _lens(case)
    d, size = m["head_dim"], 2
    wide, rows = m["n_head"] * d, sum(nq)
    if case["kind"] == "store":
        n = rows * (m["n_head"] + 2 * m["n_head_kv"]) * d
        return {"bytes": n * (4 if case["rows"] == "f32" else 2) + n * size, "flops": 3 * n}
    pairs = sum(n * k - n * (n - 1) // 2 if k >= n else k * (k + 1) // 2 for n, k in zip(nq, kv))
    return {"bytes": 2 * sum(kv) * m["n_head_kv"] * d * size + 2 * rows * wide * size, "flops": 4 * pairs * wide}


def _inputs(c, seed):
    """The tensors a serving program holds before the call, from the seed alone."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    pick = random.Random(seed)
    m, page, dt = MODELS[c["model"]], c["page"], TYPES[c["dtype"]]
    kv, nq = _lens(c)
    order = list(range(len(kv)))
    pick.shuffle(order)
    kv, nq = [kv[i] for i in order], [nq[i] for i in order]
    used = [-(-n // page) for n in kv]
    total = sum(used) + 3
    ids = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(kv), max(used), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
    shape = (total, page, m["n_head_kv"], m["head_dim"])
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32)
    pools = []
    for _ in range(2):
        if c["kind"] == "decode" and c["heads_first"]:
            pools.append(rnd(total, shape[2], page, shape[3]).to(dt).transpose(1, 2))
        else:
            pools.append(rnd(*shape).to(dt))
    if c["kind"] != "store":
        for b, n in enumerate(kv):  # rows behind a sequence's end hold whatever was there
            if n % page:
                for p in pools:
                    p[table[b, used[b] - 1].long(), n % page:] = float("nan")
    s = dict(case=c, kv=kv, nq=nq, table=table, k=pools[0], v=pools[1], kv_len=torch.tensor(kv, dtype=torch.int32, device=DEV))
    starts = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
    s["starts"] = [int(x) for x in starts]
    s["cu_q"] = torch.from_numpy(starts).to(DEV)
    rows = int(starts[-1])
    if c["kind"] == "store":
        s["qkv"] = rnd(rows, (m["n_head"] + 2 * m["n_head_kv"]) * m["head_dim"]).to(TYPES[c["rows"]])
        s["positions"] = None
        if c["axes"] > 1:  # text counts on all axes alike, an image's patches share a time and count on a grid
            pos = np.zeros((c["axes"], rows), dtype=np.int32)
            for b, (n, k) in enumerate(zip(nq, kv)):
                t = np.arange(n)
                cut = n // 3
                side = max(1, math.isqrt(max(1, n - 2 * cut)))
                img = (t >= cut) & (t < n - cut)
                grid = [np.full(n, cut), cut + (t - cut) // side, cut + (t - cut) % side][-c["axes"]:]
                for a in range(c["axes"]):
                    pos[a, starts[b]:starts[b + 1]] = k - n + np.where(img, grid[a], t)
            s["positions"] = torch.from_numpy(pos).to(DEV)
    else:
        s["q"] = (2.0 * rnd(rows, m["n_head"] * m["head_dim"])).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from dooms_amd import attention as A
        m = MODELS[case["model"]]
        shape = dict(n_head=m["n_head"], n_head_kv=m["n_head_kv"], head_dim=m["head_dim"], n_seq=len(s["kv"]), max_kv_len=max(s["kv"]))
        if case["kind"] == "decode":  # the workspace a program allocates once
            s["ws"] = A.new_workspace(A.paged_decode_workspace_bytes(n_q=case["n_q"], **shape), DEV)
        elif case["kind"] == "prefill":
            s["ws"] = A.new_workspace(A.paged_prefill_workspace_bytes(n_rows=s["starts"][-1], max_q=max(s["nq"]), **shape), DEV)
    torch.cuda.synchronize()
    return s


def run(state):
    """One call of the operator (own), or its plain form in 32 bits."""
    c = state["case"]
    m = MODELS[c["model"]]
    if own:
        from dooms_amd import attention as A
        where = (state["k"], state["v"], state["table"], state["kv_len"])
        if c["kind"] == "store":
            q = A.paged_store(state["qkv"], *where, n_head=m["n_head"], cu_q=state["cu_q"], rope_mode=m["rope"], rope_base=m["base"],
                              positions=state["positions"], axis_pairs=_axis_pairs(c), axis_restart=c["restart"])
            return [q, state["k"], state["v"]]
        if c["kind"] == "decode":
            return A.paged_decode(state["q"], *where, n_head=m["n_head"], n_q=c["n_q"], max_kv_len=max(state["kv"]), workspace=state["ws"])[0]
        return A.paged_prefill(state["q"], *where, state["cu_q"], n_head=m["n_head"], max_q=max(state["nq"]), max_kv_len=max(state["kv"]),
                               workspace=state["ws"])[0]
    return _store_plain(state, m) if c["kind"] == "store" else _attend_plain(state, m)


def _store_plain(s, m):
    c, d, dt = s["case"], m["head_dim"], s["k"].dtype
    half, nh, nkv = d // 2, m["n_head"], m["n_head_kv"]
    rows, device = s["qkv"].shape[0], s["qkv"].device
    seq = torch.repeat_interleave(torch.arange(len(s["nq"]), device=device), torch.diff(s["cu_q"]).long(), output_size=rows)
    n_new = torch.diff(s["cu_q"])[seq]
    where = (s["kv_len"][seq] - n_new + torch.arange(rows, device=device, dtype=torch.int32) - s["cu_q"][seq]).long()
    pairs = _axis_pairs(c)
    expo = torch.cat([torch.arange(n, device=device, dtype=torch.float64) / n for n in pairs]) if c["restart"] else \
        torch.arange(half, device=device, dtype=torch.float64) / half
    freq = m["base"] ** -expo
    pos = where[None] if s["positions"] is None else s["positions"]
    axis = torch.cat([torch.full((n,), a, device=device) for a, n in enumerate(pairs)])
    angle = pos.T.double()[:, axis] * freq  # 64 bits: the angles of far positions
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x):
        a, b = (x[..., 0::2], x[..., 1::2]) if m["rope"] == 0 else (x[..., :half], x[..., half:])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.stack((a, b), -1).flatten(-2) if m["rope"] == 0 else torch.cat((a, b), -1)

    x = s["qkv"].float().view(rows, nh + 2 * nkv, d)
    page = s["table"][seq, where // c["page"]].long()
    s["k"][page, where % c["page"]] = turn(x[:, nh:nh + nkv]).to(dt)
    s["v"][page, where % c["page"]] = x[:, nh + nkv:].to(dt)
    return [turn(x[:, :nh]).flatten(1).to(dt), s["k"], s["v"]]


def _attend_plain(s, m):
    c, d, nkv = s["case"], m["head_dim"], m["n_head_kv"]
    group = m["n_head"] // nkv
    out = torch.empty_like(s["q"])
    for b, (n, L) in enumerate(zip(s["nq"], s["kv"])):
        ids = s["table"][b, :-(-L // c["page"])].long()
        k = s["k"][ids].flatten(0, 1)[:L].float().permute(1, 2, 0).contiguous()  # [kv head][dim][key]
        v = s["v"][ids].flatten(0, 1)[:L].float().permute(1, 0, 2).contiguous()
        r0 = s["starts"][b]
        q = s["q"][r0:r0 + n].float().view(n, nkv, group, d).permute(1, 2, 0, 3).reshape(nkv, group * n, d)
        hide = None
        if n > 1:
            hide = torch.arange(L, device=q.device)[None] > torch.arange(L - n, L, device=q.device)[:, None]
        step = max(1, int(2e9 // (group * n * L)))  # kv heads at a time: the scores fit the memory
        for h in range(0, nkv, step):
            score = torch.bmm(q[h:h + step], k[h:h + step]) * d ** -0.5
            if hide is not None:
                score.view(-1, group, n, L).masked_fill_(hide, float("-inf"))
            score = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.bmm(score, v[h:h + step]) / score.sum(-1, keepdim=True)
            heads = o.shape[0] * group
            out[r0:r0 + n, h * group * d:(h * group + heads) * d] = o.view(heads, n, d).transpose(0, 1).reshape(n, heads * d).to(out.dtype)
    return out


def exact(case, seed):
    """The operators' definitions in 64 bits, row by row of the cache rather than by pages."""
    s = _inputs(case, seed)
    m = MODELS[case["model"]]
    d, page, nh, nkv = m["head_dim"], case["page"], m["n_head"], m["n_head_kv"]
    slots = [(s["table"][b].long()[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:L] for b, L in enumerate(s["kv"])]
    if case["kind"] == "store":
        return _store_exact(s, m, slots)
    flat_k, flat_v = (t.reshape(-1, nkv, d) for t in (s["k"], s["v"]))
    q = s["q"].double().view(-1, nh, d)
    out = torch.empty_like(q)
    for b, (n, L) in enumerate(zip(s["nq"], s["kv"])):
        k, v = flat_k[slots[b]].double(), flat_v[slots[b]].double()
        rows = slice(s["starts"][b], s["starts"][b + 1])
        for h in range(nh):
            kt = k[:, h * nkv // nh].T.contiguous()
            vh = v[:, h * nkv // nh].contiguous()
            logits = (q[rows, h].contiguous() @ kt) / math.sqrt(d)
            logits += torch.full_like(logits, float("-inf")).triu_(L - n + 1)
            out[rows, h] = torch.softmax(logits, -1) @ vh
    return out.flatten(1)


def _store_exact(s, m, slots):
    d, nh, nkv = m["head_dim"], m["n_head"], m["n_head_kv"]
    c = s["case"]
    x = s["qkv"].double().view(-1, nh + 2 * nkv, d)
    k, v = s["k"].double(), s["v"].double()
    turned = x.clone()
    pairs = _axis_pairs(c)
    for b, (n, L) in enumerate(zip(s["nq"], s["kv"])):
        rows = slice(s["starts"][b], s["starts"][b + 1])
        i = 0
        for a, count in enumerate(pairs):
            pos = torch.arange(L - n, L, device=DEV).double() if s["positions"] is None else s["positions"][a, rows].double()
            for j in range(count):
                f = math.exp(-math.log(m["base"]) * (j / count if c["restart"] else 2 * i / d))
                z = torch.polar(torch.ones_like(pos), pos * f)[:, None]
                lo, hi = (2 * i, 2 * i + 1) if m["rope"] == 0 else (i, i + d // 2)
                w = torch.complex(x[rows, :nh + nkv, lo], x[rows, :nh + nkv, hi]) * z
                turned[rows, :nh + nkv, lo], turned[rows, :nh + nkv, hi] = w.real, w.imag
                i += 1
        at = slots[b][L - n:]
        k.view(-1, nkv, d)[at] = turned[rows, nh:nh + nkv]
        v.view(-1, nkv, d)[at] = x[rows, nh + nkv:]
    return [turned[:, :nh].flatten(1), k, v]
