"""The paged-cache operators as cases that can be timed and compared.

Three operators of a serving program that keeps its key-value cache in pages:

* append: the fused q|k|v projection of new tokens (fp32) gets its per-head
  RMSNorm and rotary embedding, the queries come back in the cache's type, and
  keys and values go to the last slots of their sequence's pages;
* attention: the newest token (or the n newest, causally) of each sequence
  attends to its cached slots; the logarithm of the softmax's denominator comes
  back beside the result, and optionally every slot's weight is added to the
  slot's accumulator;
* eviction: each sequence and kv head keeps a budget of slots -- the first
  positions, the most recent ones, and those of the largest accumulated
  weight -- and the kept rows move into the evicted slots below the budget.

``run`` computes them in elementary fp32 torch operations where ``own`` is
false, and through abra_b200 where it is true.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
THETA = 1.0e6


# ------------------------------------------------------------------ cases ---
def _case(name, op, **kw):
    c = dict(op=op, dtype="f16", hq=32, hkv=8, d=128, page=16, order="HND", n_seqs=1, len_lo=1,
             len_hi=512, len_seed=0, n_q=1, accumulate=False, budget=0, sink=0, recent=0)
    if name:
        c["name"] = name
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of one conversation: the smallest append, all latency
        _case("append_1", "append", len_lo=600, len_hi=600),
        # one decode step of a batch at mixed depths
        _case("append_32", "append", dtype="bf16", n_seqs=32, len_lo=1, len_hi=4096, page=64),
        # prompts of several users arriving together, 1 to 4096 tokens each
        _case("append_prompts", "append", n_seqs=9, len_lo=1, len_hi=4096, len_seed=3, page=64, n_q=0),
        # one token of one conversation at the depth of a short chat
        _case("attend_1x600", "attention", len_lo=600, len_hi=600),
        # a decode batch of mixed depths, two of them empty slots of the batch
        _case("attend_32x4096", "attention", dtype="bf16", n_seqs=32, len_lo=1, len_hi=4096, len_seed=1),
        # the same at long contexts, the largest read
        _case("attend_64x16384", "attention", dtype="bf16", n_seqs=64, len_lo=200, len_hi=16384,
              len_seed=2, page=64),
        # one long document, where the cache's length is what there is to split
        _case("attend_1x131071", "attention", n_seqs=1, len_lo=131071, len_hi=131071, page=256),
        # verification of 15 drafts and the current token for four users
        _case("attend_verify_4x16", "attention", n_seqs=4, len_lo=400, len_hi=8192, len_seed=4, n_q=16),
        # accumulating slot weights for the eviction; wide groups, small heads, odd pages in token order
        _case("attend_weights_16x8192", "attention", dtype="bf16", hq=64, hkv=8, d=64, page=24,
              order="NHD", n_seqs=16, len_lo=1, len_hi=8192, len_seed=5, accumulate=True),
        # one page over the budget: what a decode loop does every 64 tokens
        _case("evict_1x4160", "evict", page=64, len_lo=4160, len_hi=4160, budget=4096, sink=4, recent=512),
        # prompts cut to their budget after prefill, some already inside it
        _case("evict_32x8192", "evict", dtype="bf16", n_seqs=32, len_lo=300, len_hi=8192, len_seed=6,
              budget=2048, sink=4, recent=256),
        # one long document cut to a quarter
        _case("evict_1x131072", "evict", page=256, len_lo=131072, len_hi=131072, budget=32768, sink=16,
              recent=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "evict"))
    d = rng.choice((64, 96, 128, 128))
    hkv = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    page = rng.choice((8, 16, 16, 24, 32, 64, 100, 256))
    n_seqs = _log(rng, 1, 64)
    hi = min(_log(rng, 8, 131072), 16384 * 64 // n_seqs)  # no more slots than the largest case holds
    lo = rng.choice((1, max(1, hi // 2), hi))
    c = _case(None, op, dtype=rng.choice(("f16", "bf16")), hq=hkv * group, hkv=hkv, d=d, page=page,
              order=rng.choice(("HND", "HND", "NHD")), n_seqs=n_seqs, len_lo=lo, len_hi=hi,
              len_seed=rng.randrange(1 << 20))
    if op == "append":
        c["n_q"] = rng.choice((0, 1, 1, rng.randrange(2, 17)))
        c["len_hi"] = min(c["len_hi"], 16384 // n_seqs if c["n_q"] == 0 else 16384)
        c["len_lo"] = min(c["len_lo"], c["len_hi"])
    elif op == "attention":
        c["n_q"] = rng.choice((1, 1, 1, rng.randrange(2, 17)))
        c["accumulate"] = rng.random() < 0.35
        if c["n_q"] * group > 16:  # many rows a slot: fewer slots, the same cost
            c["len_hi"] = max(1, c["len_hi"] // 8)
            c["len_lo"] = min(c["len_lo"], c["len_hi"])
    else:
        c["budget"] = max(1, int(hi * rng.uniform(0.1, 1.1)))
        c["sink"] = rng.randrange(0, 5) if c["budget"] > 8 else 0
        c["recent"] = int((c["budget"] - c["sink"]) * rng.uniform(0.0, 0.5))
    return c


def _lens(case):
    """Cached slots of each sequence, the new tokens among them: the longest
    first, the others spread between the two ends; in a ragged batch about one
    in sixteen is empty."""
    lo, hi, n = case["len_lo"], case["len_hi"], case["n_seqs"]
    if lo == hi:
        return [hi] * n
    r = random.Random(case["len_seed"])
    return [hi] + [0 if r.random() < 1 / 16 else _log(r, lo, hi) for _ in range(n - 1)]


def _new_tokens(case):
    """How many of each sequence's slots are new in an append: all of them
    (a prompt) where n_q is 0, else at most n_q."""
    lens = _lens(case)
    return lens if case["n_q"] == 0 else [min(case["n_q"], n) for n in lens]


# ----------------------------------------------------------------- inputs ---
def _inputs(case, seed):
    """The tensors of one case, on the GPU, from the seed alone."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    dt, ps, hkv, hq, d = DTYPES[case["dtype"]], case["page"], case["hkv"], case["hq"], case["d"]
    n = case["n_seqs"]
    lens = np.array(_lens(case), dtype=np.int64)
    pages = -(-lens // ps)
    n_pages, width = int(pages.sum()) + 1, max(1, int(pages.max()))
    # pages handed out in random order; the last one belongs to nobody and
    # fills the table's unused entries
    r = np.random.default_rng(seed)
    free = r.permutation(n_pages - 1)
    table = np.full((n, width), n_pages - 1, dtype=np.int32)
    at = 0
    for b in range(n):
        table[b, : pages[b]] = free[at : at + pages[b]]
        at += pages[b]
    s = {"table": torch.from_numpy(table).to(DEV), "lens": torch.from_numpy(lens.astype(np.int32)).to(DEV)}

    def pool():
        shape = (n_pages, hkv, ps, d) if case["order"] == "HND" else (n_pages, ps, hkv, d)
        t = torch.randn(shape, device=DEV, dtype=dt, generator=g)
        return t if case["order"] == "HND" else t.permute(0, 2, 1, 3)

    s["k"], s["v"] = pool(), pool()
    slots = width * ps
    # every slot's accumulated weight (float bits) and position, in one buffer: a
    # heavy-tailed weight, one slot in eight not yet attended to; positions as
    # earlier evictions leave them, distinct and in no order
    weight = torch.exp(1.5 * randn(n_pages, hkv, ps))
    weight *= torch.rand(n_pages, hkv, ps, device=DEV, generator=g) > 0.125
    s["meta"] = torch.stack([weight.view(torch.int32), torch.zeros_like(weight, dtype=torch.int32)])
    s["next_pos"] = s["lens"].clone()
    if case["op"] == "evict":
        live = torch.arange(slots, device=DEV) < s["lens"][:, None]
        key = torch.rand(n, hkv, slots, device=DEV, generator=g).masked_fill_(~live[:, None], 2.0)
        order = key.argsort(-1)
        place = torch.empty_like(order).scatter_(-1, order, torch.arange(slots, device=DEV).expand_as(order))
        odd = torch.randint(0, 2, place.shape, device=DEV, generator=g)
        page = s["table"].long().repeat_interleave(ps, 1)
        off = torch.arange(slots, device=DEV) % ps
        s["meta"][1][page[:, None], torch.arange(hkv, device=DEV)[:, None], off] = (2 * place + odd).int()
        s["meta"][1][n_pages - 1] = 0  # unused table entries met there
        s["next_pos"] = s["lens"] * 2
        s["meta0"] = s["meta"].clone()
    if case["op"] == "append":
        new = _new_tokens(case)
        total = sum(new)
        s["cu_new"] = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=DEV)
        s["qkv"] = randn(total, (hq + 2 * hkv) * d)
        s["q_norm"] = 0.8 + 0.4 * torch.rand(d, device=DEV, generator=g)
        s["k_norm"] = 0.8 + 0.4 * torch.rand(d, device=DEV, generator=g)
        length = int(lens.max())
        angle = torch.arange(length, device=DEV).double()[:, None] * THETA ** (
            -2.0 * torch.arange(d // 2, device=DEV).double() / d)
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        s["q_out"] = torch.empty(total, hq, d, device=DEV, dtype=dt)
    if case["op"] == "attention":
        s["q"] = (1.5 * randn(n, case["n_q"], hq, d)).to(dt)
        s["scale"] = d**-0.5
        s["out"] = torch.empty(n, case["n_q"], hq, d, device=DEV, dtype=dt)
        s["lse"] = torch.empty(n, case["n_q"], hq, device=DEV)
        if case["accumulate"]:
            s["meta0"] = s["meta"].clone()
    s["acc"], s["pos"] = s["meta"][0].view(torch.float32), s["meta"][1]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:  # the handle over the cache, and the workspace, that a program keeps
        import abra_b200 as A

        s["kv"] = A.PagedKV(s["k"], s["v"], s["table"], s["lens"], next_pos=s["next_pos"], pos=s["pos"],
                            acc=s["acc"])
        if case["op"] == "attention":
            s["ws"] = A.paged_attention_workspace(s["kv"], case["hq"], n_q=case["n_q"],
                                                  accumulate=case["accumulate"])
        if case["op"] == "evict":
            s["ws"] = A.paged_evict_workspace(s["kv"], case["budget"])
            s["new_lens"] = torch.empty_like(s["lens"])
    return s


# -------------------------------------------------------------------- run ---
def run(s):
    op = s["case"]["op"]
    if op != "append" and "meta0" in s:
        # weights and positions are updated in place: every pass starts from
        # the same ones
        s["meta"].copy_(s["meta0"])
    if op == "append":
        return _append_own(s) if own else _append(s)
    if op == "attention":
        return _attention_own(s) if own else _attention(s)
    return _evict_own(s) if own else _evict(s)


def _append_own(s):
    import abra_b200 as A

    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    q, k, v = s["qkv"].split((hq * d, hkv * d, hkv * d), 1)
    A.paged_append(s["kv"], k, v, q=q, q_out=s["q_out"], cu_new=s["cu_new"], q_norm=s["q_norm"],
                   k_norm=s["k_norm"], eps=EPS, rope=s["rope"])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"], "acc": s["acc"], "pos": s["pos"]}


def _attention_own(s):
    import abra_b200 as A

    c = s["case"]
    A.paged_attention(s["kv"], s["q"], s["scale"], out=s["out"], lse=s["lse"],
                      accumulate=c["accumulate"], workspace=s["ws"])
    out = {"out": s["out"], "lse": s["lse"]}
    return out | {"acc": s["acc"]} if c["accumulate"] else out


def _evict_own(s):
    import abra_b200 as A

    c = s["case"]
    A.paged_evict(s["kv"], c["budget"], n_sink=c["sink"], n_recent=c["recent"], new_lens=s["new_lens"],
                  workspace=s["ws"])
    return {"k": s["k"], "v": s["v"], "acc": s["acc"], "pos": s["pos"], "lens": s["new_lens"]}


def _norm_rope(x, weight, table):
    """RMSNorm over each head, then the rotation of the pairs (i, i + d/2)."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    lo, hi = x.chunk(2, -1)
    cos, sin = table[:, None, :, 0], table[:, None, :, 1]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _append(s):
    c = s["case"]
    n, total = c["n_seqs"], s["qkv"].shape[0]
    hq, hkv, d, ps = c["hq"], c["hkv"], c["d"], c["page"]
    cu = s["cu_new"].long()
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), cu[1:] - cu[:-1], output_size=total)
    back = cu[seq + 1] - torch.arange(total, device=DEV)  # 1 for a sequence's last token
    slot = s["lens"].long()[seq] - back
    at = s["next_pos"].long()[seq] - back
    q, k, v = s["qkv"].view(total, hq + 2 * hkv, d).split((hq, hkv, hkv), 1)
    rope = s["rope"][at]
    s["q_out"].copy_(_norm_rope(q, s["q_norm"], rope))
    page, off = s["table"].long()[seq, slot // ps], slot % ps
    s["k"][page, :, off] = _norm_rope(k, s["k_norm"], rope).to(s["k"].dtype)
    s["v"][page, :, off] = v.to(s["v"].dtype)
    s["pos"][page, :, off] = at.int()[:, None].expand(total, hkv)
    s["acc"][page, :, off] = torch.zeros(total, hkv, device=DEV)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"], "acc": s["acc"], "pos": s["pos"]}


def _rows(s, pool):
    """Every sequence's slots of a pool, [n_seqs, kv heads, slots, ...]."""
    ps = s["case"]["page"]
    slot = torch.arange(s["table"].shape[1] * ps, device=DEV)
    page = s["table"].long()[:, slot // ps]
    return pool[page[:, None], torch.arange(pool.shape[1], device=DEV)[:, None], slot % ps]


def _attention(s):
    c = s["case"]
    n, nq, hq, hkv, d = c["n_seqs"], c["n_q"], c["hq"], c["hkv"], c["d"]
    slot = torch.arange(s["table"].shape[1] * c["page"], device=DEV)
    lens = s["lens"].long()
    live = slot < lens[:, None]
    seen = slot < lens[:, None, None] - torch.arange(nq - 1, -1, -1, device=DEV)[:, None]  # [n, nq, slots]
    q = s["q"].float().view(n, nq, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4)
    k = _rows(s, s["k"]).float().masked_fill_(~live[:, None, :, None], 0.0)
    score = (q.reshape(n, hkv, -1, d) @ k.transpose(-1, -2)).view(n, hkv, nq, hq // hkv, -1) * s["scale"]
    del k
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min_(-3.0e38)
    w = (score - top).exp_()
    total = w.sum(-1, keepdim=True)
    s["lse"].copy_((top + total.log()).permute(0, 2, 1, 3, 4).reshape(n, nq, hq))
    w /= total.clamp_min_(1.0e-38)
    del score
    v = _rows(s, s["v"]).float().masked_fill_(~live[:, None, :, None], 0.0)
    out = (w.reshape(n, hkv, nq * (hq // hkv), -1) @ v).view(n, hkv, nq, hq // hkv, d)
    s["out"].copy_(out.permute(0, 2, 1, 3, 4).reshape(n, nq, hq, d))
    if not c["accumulate"]:
        return {"out": s["out"], "lse": s["lse"]}
    # a page has one owner, so adding at every slot of the table (zero past a
    # sequence's end) touches each live slot once
    page = s["table"].long()[:, slot // c["page"]]
    head = torch.arange(hkv, device=DEV)[:, None]
    s["acc"].index_put_((page[:, None], head, slot % c["page"]), w.sum((2, 3)), accumulate=True)
    return {"out": s["out"], "lse": s["lse"], "acc": s["acc"]}


def _evict(s):
    c = s["case"]
    ps, hkv, budget = c["page"], c["hkv"], c["budget"]
    lens = s["lens"].long()
    new = lens.clamp(max=budget)
    slot = torch.arange(s["table"].shape[1] * ps, device=DEV)
    live = (slot < lens[:, None])[:, None]
    acc, pos = _rows(s, s["acc"]), _rows(s, s["pos"]).long()
    hold = (pos < c["sink"]) | (pos >= (s["next_pos"].long() - c["recent"])[:, None, None])
    # three stable sorts, the least important first: by slot (as they lie), by
    # weight, by protection; dead slots last
    order = acc.argsort(dim=-1, descending=True, stable=True)
    first = (hold.int() - 2 * (~live).int()).gather(-1, order)
    order = order.gather(-1, first.argsort(dim=-1, descending=True, stable=True))
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order).contiguous())
    keep = (rank < budget) & live
    below = slot < new[:, None, None]
    hole, mover = ~keep & below, keep & ~below
    # the i-th hole takes the i-th mover; other slots keep what they have
    spare = slot.numel()
    place = torch.where(mover, mover.cumsum(-1) - 1, spare)
    source = torch.zeros(*place.shape[:2], spare + 1, dtype=torch.long, device=DEV)
    source.scatter_(-1, place, slot.expand_as(place))
    source = torch.where(hole, source.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), slot)
    page = s["table"].long()[:, slot // ps][:, None]
    head = torch.arange(hkv, device=DEV)[:, None]
    seq = torch.arange(c["n_seqs"], device=DEV)[:, None, None]
    from_page = s["table"].long()[seq, source // ps]
    where = (from_page, head, source % ps)
    moved = [s[x][where] for x in ("k", "v", "acc", "pos")]
    s["k"][page, head, slot % ps] = moved[0]
    s["v"][page, head, slot % ps] = moved[1]
    s["acc"][page, head, slot % ps] = moved[2]
    s["pos"][page, head, slot % ps] = moved[3]
    return {"k": s["k"], "v": s["v"], "acc": s["acc"], "pos": s["pos"], "lens": new.int()}


# ------------------------------------------------------------------- work ---
def work(case):
    lens = _lens(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        t = sum(_new_tokens(case))
        heads = (hq + 2 * hkv) * d
        # fp32 in, 16 bits out, a table row a token, weight and position of a slot
        return {"bytes": t * (heads * 6 + d * 4 + hkv * 8), "flops": t * (hq + hkv) * d * 8}
    if case["op"] == "attention":
        nq = case["n_q"]
        seen = sum(max(0, n - j) for n in lens for j in range(nq))
        b = sum(lens) * hkv * d * 4 + len(lens) * nq * hq * (d + 1) * 4
        if case["accumulate"]:
            b += sum(lens) * hkv * 8
        return {"bytes": b, "flops": 4 * d * hq * seen}
    # weight and position of every slot that is chosen among; of a sequence of
    # L slots with budget B, about B (L - B) / L kept rows lie above the budget
    # and move: a read and a write of both rows, the weight and the position
    over = [n for n in lens if n > case["budget"]]
    moves = sum(case["budget"] * (n - case["budget"]) / n for n in over)
    return {"bytes": hkv * (sum(over) * 8 + moves * 2 * (4 * d + 8)) + 8 * len(lens), "flops": hkv * sum(over)}


# ------------------------------------------------------------------ exact ---
def exact(case, seed):
    s = _inputs(case, seed)
    lens, table, ps = _lens(case), s["table"].cpu().numpy(), case["page"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    group = hq // hkv

    def where(b, slots):
        """Page and offset of some slots of sequence b."""
        return (torch.from_numpy(table[b][slots // ps].astype(np.int64)).to(DEV),
                torch.from_numpy(slots % ps).to(DEV))

    if case["op"] == "append":
        new = _new_tokens(case)
        k, v = s["k"].double(), s["v"].double()
        q_out = torch.empty(sum(new), hq, d, dtype=torch.float64, device=DEV)
        i = torch.arange(d // 2, device=DEV)

        def turned(x, w, positions):  # as a product of complex numbers
            x = x / ((x**2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
            unit = torch.view_as_complex(s["rope"].double())[positions][:, None]
            z = torch.complex(x[..., i], x[..., i + d // 2]) * unit
            return torch.cat([z.real, z.imag], -1)

        at = 0
        for b, m in enumerate(new):
            if not m:
                continue
            slots = np.arange(lens[b] - m, lens[b])
            x = s["qkv"][at : at + m].double().view(m, -1, d)
            page, off = where(b, slots)
            p = torch.from_numpy(slots).to(DEV)
            q_out[at : at + m] = turned(x[:, :hq], s["q_norm"], p)
            k[page, :, off] = turned(x[:, hq : hq + hkv], s["k_norm"], p)
            v[page, :, off] = x[:, hq + hkv :]
            s["acc"][page, :, off] = 0.0
            at += m
        return {"q": q_out, "k": k, "v": v, "acc": s["acc"], "pos": None}

    if case["op"] == "attention":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=DEV)
        acc = s["acc"].double()
        for b, n in enumerate(lens):
            if not n:
                continue
            page, off = where(b, np.arange(n))
            for h in range(hkv):
                k, v = s["k"][page, h, off].double(), s["v"][page, h, off].double()
                for j in range(case["n_q"]):
                    m = n - (case["n_q"] - 1 - j)
                    if m <= 0:
                        continue
                    q = s["q"][b, j, h * group : (h + 1) * group].double()
                    t = q @ k[:m].T * s["scale"]
                    p = torch.softmax(t, -1)
                    lse[b, j, h * group : (h + 1) * group] = torch.logsumexp(t, -1)
                    out[b, j, h * group : (h + 1) * group] = p @ v[:m]
                    acc[page[:m], h, off[:m]] += p.sum(0)
        out = {"out": out, "lse": lse}
        return out | {"acc": acc} if case["accumulate"] else out

    acc, pos = s["acc"].cpu().numpy(), s["pos"].cpu().numpy()
    next_pos = s["next_pos"].cpu().numpy()
    budget = case["budget"]
    for b, n in enumerate(lens):
        if n <= budget:
            continue
        slots = np.arange(n)
        pg, off = table[b][slots // ps], slots % ps
        source, target = [], []
        for h in range(hkv):
            a, p = acc[pg, h, off], pos[pg, h, off]
            held = (p < case["sink"]) | (p >= next_pos[b] - case["recent"])
            kept = np.lexsort((slots, -a, ~held))[:budget]
            mover = np.sort(kept[kept >= budget])
            hole = np.setdiff1d(np.arange(budget), kept)
            source.append(np.stack([np.full_like(mover, h), mover]))
            target.append(hole)
        (hs, src), dst = np.concatenate(source, 1), np.concatenate(target)
        hs = torch.from_numpy(hs).to(DEV)
        (p0, o0), (p1, o1) = where(b, src), where(b, dst)
        for x in (s["k"], s["v"], s["acc"], s["pos"]):
            x[p1, hs, o1] = x[p0, hs, o0]
    return {"k": s["k"], "v": s["v"], "acc": s["acc"], "pos": s["pos"],
            "lens": s["lens"].clamp(max=budget)}
