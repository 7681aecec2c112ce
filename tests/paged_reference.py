"""The paged-cache operators in 64 bits, slot by slot from their definitions,
and the caches the tests run them on (CPU tensors)."""
from __future__ import annotations

import numpy as np
import torch

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f16": 2.0**-11, "bf16": 2.0**-8}  # half a unit in the last place, relative


def make_cache(rng, lens, hkv, d, page, dtype, order="HND", spare=2):
    """A cache of random rows: pages in random order, `spare` pages in nobody's
    hands.  Whatever no sequence may read is poison: NaN in the unused slots and
    pages, page numbers outside the pool in the unused table entries."""
    need = [-(-n // page) for n in lens]
    n_pages, width = sum(need) + spare, max(1, max(need, default=1)) + 1
    order_of = rng.permutation(n_pages)
    table = np.full((len(lens), width), -7, dtype=np.int32)
    table[:, -1] = 2**30
    shape = (n_pages, hkv, page, d)
    k = np.full(shape, np.nan)
    v = np.full(shape, np.nan)
    acc = np.full(shape[:3], np.nan, dtype=np.float32)
    pos = np.full(shape[:3], -(2**31), dtype=np.int32)
    at = 0
    for b, n in enumerate(lens):
        table[b, : need[b]] = order_of[at : at + need[b]]
        at += need[b]
        t = np.arange(n)
        pg, off = table[b][t // page], t % page
        k[pg, :, off] = rng.standard_normal((n, hkv, d))
        v[pg, :, off] = rng.standard_normal((n, hkv, d))
        acc[pg, :, off] = np.exp(rng.standard_normal((n, hkv)))
        pos[pg, :, off] = t[:, None]
    dt = DTYPE[dtype]

    def pool(x):
        x = torch.from_numpy(x).to(dt)
        return x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) if order == "NHD" else x

    return {"k": pool(k), "v": pool(v), "acc": torch.from_numpy(acc), "pos": torch.from_numpy(pos),
            "table": torch.from_numpy(table), "lens": torch.tensor(lens, dtype=torch.int32), "page": page}


def to_dev(c, dev):
    """The cache's tensors on the device, with their strides."""
    out = {}
    for name, t in c.items():
        if isinstance(t, torch.Tensor):
            u = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev)
            out[name] = u.copy_(t)
        else:
            out[name] = t
    return out


def rows(c, x, b, n):
    """Slots 0..n-1 of sequence b of a pool or of acc/pos: [heads, n, ...]."""
    t = np.arange(n)
    pg = torch.from_numpy(c["table"][b].numpy()[t // c["page"]].astype(np.int64))
    return x[pg, :, torch.from_numpy(t % c["page"])].transpose(0, 1)


def attention(c, q, scale):
    """out, lse, the weights [heads, slots] of each sequence, and for each
    output the bound's ingredients: sum p|v| and the largest sum |q||k|."""
    n_seqs, n_q, hq, d = q.shape
    hkv = c["k"].shape[1]
    g = hq // hkv
    out = np.zeros(q.shape)
    lse = np.full(q.shape[:3], -np.inf)
    mag, dot = np.zeros(q.shape), np.zeros(q.shape[:3])
    weights = []
    for b in range(n_seqs):
        n = int(c["lens"][b])
        k, v = rows(c, c["k"], b, n).double().numpy(), rows(c, c["v"], b, n).double().numpy()
        w = np.zeros((n_q, hq, n))
        for j in range(n_q):
            m = n - (n_q - 1 - j)
            if m <= 0:
                continue
            for h in range(hq):
                x = q[b, j, h].double().numpy()
                s = scale * (k[h // g, :m] @ x)
                top = s.max()
                e = np.exp(s - top)
                lse[b, j, h] = top + np.log(e.sum())
                w[j, h, :m] = e / e.sum()
                out[b, j, h] = w[j, h, :m] @ v[h // g, :m]
                mag[b, j, h] = w[j, h, :m] @ np.abs(v[h // g, :m])
                dot[b, j, h] = (np.abs(k[h // g, :m]) @ np.abs(x)).max()
        weights.append(w.sum(0).reshape(hkv, g, n).sum(1))
    return out, lse, weights, mag, dot


def append(c, cu, q, k, v, q_norm, k_norm, eps, rope, next_pos):
    """The queries, and {(sequence, slot): (k, v, position)} of the new tokens."""
    d = k.shape[-1]

    def turned(x, w, at):
        x = x.double().numpy()
        if w is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.double().numpy()
        if rope is not None:
            cos, sin = rope[at].double().numpy().T
            lo, hi = x[..., : d // 2], x[..., d // 2 :]
            x = np.concatenate([lo * cos - hi * sin, hi * cos + lo * sin], -1)
        return x

    qs, new = [], {}
    for b in range(len(cu) - 1):
        for t in range(cu[b], cu[b + 1]):
            back = cu[b + 1] - t
            at = int(next_pos[b]) - back
            if q is not None:
                qs.append(turned(q[t], q_norm, at))
            new[b, int(c["lens"][b]) - back] = (turned(k[t], k_norm, at), v[t].double().numpy(), at)
    return np.array(qs), new


def evict(acc, pos, budget, n_sink, recent_from):
    """(holes, movers) of one sequence's kv head."""
    n = len(acc)
    if n <= budget:
        return np.zeros(0, int), np.zeros(0, int)
    a = np.where(np.isnan(acc), -np.inf, acc) + 0.0
    held = (pos < n_sink) | (pos >= recent_from)
    slot = np.arange(n)
    kept = np.zeros(n, bool)
    # protected first, then by weight, then by slot
    kept[np.lexsort((slot, -a, ~held))[:budget]] = True
    return slot[~kept & (slot < budget)], slot[kept & (slot >= budget)]
