"""The paged operators where their inner paths change: many rows a kv head
(tensor memory), hundreds of sequences, thousands of new tokens, caches longer
than a cluster's shared memory."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as R
from test_paged_gpu import EPS32, _check_attention, _kv, _no_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d,order", [("f16", 128, "HND"), ("bf16", 64, "NHD"), ("bf16", 96, "HND")])
@pytest.mark.parametrize("hq,hkv,n_q,page", [(9, 1, 1, 16), (32, 2, 1, 64), (17, 1, 1, 7), (8, 2, 4, 24), (40, 1, 3, 16),
                                             (6, 2, 40, 100)])
def test_many_rows(dev, dtype, d, order, hq, hkv, n_q, page):
    import abra_b200 as A

    rng = np.random.default_rng(hq * n_q + d)
    lens = [0, 1, 127, 128, 129, 300, 1000]
    c = R.make_cache(rng, lens, hkv, d, page, dtype, order)
    q = torch.from_numpy(2 * rng.standard_normal((len(lens), n_q, hq, d))).to(R.DTYPE[dtype])
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"])
    before = cd["acc"].clone()
    lse = torch.full((len(lens), n_q, hq), float("nan"), device=dev)
    out = A.paged_attention(kv, q.to(dev), d**-0.5, lse=lse, accumulate=True)
    _no_error()
    _check_attention(c, q, d**-0.5, out, lse, dtype, before, cd["acc"])
    out32 = torch.full(q.shape, float("nan"), device=dev)
    A.paged_attention(kv, q.to(dev), d**-0.5, out=out32)
    _no_error()
    _check_attention(c, q, d**-0.5, out32, None, dtype)
    assert torch.equal(out32.to(q.dtype), out)


@pytest.mark.parametrize("n,hq,hkv,n_q", [(9000, 16, 1, 1), (6000, 8, 2, 8), (3000, 64, 8, 16)])
def test_many_rows_split_over_a_long_cache(dev, n, hq, hkv, n_q):
    import abra_b200 as A

    rng = np.random.default_rng(n)
    c = R.make_cache(rng, [n, 40], hkv, 128, 64, "bf16")
    q = torch.from_numpy(2 * rng.standard_normal((2, n_q, hq, 128))).bfloat16()
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"])
    before = cd["acc"].clone()
    lse = torch.empty(2, n_q, hq, device=dev)
    out = A.paged_attention(kv, q.to(dev), 128**-0.5, lse=lse, accumulate=True)
    _no_error()
    _check_attention(c, q, 128**-0.5, out, lse, "bf16", before, cd["acc"])


def test_many_rows_extreme_scores(dev):
    """Scores of +-30000 rising, falling and all equal along the cache."""
    import abra_b200 as A

    rng = np.random.default_rng(3)
    n, d, hq = 1500, 128, 24
    c = R.make_cache(rng, [n, n, n], 1, d, 16, "f16")
    for b, ramp in enumerate((np.linspace(-1, 1, n), np.linspace(1, -1, n), np.zeros(n))):
        t = np.arange(n)
        pg, off = c["table"][b].long()[t // 16], torch.from_numpy(t % 16)
        c["k"][pg, 0, off] = torch.from_numpy(np.repeat(ramp[:, None] * 15.0, d, 1)).half()
    q = torch.full((3, 1, hq, d), 16.0, dtype=torch.float16)
    out = A.paged_attention(_kv(R.to_dev(c, dev)), q.to(dev), 1.0)
    _no_error()
    want, _, _, mag, _ = R.attention(c, q, 1.0)
    assert (np.abs(out.cpu().double().numpy() - want) <= 2.0**-9 * mag + 2.0**-10 * np.abs(want) + 2.0**-24).all()


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("d", [64, 128])
def test_many_rows_masked_values_stay_out(dev, what, d):
    import abra_b200 as A

    rng = np.random.default_rng(4)
    n_q, hq = 6, 4
    for n in (6, 7, 16, 130, 256, 700):
        c = R.make_cache(rng, [n], 1, d, 16, "bf16")
        q = torch.from_numpy(rng.standard_normal((1, n_q, hq, d))).bfloat16()
        bad = dict(c)
        bad["k"], bad["v"] = c["k"].clone(), c["v"].clone()
        pg, off = int(c["table"][0, (n - 1) // 16]), (n - 1) % 16
        for x in ("k", "v"):
            bad[x][pg, 0, off] = float(what)
        clean = A.paged_attention(_kv(R.to_dev(c, dev)), q.to(dev), 0.1)
        got = A.paged_attention(_kv(R.to_dev(bad, dev)), q.to(dev), 0.1)
        _no_error()
        assert torch.isfinite(got[:, :-1]).all()
        assert (got[:, :-1].float() - clean[:, :-1].float()).abs().max() <= 2.0**-7 * clean.float().abs().max()
        assert not torch.isfinite(got[:, -1]).all()


@pytest.mark.parametrize("hq,n_q", [(4, 1), (4, 8)])
def test_hundreds_of_sequences(dev, hq, n_q):
    import abra_b200 as A

    rng = np.random.default_rng(11)
    lens = [int(x) for x in rng.integers(0, 60, 400)]
    lens[0] = lens[399] = 0
    lens[200], lens[257] = 500, 129
    c = R.make_cache(rng, lens, 2, 64, 16, "f16")
    q = torch.from_numpy(rng.standard_normal((len(lens), n_q, hq, 64))).half()
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"])
    before = cd["acc"].clone()
    lse = torch.empty(len(lens), n_q, hq, device=dev)
    out = A.paged_attention(kv, q.to(dev), 0.125, lse=lse, accumulate=True)
    _no_error()
    _check_attention(c, q, 0.125, out, lse, "f16", before, cd["acc"])


def test_thousands_of_new_tokens(dev):
    """300 prompts, some empty, 4 tokens a CTA whose sequences change inside it."""
    import abra_b200 as A

    rng = np.random.default_rng(12)
    hq, hkv, d, page = 6, 3, 64, 16
    new = [int(x) for x in rng.integers(0, 12, 300)]
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, 40, 300))]
    c = R.make_cache(rng, lens, hkv, d, page, "bf16")
    cu = np.concatenate([[0], np.cumsum(new)])
    total = int(cu[-1])
    assert total > 1300
    x = torch.from_numpy(rng.standard_normal((total, (hq + 2 * hkv) * d))).float()
    q, k, v = x.split((hq * d, hkv * d, hkv * d), 1)
    angle = rng.uniform(-3, 3, (64, d // 2))
    rope = torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], -1)).float()
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"], pos=cd["pos"])
    xd = x.to(dev)
    qd, kd, vd = xd.split((hq * d, hkv * d, hkv * d), 1)
    got = A.paged_append(kv, kd, vd, q=qd, cu_new=torch.from_numpy(cu.astype(np.int32)).to(dev), rope=rope.to(dev))
    _no_error()
    want, rows = R.append(c, cu, q.reshape(total, hq, d), k.reshape(total, hkv, d), v.reshape(total, hkv, d), None, None, 0.0,
                          rope, c["lens"])
    tol = 2.0**-8 * np.abs(want) + 64 * EPS32 * 2 * np.abs(want).max() + 2.0**-25
    assert (np.abs(got.cpu().double().numpy() - want) <= tol).all()
    kc, vc, pos = cd["k"].cpu().double().numpy(), cd["v"].cpu().double().numpy(), cd["pos"].cpu().numpy()
    for (b, t), (kk, vv, at) in rows.items():
        pg, off = int(c["table"][b, t // page]), t % page
        assert (np.abs(kc[pg, :, off] - kk) <= 2.0**-8 * np.abs(kk) + 128 * EPS32 * np.abs(kk).max() + 2.0**-25).all()
        assert (np.abs(vc[pg, :, off] - vv) <= 2.0**-8 * np.abs(vv) + 2.0**-25).all()
        assert (pos[pg, :, off] == at).all()


@pytest.mark.parametrize("n,budget", [(360000, 9000), (330000, 329000)])
def test_evict_from_a_cache_beyond_shared_memory(dev, n, budget):
    import abra_b200 as A

    rng = np.random.default_rng(n)
    page, d = 256, 64
    pages = -(-n // page)
    order = torch.from_numpy(rng.permutation(pages).astype(np.int32))
    k, v = (torch.randn(pages, 1, page, d, device=dev).half() for _ in range(2))
    weight = np.exp(rng.standard_normal((pages, 1, page))).astype(np.float32)
    weight[rng.random(weight.shape) < 0.3] = 0.0
    acc = torch.from_numpy(weight).to(dev)
    slot = np.arange(n)
    pg, off = order.numpy()[slot // page], slot % page
    pos = np.zeros((pages, 1, page), np.int32)
    pos[pg, 0, off] = slot
    pos = torch.from_numpy(pos).to(dev)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    kv = A.PagedKV(k, v, order[None].to(dev), lens, acc=acc, pos=pos)
    k0, v0 = k.clone(), v.clone()
    assert A.paged_evict(kv, budget, 16, 1000).tolist() == [budget]
    _no_error()
    holes, movers = R.evict(weight[pg, 0, off], slot.astype(np.int32), budget, 16, n - 1000)
    assert len(holes) > 100
    for now, was in ((k, k0), (v, v0)):
        want = was.clone()
        want[pg[holes], 0, off[holes]] = was[pg[movers], 0, off[movers]]
        assert torch.equal(now, want)
    want = np.zeros_like(weight)
    want[:] = weight
    want[pg[holes], 0, off[holes]] = weight[pg[movers], 0, off[movers]]
    assert np.array_equal(acc.cpu().numpy(), want)


@pytest.mark.parametrize("scale", [0.0, -0.1])
@pytest.mark.parametrize("hq,n_q", [(4, 1), (4, 2), (12, 3)])
def test_scales_of_zero_and_below(dev, scale, hq, n_q):
    """Zero: the mean of the seen rows."""
    import abra_b200 as A

    rng = np.random.default_rng(13)
    lens = [1, 2, 17, 200]
    c = R.make_cache(rng, lens, 1, 64, 16, "f16")
    q = torch.from_numpy(rng.standard_normal((len(lens), n_q, hq, 64))).half()
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"])
    before = cd["acc"].clone()
    lse = torch.empty(len(lens), n_q, hq, device=dev)
    out = A.paged_attention(kv, q.to(dev), scale, lse=lse, accumulate=True)
    _no_error()
    _check_attention(c, q, scale, out, lse, "f16", before, cd["acc"])


def test_results_do_not_go_over_the_queries(dev):
    import abra_b200 as A

    rng = np.random.default_rng(14)
    c = R.make_cache(rng, [20], 1, 64, 16, "f16")
    q = torch.zeros(1, 1, 2, 64, dtype=torch.float16, device=dev)
    with pytest.raises(ValueError, match="memory"):
        A.paged_attention(_kv(R.to_dev(c, dev)), q, 0.1, out=q)


@pytest.mark.parametrize("dtype,d", [("f16", 128), ("bf16", 96)])
@pytest.mark.parametrize("hq,n_q", [(4, 1), (4, 2), (3, 7), (24, 1), (8, 8), (30, 4)])
def test_visible_infinities(dev, dtype, d, hq, n_q):
    """An infinity or NaN among the values reaches its own element of the
    queries that see the slot, as the sum of the formula does, and nothing else:
    the other elements are the bits of a cache without it."""
    import abra_b200 as A

    rng = np.random.default_rng(hq + n_q)
    lens = [5, 70, 200, 9000]
    c = R.make_cache(rng, lens, 1, d, 16, dtype)
    q = torch.from_numpy(2 * rng.standard_normal((len(lens), n_q, hq, d))).to(R.DTYPE[dtype])
    bad = dict(c)
    bad["v"], c["v"] = c["v"].clone(), c["v"].clone()
    add = np.zeros((len(lens), max(lens), d))  # what a slot adds beside finite values
    inf, nan = np.inf, np.nan
    for b, n in enumerate(lens):
        for e, t, x in ((0, 0, inf), (1, n - 1, -inf), (2, n // 2, nan), (3, n - 2, inf), (3, n // 3, inf), (4, n - 1, inf),
                        (4, n // 3, -inf), (d - 1, n - 1, nan), (d - 2, n // 2, -inf)):
            pg, off = int(c["table"][b, t // 16]), t % 16
            bad["v"][pg, 0, off, e], c["v"][pg, 0, off, e] = x, 0.0
            add[b, t, e] = x
    for out_type in (R.DTYPE[dtype], torch.float32):
        clean, got = (A.paged_attention(_kv(R.to_dev(x, dev)), q.to(dev), d**-0.5,
                                        out=torch.empty(q.shape, dtype=out_type, device=dev)).cpu() for x in (c, bad))
        _no_error()
        assert torch.isfinite(clean).all()
        for b, n in enumerate(lens):
            for j in range(n_q):
                seen = max(0, n - (n_q - 1 - j))
                want = clean[b, j].double().numpy() + add[b, :seen].sum(0)
                assert np.array_equal(got[b, j].double().numpy(), want, equal_nan=True), (b, j)


def test_memory_on_the_calls_stream(dev, monkeypatch):
    """Results and workspaces that a call allocates come from the pool of the
    stream it runs on, where the memory is reused in the order of its work."""
    import abra_b200 as A
    from abra_b200 import paged

    rng = np.random.default_rng(1)
    c = R.make_cache(rng, [300], 2, 64, 16, "f16")
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"], pos=cd["pos"])
    q = torch.from_numpy(rng.standard_normal((1, 4, 64))).half().to(dev)
    row = torch.randn(1, 2 * 64, device=dev)
    taken = []
    bytes_of = paged._bytes
    monkeypatch.setattr(paged, "_bytes", lambda ws, kv: taken.append(ws) or bytes_of(ws, kv))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        taken += [A.paged_attention(kv, q, 0.1, accumulate=True, stream=stream), A.paged_evict(kv, 100, stream=stream),
                  A.paged_append(kv, row, row, q=row, stream=stream)]
    _no_error()
    pool = {}
    for seg in torch.cuda.memory_snapshot():
        at = seg["address"]
        for block in seg["blocks"]:
            pool[at] = seg["stream"]
            at += block["size"]
    assert len(taken) == 10 and [pool[t.data_ptr()] for t in taken] == [side.cuda_stream] * 10
