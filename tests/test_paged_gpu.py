"""The paged cache's append, attention and eviction on a B200 against their
definitions in 64 bits (tests/paged_reference.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

EPS32 = 2.0**-24


def _kv(c, **kw):
    import abra_b200 as A

    return A.PagedKV(c["k"], c["v"], c["table"], c["lens"], **kw)


def _no_error():
    import abra_b200 as A

    torch.cuda.synchronize()
    assert A.device_error() == 0


def _check_attention(c, q, scale, out, lse, dtype, acc_before=None, acc_after=None):
    """Bounds.  A score is a dot of d exact 16-bit products in fp32 (d + 4
    roundings, a unit of 2^-23 each): ds.  The softmax weight is off by twice
    that, by its own rounding to 16 bits and by the sums' roundings (at most one
    for each sixteen slots and a fixed number for the joins); the result is
    rounded once more where it is stored in 16 bits."""
    want, lse64, weights, mag, dot = R.attention(c, q, scale)
    d = q.shape[-1]
    n = c["lens"].double().numpy()[:, None, None]
    ds = (d + 4) * 2 * EPS32 * abs(scale) * dot + 4 * EPS32
    sums = (n / 16 + 64) * 2 * EPS32
    got = out.cpu().double().numpy()
    unit = R.UNIT[dtype] if out.dtype != torch.float32 else EPS32
    tol = mag * (2 * ds + R.UNIT[dtype] + sums)[..., None] + unit * np.abs(want) + 2.0**-25
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    if lse is not None:
        got = lse.cpu().double().numpy()
        empty = np.isinf(lse64)
        assert (np.isneginf(got) == empty).all()
        tol = (ds + sums + 2 * EPS32 * np.abs(np.where(empty, 0, lse64)))[~empty]
        assert (np.abs(got[~empty] - lse64[~empty]) <= tol).all()
    if acc_after is None:
        return
    worst = (ds + sums + 2 * EPS32 * np.abs(np.where(np.isinf(lse64), 0, lse64))).max((1, 2))
    touched = torch.zeros(c["acc"].shape, dtype=torch.bool)
    for b, w in enumerate(weights):
        m = w.shape[1]
        before, after = (R.rows(c, x.cpu(), b, m).double().numpy() for x in (acc_before, acc_after))
        tol = w * (2 * worst[b] + 8 * EPS32) + 2 * EPS32 * (np.abs(before) + w)
        assert (np.abs(after - before - w) <= tol).all()
        t = np.arange(m)
        touched[c["table"][b].long()[t // c["page"]], :, torch.from_numpy(t % c["page"])] = True
    a, b = acc_before.cpu()[~touched], acc_after.cpu()[~touched]
    assert torch.equal(a.view(torch.int32), b.view(torch.int32)), "a weight changed beside the live slots"


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 100, 257, 700]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("hq,hkv,page,order", [(8, 8, 16, "HND"), (8, 2, 64, "NHD"), (6, 2, 8, "HND"),
                                               (16, 2, 24, "NHD"), (16, 1, 1, "HND"), (35, 5, 100, "HND"),
                                               (24, 1, 256, "HND")])
def test_attention_one_token(dev, dtype, d, hq, hkv, page, order):
    import abra_b200 as A

    rng = np.random.default_rng(d + hq + page)
    c = R.make_cache(rng, LENS, hkv, d, page, dtype, order)
    q = torch.from_numpy(2 * rng.standard_normal((len(LENS), 1, hq, d))).to(R.DTYPE[dtype])
    kv = _kv(R.to_dev(c, dev))
    lse = torch.full((len(LENS), 1, hq), float("nan"), device=dev)
    scale = d**-0.5
    out = A.paged_attention(kv, q.to(dev), scale, lse=lse)
    _no_error()
    assert out.dtype == q.dtype and out.shape == q.shape
    _check_attention(c, q, scale, out, lse, dtype)
    # fp32 results, and the same bits from a second call
    out32 = torch.full(q.shape, float("nan"), device=dev)
    A.paged_attention(kv, q.to(dev), scale, out=out32)
    _no_error()
    _check_attention(c, q, scale, out32, None, dtype)
    assert torch.equal(out32.to(q.dtype), out)


@pytest.mark.parametrize("dtype,d", [("f16", 128), ("bf16", 64), ("bf16", 96)])
@pytest.mark.parametrize("n_q", [2, 5, 16, 33])
@pytest.mark.parametrize("hq,hkv,page", [(2, 2, 16), (8, 2, 24), (16, 2, 64), (7, 1, 8)])
def test_attention_several_tokens(dev, dtype, d, n_q, hq, hkv, page):
    """Causal among the new tokens; queries before a short sequence's first
    slot see nothing."""
    import abra_b200 as A

    rng = np.random.default_rng(n_q * hq + page)
    lens = [0, 1, n_q - 1, n_q, n_q + 1, 48, 130, 400]
    c = R.make_cache(rng, lens, hkv, d, page, dtype)
    q = torch.from_numpy(2 * rng.standard_normal((len(lens), n_q, hq, d))).to(R.DTYPE[dtype])
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"])
    before = cd["acc"].clone()
    lse = torch.full((len(lens), n_q, hq), float("nan"), device=dev)
    out = A.paged_attention(kv, q.to(dev), 0.1, lse=lse, accumulate=True)
    _no_error()
    _check_attention(c, q, 0.1, out, lse, dtype, before, cd["acc"])


@pytest.mark.parametrize("dtype,d,hq,hkv,page,order", [("f16", 128, 32, 8, 16, "HND"), ("bf16", 64, 64, 8, 24, "NHD"),
                                                       ("bf16", 96, 3, 3, 100, "HND"), ("f16", 64, 40, 2, 8, "HND")])
def test_accumulated_weights(dev, dtype, d, hq, hkv, page, order):
    import abra_b200 as A

    rng = np.random.default_rng(7)
    lens = [300, 0, 1, 64, 1999]
    c = R.make_cache(rng, lens, hkv, d, page, dtype, order)
    q = torch.from_numpy(2 * rng.standard_normal((len(lens), 1, hq, d))).to(R.DTYPE[dtype])
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"])
    ws = A.paged_attention_workspace(kv, hq, accumulate=True)
    for _ in range(2):  # the second call adds to the first's
        before = cd["acc"].clone()
        out = A.paged_attention(kv, q[:, 0].to(dev), d**-0.5, accumulate=True, workspace=ws)
        _no_error()
        _check_attention(c, q, d**-0.5, out[:, None], None, dtype, before, cd["acc"])


@pytest.mark.parametrize("n,hq,hkv,n_q", [(20000, 8, 1, 1), (5000, 32, 8, 2)])
def test_attention_split_over_a_long_cache(dev, n, hq, hkv, n_q):
    import abra_b200 as A

    rng = np.random.default_rng(n)
    c = R.make_cache(rng, [n, 40], hkv, 128, 64, "f16")
    q = torch.from_numpy(2 * rng.standard_normal((2, n_q, hq, 128))).half()
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"])
    before = cd["acc"].clone()
    lse = torch.empty(2, n_q, hq, device=dev)
    out = A.paged_attention(kv, q.to(dev), 128**-0.5, lse=lse, accumulate=True)
    _no_error()
    _check_attention(c, q, 128**-0.5, out, lse, "f16", before, cd["acc"])


def test_attention_extreme_scores(dev):
    """Scores of +-30000 (one slot takes everything), falling and rising along
    the cache, and all equal: no overflow, no lost maximum."""
    import abra_b200 as A

    rng = np.random.default_rng(3)
    n, d = 1500, 128
    c = R.make_cache(rng, [n, n, n], 1, d, 16, "f16")
    for b, ramp in enumerate((np.linspace(-1, 1, n), np.linspace(1, -1, n), np.zeros(n))):
        t = np.arange(n)
        pg, off = c["table"][b].long()[t // 16], torch.from_numpy(t % 16)
        c["k"][pg, 0, off] = torch.from_numpy(np.repeat(ramp[:, None] * 15.0, d, 1)).half()
    q = torch.full((3, 1, 2, d), 16.0, dtype=torch.float16)
    kv = _kv(R.to_dev(c, dev))
    out = A.paged_attention(kv, q.to(dev), 1.0)
    _no_error()
    # exact products and sums of few bits: only the weights' rounding is left
    want, _, _, mag, _ = R.attention(c, q, 1.0)
    assert (np.abs(out.cpu().double().numpy() - want) <= 2.0**-9 * mag + 2.0**-10 * np.abs(want) + 2.0**-24).all()


@pytest.mark.parametrize("what", ["nan", "inf"])
def test_attention_masked_values_stay_out(dev, what):
    """A NaN or infinity in a newer token's key and value does not reach the
    queries that may not see it."""
    import abra_b200 as A

    rng = np.random.default_rng(4)
    n_q, d, hq = 4, 128, 4
    for n in (4, 7, 16, 18, 130):
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
        # and they are what they were without it, up to the split of the slots
        assert (got[:, :-1].float() - clean[:, :-1].float()).abs().max() <= 2.0**-7 * clean.float().abs().max()
        assert not torch.isfinite(got[:, -1]).all()


def test_attention_strides_and_streams(dev):
    """Queries and results inside wider rows, a table with a row stride, a
    stream of its own, the workspace shared by calls that follow one another."""
    import abra_b200 as A

    rng = np.random.default_rng(5)
    lens, hq, hkv, d = [77, 513, 3], 8, 2, 64
    c = R.make_cache(rng, lens, hkv, d, 16, "bf16")
    cd = R.to_dev(c, dev)
    wide = torch.full((3, cd["table"].shape[1] + 5), -1, dtype=torch.int32, device=dev)
    wide[:, : cd["table"].shape[1]] = cd["table"]
    cd["table"] = wide[:, : cd["table"].shape[1]]
    kv = _kv(cd)
    q = torch.from_numpy(rng.standard_normal((3, 1, hq, d))).bfloat16()
    big = torch.zeros(3, 1, hq * d + 128, dtype=torch.bfloat16, device=dev)
    inner = big[..., 64 : 64 + hq * d].unflatten(-1, (hq, d))
    inner.copy_(q)
    res = torch.full_like(big, 7.0)
    out = res[..., 8 : 8 + hq * d].unflatten(-1, (hq, d))
    ws = A.paged_attention_workspace(kv, hq)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            A.paged_attention(kv, inner, d**-0.5, out=out, workspace=ws)
    side.synchronize()
    _no_error()
    _check_attention(c, q, d**-0.5, out, None, "bf16")
    assert (res[..., :8] == 7).all() and (res[..., 8 + hq * d :] == 7).all()
    # the same on the side stream while the current one is another
    A.paged_attention(kv, inner, d**-0.5, out=out, workspace=ws, stream=side)
    side.synchronize()
    _check_attention(c, q, d**-0.5, out, None, "bf16")


def test_offsets_past_32_bits(dev):
    """Pools of more than 2^31 elements whose used pages lie at the far end."""
    import abra_b200 as A

    rng = np.random.default_rng(6)
    n, hkv, d, page = 300, 8, 128, 256
    n_pages = 2**31 // (hkv * d * page) + 8
    c = R.make_cache(rng, [n], hkv, d, page, "f16", spare=0)
    used = c["table"][0, : -(-n // page)].long()
    q = torch.from_numpy(rng.standard_normal((1, 1, 32, d))).half()
    k, v = (torch.empty(n_pages, hkv, page, d, dtype=torch.float16, device=dev) for _ in range(2))
    acc = torch.zeros(n_pages, hkv, page, device=dev)
    pos = torch.zeros(n_pages, hkv, page, dtype=torch.int32, device=dev)
    far = n_pages - 1 - torch.arange(len(used))
    for mine, theirs in ((k, "k"), (v, "v"), (pos, "pos")):
        mine[far.to(dev)] = c[theirs][used].to(dev)
    acc[far.to(dev)] = 0.0
    table = far.int()[None].to(dev)
    kv = A.PagedKV(k, v, table, c["lens"].to(dev), acc=acc, pos=pos)
    out = A.paged_attention(kv, q.to(dev), 0.1, accumulate=True)
    _no_error()
    c["acc"] = torch.zeros_like(c["acc"])
    after = torch.zeros_like(c["acc"])
    after[used] = acc[far.to(dev)].cpu()
    _check_attention(c, q, 0.1, out, None, "f16", c["acc"], after)
    # eviction and append at the same offsets
    a, p = (R.rows(c, x, 0, n).numpy() for x in (after, c["pos"]))
    k0 = k[far.to(dev)].clone()
    new = A.paged_evict(kv, 100, n_recent=10)
    _no_error()
    assert new.tolist() == [100]
    where = {int(u): i for i, u in enumerate(used.tolist())}
    for h in range(hkv):
        holes, movers = R.evict(a[h], p[h], 100, 0, n - 10)
        for t, u in zip(holes, movers):
            assert torch.equal(k[far[t // page], h, t % page], k0[where[int(used[u // page])], h, u % page])
    row = torch.randn(1, hkv * d, device=dev)
    A.paged_append(kv, row, row)
    _no_error()
    assert torch.equal(k[far[(n - 1) // page], :, (n - 1) % page], row.view(hkv, d).half())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tin", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,hq,hkv,page,order", [(128, 32, 8, 16, "HND"), (64, 5, 5, 24, "NHD"), (96, 6, 2, 1, "HND")])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 0, 40, 1], None])
def test_append(dev, dtype, tin, d, hq, hkv, page, order, new):
    """A head is 32-odd fp32 operations deep (the sum of squares, the root, the
    norm, the rotation): 64 units of 2^-24 of the pair's size, and the one
    rounding to 16 bits."""
    import abra_b200 as A

    rng = np.random.default_rng(d + page)
    lens = [1, 30, 40, 129]
    c = R.make_cache(rng, lens, hkv, d, page, dtype, order)
    next_pos = torch.tensor([1, 55, 40, 400], dtype=torch.int32)
    cu = np.concatenate([[0], np.cumsum([1] * 4 if new is None else [min(m, n) for m, n in zip(new, lens)])])
    total = int(cu[-1])
    fused = torch.from_numpy(rng.standard_normal((total, (hq + 2 * hkv) * d + 16))).to(tin)
    q, k, v = fused[:, : (hq + 2 * hkv) * d].split((hq * d, hkv * d, hkv * d), 1)
    q_norm, k_norm = (torch.from_numpy(rng.uniform(0.5, 1.5, d)).float() for _ in range(2))
    angle = rng.uniform(-3, 3, (400, d // 2))
    rope = torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], -1)).float()
    for norm, turn in ((True, True), (False, True), (True, False), (False, False)):
        cd = R.to_dev(c, dev)
        kv = _kv(cd, acc=cd["acc"], pos=cd["pos"], next_pos=next_pos.to(dev))
        fd = fused.to(dev)
        qd, kd, vd = fd[:, : (hq + 2 * hkv) * d].split((hq * d, hkv * d, hkv * d), 1)
        got = A.paged_append(kv, kd, vd, q=qd,
                             cu_new=None if new is None else torch.from_numpy(cu.astype(np.int32)).to(dev),
                             q_norm=q_norm.to(dev) if norm else None, k_norm=k_norm.to(dev) if norm else None,
                             eps=1e-5, rope=rope.to(dev) if turn else None)
        _no_error()
        want, rows = R.append(c, cu, q.reshape(total, hq, d), k.reshape(total, hkv, d), v.reshape(total, hkv, d),
                              q_norm if norm else None, k_norm if norm else None, 1e-5, rope if turn else None, next_pos)
        unit = R.UNIT[dtype]

        def close(x, y):
            x, size = x.cpu().double().numpy(), np.abs(y)
            pair = size + np.concatenate([size[..., d // 2 :], size[..., : d // 2]], -1)
            assert (np.abs(x - y) <= unit * size + 64 * EPS32 * 2 * pair + 2.0**-25).all()

        assert got.shape == (total, hq, d) and got.dtype == R.DTYPE[dtype]
        close(got, want)
        expect = {x: c[x].clone() for x in ("k", "v", "acc", "pos")}
        for (b, t), (kk, vv, at) in rows.items():
            pg, off = int(c["table"][b, t // page]), t % page
            close(cd["k"][pg, :, off], kk)
            close(cd["v"][pg, :, off], vv)
            expect["k"][pg, :, off], expect["v"][pg, :, off] = cd["k"][pg, :, off].cpu(), cd["v"][pg, :, off].cpu()
            expect["acc"][pg, :, off], expect["pos"][pg, :, off] = 0.0, at
        for x, e in expect.items():  # nothing else was written
            bits = torch.int16 if e.element_size() == 2 else torch.int32
            assert torch.equal(cd[x].cpu().contiguous().view(bits), e.contiguous().view(bits)), x


def test_append_keys_and_values_alone(dev):
    import abra_b200 as A

    rng = np.random.default_rng(8)
    c = R.make_cache(rng, [20, 5], 2, 64, 16, "f16")
    cd = R.to_dev(c, dev)
    kv = _kv(cd)
    k, v = (torch.randn(4, 2, 64, device=dev) for _ in range(2))
    assert A.paged_append(kv, k, v) is None
    _no_error()
    for b, n in enumerate((20, 5)):
        for i in range(2):
            pg, off = int(c["table"][b, (n - 2 + i) // 16]), (n - 2 + i) % 16
            assert torch.equal(cd["k"][pg, :, off], k[2 * b + i].half())
            assert torch.equal(cd["v"][pg, :, off], v[2 * b + i].half())


def _weights(kind, rng, shape):
    w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 3, shape).astype(np.float32)
    elif kind == "equal":
        w[:] = 0.25
    elif kind == "odd":
        w = rng.choice(np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 1.0, -1.0, 1e-42, -1e-42], np.float32), shape)
    return w


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("dtype,hkv,d,page,order", [("f16", 8, 128, 16, "HND"), ("bf16", 3, 64, 24, "NHD"), ("f16", 1, 96, 7, "HND")])
@pytest.mark.parametrize("budget,n_sink,n_recent", [(1, 0, 0), (64, 4, 32), (100, 0, 100), (255, 200, 55), (513, 3, 60)])
def test_evict(dev, kind, dtype, hkv, d, page, order, budget, n_sink, n_recent):
    import abra_b200 as A

    rng = np.random.default_rng(budget + page)
    lens = [0, 1, budget, budget + 1, 300, 2 * budget + 17, 1500]
    c = R.make_cache(rng, lens, hkv, d, page, dtype, order)
    next_pos = torch.tensor([2 * n for n in lens], dtype=torch.int32)
    for b, n in enumerate(lens):
        t = np.arange(n)
        pg, off = c["table"][b].long()[t // page], torch.from_numpy(t % page)
        c["acc"][pg, :, off] = torch.from_numpy(_weights(kind, rng, (n, hkv)))
        place = np.stack([rng.permutation(n) for _ in range(hkv)], 1).reshape(n, hkv)
        c["pos"][pg, :, off] = torch.from_numpy((2 * place + rng.integers(0, 2, (n, hkv))).astype(np.int32))
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"], pos=cd["pos"], next_pos=next_pos.to(dev))
    new = A.paged_evict(kv, budget, n_sink, n_recent)
    _no_error()
    assert new.tolist() == [min(n, budget) for n in lens]
    assert torch.equal(cd["lens"].cpu(), c["lens"])
    want = {x: c[x].clone() for x in ("k", "v", "acc", "pos")}
    for b, n in enumerate(lens):
        acc, pos = R.rows(c, c["acc"], b, n).numpy(), R.rows(c, c["pos"], b, n).numpy()
        for h in range(hkv):
            holes, movers = R.evict(acc[h], pos[h], budget, n_sink, 2 * n - n_recent)
            pt, pf = c["table"][b].long()[holes // page], c["table"][b].long()[movers // page]
            for x in want:
                want[x][pt, h, torch.from_numpy(holes % page)] = c[x][pf, h, torch.from_numpy(movers % page)]
    for x, w in want.items():
        bits = torch.int16 if w.element_size() == 2 else torch.int32
        assert torch.equal(cd[x].cpu().contiguous().view(bits), w.contiguous().view(bits)), x


def test_evict_more_protected_slots_than_the_budget(dev):
    """Positions that claim protection everywhere: the lowest slots stay."""
    import abra_b200 as A

    rng = np.random.default_rng(9)
    c = R.make_cache(rng, [200], 2, 64, 16, "f16")
    cd = R.to_dev(c, dev)
    cd["pos"].zero_()
    kv = _kv(cd, acc=cd["acc"], pos=cd["pos"])
    A.paged_evict(kv, 50, n_sink=1)
    _no_error()
    for x in ("k", "v"):
        assert torch.equal(cd[x].cpu().view(torch.int16), c[x].view(torch.int16))


@pytest.mark.parametrize("n,budget", [(70000, 20000), (140000, 139000)])
def test_evict_long(dev, n, budget):
    import abra_b200 as A

    rng = np.random.default_rng(n)
    hkv, d, page = 2, 64, 64
    c = R.make_cache(rng, [n, n // 3], hkv, d, page, "bf16")
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"], pos=cd["pos"])
    new = A.paged_evict(kv, budget, 4, 1000)
    _no_error()
    for b, m in enumerate((n, n // 3)):
        assert int(new[b]) == min(m, budget)
        acc, pos = R.rows(c, c["acc"], b, m).numpy(), R.rows(c, c["pos"], b, m).numpy()
        after = {x: R.rows(c, cd[x].cpu(), b, m) for x in ("k", "v", "acc", "pos")}
        before = {x: R.rows(c, c[x], b, m) for x in ("k", "v", "acc", "pos")}
        for h in range(hkv):
            holes, movers = R.evict(acc[h], pos[h], budget, 4, m - 1000)
            for x in after:
                w = before[x][h].clone()
                w[holes] = before[x][h][movers]
                assert torch.equal(after[x][h], w), x


def test_lengths_and_pages_outside_their_range_are_reported(dev):
    """The kernels' own checks: error bit 4, no access outside the pools, the
    other sequences' results untouched."""
    import abra_b200 as A

    rng = np.random.default_rng(10)
    lens, hq, hkv, d = [50, 33], 4, 2, 64
    c = R.make_cache(rng, lens, hkv, d, 16, "f16")
    c["k"], c["v"] = torch.nan_to_num(c["k"]), torch.nan_to_num(c["v"])
    q = torch.from_numpy(rng.standard_normal((2, 1, hq, d))).half()
    for fault in ("page", "long", "negative"):
        cd = R.to_dev(c, dev)
        if fault == "page":
            cd["table"][0, 1] = cd["k"].shape[0]
        else:
            cd["table"][0] = cd["table"][0, 0]
            cd["lens"][0] = 10**6 if fault == "long" else -3
        kv = _kv(cd, acc=cd["acc"], pos=cd["pos"])
        out = A.paged_attention(kv, q.to(dev), 0.125, accumulate=True)
        torch.cuda.synchronize()
        assert A.device_error() & 16, fault
        good = {**c, "lens": c["lens"][1:], "table": c["table"][1:]}
        _check_attention(good, q[1:], 0.125, out[1:], None, "f16")
        A.paged_evict(kv, 20)
        torch.cuda.synchronize()
        assert A.device_error() & 16, fault
        if fault != "negative":
            x = torch.randn(2 * 40, hkv * d, device=dev)
            A.paged_append(kv, x, x)  # more tokens than the second sequence has slots
            torch.cuda.synchronize()
            assert A.device_error() & 16, fault


def test_a_decode_loop_in_a_graph(dev):
    """Append, attention and a growing length captured once and replayed."""
    import abra_b200 as A

    torch.manual_seed(0)
    hq, hkv, d, page, n = 8, 2, 64, 16, 40
    k, v = (torch.zeros(8, hkv, page, d, dtype=torch.float16, device=dev) for _ in range(2))
    table = torch.tensor([[1, 4, 0], [7, 2, 5]], dtype=torch.int32, device=dev)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    kv = A.PagedKV(k, v, table, lens)
    xs = torch.randn(n, 2, (hq + 2 * hkv) * d, device=dev)
    x = xs[0].clone()
    out = torch.empty(2, hq, d, dtype=torch.float16, device=dev)
    q16 = torch.empty_like(out)
    ws = A.paged_attention_workspace(kv, hq)

    def step():
        lens.add_(1)
        a, b, c = x.split((hq * d, hkv * d, hkv * d), 1)
        A.paged_append(kv, b, c, q=a, q_out=q16)
        A.paged_attention(kv, q16, d**-0.5, out=out, workspace=ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    lens.zero_()
    got = []
    for t in range(n):
        x.copy_(xs[t])
        g.replay()
        got.append(out.clone())
    _no_error()
    q, kk, vv = xs.half().double().cpu().split((hq * d, hkv * d, hkv * d), 2)
    kk, vv, q = kk.view(n, 2, hkv, d), vv.view(n, 2, hkv, d), q.view(n, 2, hkv, hq // hkv, d)
    for t in range(n):
        s = torch.einsum("bhgd,nbhd->bhgn", q[t], kk[: t + 1]) * d**-0.5
        want = torch.einsum("bhgn,nbhd->bhgd", s.softmax(-1), vv[: t + 1]).reshape(2, hq, d)
        # two 16-bit roundings of values of a few units
        assert (got[t].cpu().double() - want).abs().max() <= 4 * 2.0**-10
