"""Paged attention beside one sequence's broken data -- a page number outside the
pool, a NaN among its queries or keys -- keeps the other sequences' results to
the bit, and takes no longer for them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as R
from test_paged_gpu import _kv, _no_error

pytestmark = pytest.mark.gpu

ROWS = [(4, 1), (2, 3), (24, 1), (4, 4), (8, 8)]  # heads of one kv head, queries: two of the narrow kernel, three of the wide


def _run(dev, c, q, error=0):
    import abra_b200 as A

    cd = R.to_dev(c, dev)
    lse = torch.full(q.shape[:3], float("nan"), device=dev)
    out = A.paged_attention(_kv(cd, acc=cd["acc"]), q.to(dev), 0.125, lse=lse, accumulate=True)
    torch.cuda.synchronize()
    assert A.device_error() == error
    return out.cpu(), lse.cpu(), cd["acc"].cpu()


@pytest.mark.parametrize("dtype,d,page", [("f16", 64, 16), ("bf16", 128, 24)])
@pytest.mark.parametrize("hq,n_q", ROWS)
def test_weights_of_the_owner_of_page_zero(dev, dtype, d, page, hq, n_q):
    """A table entry outside the pool has no scores, and so changes none of the
    sequence that owns the pool's first page."""
    rng = np.random.default_rng(hq + d)
    lens = [400, 300]
    c = R.make_cache(rng, lens, 2, d, page, dtype)
    for x in ("k", "v"):  # what the bad entry reads instead is finite
        c[x] = torch.nan_to_num(c[x])
    c["acc"] = torch.nan_to_num(c["acc"])
    mine = int(c["table"][1, 0])  # now page 0
    for x in ("k", "v", "acc", "pos"):
        c[x][[0, mine]] = c[x][[mine, 0]]
    was = c["table"].clone()
    c["table"][was == mine], c["table"][was == 0] = 0, mine
    q = torch.from_numpy(2 * rng.standard_normal((2, n_q, hq * 2, d))).to(R.DTYPE[dtype])
    good = _run(dev, c, q)
    bad = dict(c, table=c["table"].clone())
    for entry, to in ((0, c["k"].shape[0]), (3, -1), (5, 2**31 - 1)):
        bad["table"][0, entry] = to
    got = _run(dev, bad, q, error=16)
    assert torch.equal(got[0][1], good[0][1]) and torch.equal(got[1][1], good[1][1])
    assert torch.equal(R.rows(c, got[2], 1, lens[1]), R.rows(c, good[2], 1, lens[1]))


@pytest.mark.parametrize("dtype,d,page", [("f16", 128, 16), ("bf16", 64, 24)])
@pytest.mark.parametrize("hq,n_q", ROWS)
@pytest.mark.parametrize("where", ["query", "key"])
def test_nan_beside_healthy_sequences(dev, dtype, d, page, hq, n_q, where):
    """A NaN in one query makes its own row NaN, one in a key the rows of its kv
    head that see it; the other kv head and the other sequences do not notice."""
    rng = np.random.default_rng(hq + d)
    lens, hkv = [700, 6000, 2500, 40], 2
    c = R.make_cache(rng, lens, hkv, d, page, dtype)
    c["acc"] = torch.nan_to_num(c["acc"])
    q = torch.from_numpy(2 * rng.standard_normal((len(lens), n_q, hq * hkv, d))).to(R.DTYPE[dtype])
    good = _run(dev, c, q)
    bad, q_bad = dict(c, k=c["k"].clone()), q.clone()
    hit = torch.zeros(n_q, hq * hkv, dtype=torch.bool)  # the rows of sequence 1 that become NaN
    if where == "query":
        q_bad[1, n_q - 1, hq - 1, 5] = float("nan")
        hit[n_q - 1, hq - 1] = True
    else:
        bad["k"][int(c["table"][1, 100 // page]), 0, 100 % page, 7] = float("nan")
        hit[:, :hq] = True
    out, lse, acc = _run(dev, bad, q_bad)
    others = [0, 2, 3]
    assert torch.equal(out[others], good[0][others]) and torch.equal(lse[others], good[1][others])
    assert torch.equal(out[1, :, hq:], good[0][1, :, hq:]) and torch.equal(lse[1, :, hq:], good[1][1, :, hq:])
    assert torch.isnan(out[1][hit]).all() and torch.isnan(lse[1][hit]).all()
    assert torch.isfinite(out[1][~hit]).all() and torch.isfinite(lse[1][~hit]).all()
    for b, n in enumerate(lens):
        now, was = R.rows(c, acc, b, n), R.rows(c, good[2], b, n)
        assert torch.equal(now[1], was[1])
        assert torch.isnan(now[0][: n - n_q + 1]).all() if b == 1 else torch.equal(now[0], was[0])


@pytest.mark.parametrize("dtype,d", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("hq,n_q", [(2, 3), (4, 4), (8, 8), (3, 2)])
def test_weights_of_slots_that_a_nan_query_does_not_see(dev, dtype, d, hq, n_q):
    """The newest slots' weights come from the queries that see them: within
    their roundings (a row's maximum may be raised at other slots) what they are
    with a first query of numbers."""
    rng = np.random.default_rng(hq)
    lens = [n_q, 50, 3000]
    c = R.make_cache(rng, lens, 1, d, 16, dtype)
    c["acc"] = torch.zeros_like(c["acc"])
    q = torch.from_numpy(2 * rng.standard_normal((len(lens), n_q, hq, d))).to(R.DTYPE[dtype])
    bad, none = q.clone(), q.clone()
    bad[:, 0, 0] = float("nan")
    got = _run(dev, c, bad)[2]
    _, _, weights, _, _ = R.attention(c, none, 0.125)
    for b, n in enumerate(lens):
        new = R.rows(c, got, b, n)[0]
        assert torch.isnan(new[: n - n_q + 1]).all()
        want = torch.from_numpy(weights[b][0, n - n_q + 1 :])  # the first query adds nothing to them
        assert ((new[n - n_q + 1 :].double() - want).abs() <= 1e-4 * want).all()


@pytest.mark.parametrize("hq,n_q", [(4, 1), (8, 8)])
@pytest.mark.parametrize("where", ["query", "value"])
def test_what_is_not_finite_costs_little(dev, hq, n_q, where):
    """NaNs in every query change nothing about the work; an infinity among every
    sequence's values has each piece look through its values once more, half of
    what it has read already.  Four times the call without them is enough for
    either, and thousands of times less than a look at each slot in turn."""
    import abra_b200 as A

    n_seqs, n, hkv, d, page = 8, 4096, 4, 128, 64
    g = torch.Generator(device=dev).manual_seed(0)
    k, v = (torch.randn(n_seqs * n // page, hkv, page, d, device=dev, generator=g).half() for _ in range(2))
    table = torch.arange(n_seqs * n // page, dtype=torch.int32, device=dev).view(n_seqs, -1)
    kv = A.PagedKV(k, v, table, torch.full((n_seqs,), n, dtype=torch.int32, device=dev))
    q = torch.randn(n_seqs, n_q, hq * hkv, d, device=dev, generator=g).half()
    out, ws = torch.empty_like(q), A.paged_attention_workspace(kv, hq * hkv, n_q)

    def took():
        times = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(5):
                A.paged_attention(kv, q, 0.1, out=out, workspace=ws)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    took()
    before = took()
    if where == "query":
        q.fill_(float("nan"))
    else:
        v[table[:, 1].long(), :, 3] = float("inf")
    after = took()
    _no_error()
    assert torch.isnan(out).all() if where == "query" else torch.isinf(out).all()
    assert after <= 4 * before, (before, after)


def test_queries_and_results_in_the_same_rows(dev):
    """Columns of one wider tensor, the same as in tensors of their own."""
    import abra_b200 as A

    rng = np.random.default_rng(5)
    lens, hq, d = [70, 300, 9], 4, 64
    c = R.make_cache(rng, lens, 2, d, 16, "f16")
    kv = _kv(R.to_dev(c, dev))
    rows = torch.zeros(3, 2 * hq * d + 64, dtype=torch.float16, device=dev)
    q, out = rows[:, : hq * d].unflatten(1, (hq, d)), rows[:, hq * d : 2 * hq * d].unflatten(1, (hq, d))
    q.copy_(torch.from_numpy(rng.standard_normal((3, hq, d))))
    want = A.paged_attention(kv, q.clone(), 0.1)
    was = q.clone()
    assert A.paged_attention(kv, q, 0.1, out=out) is out
    _no_error()
    assert torch.equal(out, want) and torch.equal(q, was) and (rows[:, 2 * hq * d :] == 0).all()
    with pytest.raises(ValueError, match="share"):
        A.paged_attention(kv, q, 0.1, out=rows[:, 8 : 8 + hq * d].unflatten(1, (hq, d)))
