"""Paged attention beside one sequence's broken data keeps the other sequences'
results to the bit."""
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
