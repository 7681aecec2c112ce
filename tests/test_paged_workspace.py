"""What an accumulating attention asks of its workspace: scores of the slots that
its tables can name, or of the pools' where these are fewer."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from test_paged import _desc


@pytest.mark.parametrize("n_heads,n_q,padded", [(4, 1, 8), (32, 1, 16), (32, 4, 64), (32, 5, 128)])
def test_room_for_scores(n_heads, n_q, padded):
    """Two kv heads, pages of 16: rows a kv head rounded up to blocks, 4 bytes each."""
    from abra_b200 import _lib as L

    def more(**kw):  # what accumulation adds
        d = _desc(**kw)
        with_, without = (L.lib.abra_paged_attention_workspace(C.byref(d), n_heads, n_q, f) for f in (1, 0))
        assert with_ > without >= 0
        return with_ - without

    rows = 3 * n_heads * n_q * 4  # the rows' log-sum-exps
    slot = 2 * 16 * padded * 4
    for n_pages, pages in ((8, 8), (12, 12), (13, 12), (10**6, 12), (2**31 - 1, 12)):
        assert 0 <= more(n_pages=n_pages) - rows - pages * slot < 512


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,page", [("f16", 128, 16), ("bf16", 64, 24)])
@pytest.mark.parametrize("hq,n_q", [(4, 1), (2, 3), (24, 1), (4, 4), (40, 3)])
def test_weights_in_a_large_pool(dev, dtype, d, page, hq, n_q):
    """The same sequences in a pool that they fill and in one of many more pages."""
    import abra_b200 as A
    import paged_reference as R
    from test_paged_gpu import _check_attention, _kv, _no_error

    lens, sizes = [1500, 0, 700, 1, 4000], []
    for spare in (2, 4000):
        c = R.make_cache(np.random.default_rng(1), lens, 2, d, page, dtype, spare=spare)
        q = torch.from_numpy(np.random.default_rng(2).standard_normal((len(lens), n_q, 2 * hq, d))).to(R.DTYPE[dtype])
        cd = R.to_dev(c, dev)
        kv = _kv(cd, acc=cd["acc"])
        before = cd["acc"].clone()
        lse = torch.empty(len(lens), n_q, 2 * hq, device=dev)
        ws = A.paged_attention_workspace(kv, 2 * hq, n_q, accumulate=True).fill_(255)
        out = A.paged_attention(kv, q.to(dev), d**-0.5, lse=lse, accumulate=True, workspace=ws)
        _no_error()
        _check_attention(c, q, d**-0.5, out, lse, dtype, before, cd["acc"])
        sizes.append(ws.numel())
    assert sizes[1] < 6 * sizes[0]  # five tables as long as the longest sequence's
