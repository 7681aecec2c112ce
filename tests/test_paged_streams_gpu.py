"""The paged calls on the default stream while another one is current."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as R
from test_paged_gpu import _kv, _no_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("handle", ["number", "object"])
def test_memory_of_calls_on_the_default_stream(dev, handle):
    """What a call allocates belongs to the stream it runs on, the default one by
    its number 0 among them."""
    import abra_b200 as A

    rng = np.random.default_rng(1)
    c = R.make_cache(rng, [300], 2, 64, 16, "f16")
    cd = R.to_dev(c, dev)
    kv = _kv(cd, acc=cd["acc"], pos=cd["pos"])
    q = torch.from_numpy(rng.standard_normal((1, 4, 64))).half().to(dev)
    row = torch.randn(1, 2 * 64, device=dev)
    want = A.paged_attention(kv, q, 0.1)
    torch.cuda.synchronize()
    stream = 0 if handle == "number" else torch.cuda.default_stream()
    with torch.cuda.stream(torch.cuda.Stream()):
        taken = [A.paged_attention(kv, q, 0.1, stream=stream), A.paged_attention_workspace(kv, 4, stream=stream),
                 A.paged_evict(kv, 300, stream=stream), A.paged_evict_workspace(kv, 100, stream=stream),
                 A.paged_append(kv, row, row, q=row, stream=stream)]
    _no_error()
    assert torch.equal(taken[0], want)
    pool = {}
    for seg in torch.cuda.memory_snapshot():
        at = seg["address"]
        for block in seg["blocks"]:
            pool[at] = seg["stream"]
            at += block["size"]
    assert [pool[t.data_ptr()] for t in taken] == [0] * 5
