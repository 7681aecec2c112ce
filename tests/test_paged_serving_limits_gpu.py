"""The serving example at its limits: a call that does not fit changes nothing."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_paged_serving_gpu import ex  # noqa: F401

pytestmark = pytest.mark.gpu


def _state(d):
    return list(d.lens), list(d.seen), [list(p) for p in d.pages], list(d.free), d.state.tolist(), d.table.tolist()


@pytest.fixture(scope="module")
def weights(ex):  # noqa: F811
    return ex.random_weights(ex.Shape(layers=1), 5)


def test_a_pool_that_is_used_up(dev, ex, weights):  # noqa: F811
    import abra_b200 as A

    shape, rng = ex.Shape(layers=1), np.random.default_rng(1)
    prompts = [rng.integers(0, shape.vocab, n) for n in (44, 48)]
    token = torch.as_tensor(rng.integers(0, shape.vocab, (2, 1)), device=dev)
    d, other = (ex.PagedDecoder(shape, weights, n_pages=n) for n in (6, 64))
    for x in (d, other):
        for p in prompts:
            x.feed(x.add(), p)
    was = _state(d)
    with pytest.raises(RuntimeError, match="used up"):
        d.forward(token, 0)  # room for the first conversation's token, none for the second's
    assert _state(d) == was
    # the first goes on as if nothing had been asked
    assert torch.equal(d.forward(token[:1], 0), other.forward(token[:1], 0))
    torch.cuda.synchronize()
    assert A.device_error() == 0


@pytest.mark.parametrize("budget", [None, 20])
def test_a_conversation_at_its_longest(dev, ex, weights, budget):  # noqa: F811
    import abra_b200 as A

    shape, rng = ex.Shape(layers=1), np.random.default_rng(2)
    d = ex.PagedDecoder(shape, weights, n_pages=16, max_len=44, budget=budget, recent=8)
    d.feed(d.add(), rng.integers(0, shape.vocab, 44))
    was = _state(d)
    with pytest.raises(ValueError, match="max_len"):
        d.forward(torch.zeros(1, 1, dtype=torch.long, device=dev), 0)
    assert _state(d) == was
    torch.cuda.synchronize()
    assert A.device_error() == 0
