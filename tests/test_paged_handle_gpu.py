"""PagedKV stays with the tensors that it was made of."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _kv(dev):
    import abra_b200 as A

    k, v = (torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=dev) for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    pos = torch.zeros(4, 2, 16, dtype=torch.int32, device=dev)
    return A.PagedKV(k, v, table, lens, next_pos=lens.clone(), pos=pos, acc=pos.float())


@pytest.mark.parametrize("name", ["k", "v", "table", "lens", "next_pos", "pos", "acc"])
def test_another_tensor_in_its_place_is_refused(dev, name):
    kv = _kv(dev)
    was = getattr(kv, name)
    with pytest.raises(AttributeError, match="in place"):
        setattr(kv, name, was + 1)
    with pytest.raises(AttributeError, match="in place"):
        setattr(kv, name, None)
    assert getattr(kv, name) is was


def test_what_is_done_in_place_reaches_the_calls(dev):
    import abra_b200 as A

    kv = _kv(dev)
    kv.lens += 1
    kv.next_pos += 7
    x = torch.ones(2, 2, 64, device=dev)
    A.paged_append(kv, x, 2 * x)
    kv.acc += 3
    torch.cuda.synchronize()
    assert A.device_error() == 0
    assert (kv.k[[0, 2], :, 0] == 1).all() and (kv.v[[0, 2], :, 0] == 2).all()
    assert (kv.pos[[0, 2], :, 0] == 6).all() and (kv.acc == 3).all()


def test_a_tensor_that_was_not_given_stays_away(dev):
    import abra_b200 as A

    kv = _kv(dev)
    bare = A.PagedKV(kv.k, kv.v, kv.table, kv.lens)
    with pytest.raises(AttributeError, match="in place"):
        bare.acc = kv.acc
