"""The paged calls with nothing to do: no sequences, no tokens."""
from __future__ import annotations

import pytest
import torch

from test_paged import _append, _attend, _desc, _evict


def test_no_sequences_need_no_memory():
    """What an empty tensor gives for its address is null."""
    from abra_b200 import _lib as L

    empty = _desc(n_seqs=0, table=0, lens=0, max_pages=0, table_stride=0)
    nothing = dict(q=None, out=None, workspace=None, workspace_bytes=0)
    assert _attend(L, empty, **nothing) == L.ABRA_OK, L.last_error()
    assert _attend(L, empty, flags=1, **nothing) == L.ABRA_OK
    assert _append(L, empty, n_tokens=0, q=None, q_out=None, k=None, v=None) == L.ABRA_OK
    assert _evict(L, empty, new_lens=None, workspace=None, workspace_bytes=0) == L.ABRA_OK


def test_other_arguments_are_checked_all_the_same():
    from abra_b200 import _lib as L

    empty = dict(n_seqs=0, table=0, lens=0)
    assert _attend(L, _desc(**empty), n_heads=3) == L.ABRA_E_INVALID
    assert _attend(L, _desc(**empty), out_type=12) == L.ABRA_E_UNSUPPORTED
    assert _attend(L, _desc(**empty, acc=0), flags=1) == L.ABRA_E_INVALID
    assert _evict(L, _desc(**empty), budget=0) == L.ABRA_E_INVALID
    assert _evict(L, _desc(**empty, pos=0)) == L.ABRA_E_INVALID
    assert _append(L, _desc(**empty), n_tokens=3) == L.ABRA_E_INVALID
    assert _attend(L, _desc(**empty, k=0)) == L.ABRA_E_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("width", [0, 4])
def test_no_sequences_from_python(dev, width):
    import abra_b200 as A

    k, v = (torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=dev) for _ in range(2))
    acc = torch.zeros(4, 2, 16, device=dev)
    table = torch.zeros(0, width, dtype=torch.int32, device=dev)
    lens = torch.zeros(0, dtype=torch.int32, device=dev)
    kv = A.PagedKV(k, v, table, lens, next_pos=lens.clone(), acc=acc, pos=acc.int())
    x = torch.zeros(0, 2 * 64, device=dev)
    q = A.paged_append(kv, x, x, q=torch.zeros(0, 8 * 64, device=dev))
    assert q.shape == (0, 8, 64)
    assert A.paged_append(kv, x, x, cu_new=torch.zeros(1, dtype=torch.int32, device=dev)) is None
    for accumulate in (False, True):
        out = A.paged_attention(kv, q, 0.1, accumulate=accumulate, lse=torch.zeros(0, 1, 8, device=dev))
        assert out.shape == (0, 8, 64) and out.dtype == torch.float16
    assert A.paged_attention(kv, torch.zeros(0, 3, 8, 64, dtype=torch.float16, device=dev), 0.1).shape == (0, 3, 8, 64)
    assert A.paged_evict(kv, 16).shape == (0,)
    torch.cuda.synchronize()
    assert A.device_error() == 0


@pytest.mark.gpu
def test_no_tokens_for_some_sequences(dev):
    import abra_b200 as A

    k, v = (torch.ones(4, 2, 16, 64, dtype=torch.float16, device=dev) for _ in range(2))
    kv = A.PagedKV(k, v, torch.zeros(2, 2, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev))
    x = torch.zeros(0, 2, 64, device=dev)
    assert A.paged_append(kv, x, x) is None
    assert A.paged_append(kv, x, x, cu_new=torch.zeros(3, dtype=torch.int32, device=dev)) is None
    assert (A.paged_attention(kv, torch.ones(2, 4, 64, dtype=torch.float16, device=dev), 0.1) == 0).all()
    torch.cuda.synchronize()
    assert A.device_error() == 0 and (k == 1).all()
