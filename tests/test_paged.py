"""The paged cache's argument checks, which run before any launch (no GPU)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch


def _desc(**kw):
    from abra_b200.paged import PagedKvDesc

    d = dict(k=4096, v=4096, acc=4096, pos=4096, table=4096, lens=4096, next_pos=0, k_page_stride=2048,
             k_head_stride=1024, k_slot_stride=64, v_page_stride=2048, v_head_stride=1024, v_slot_stride=64,
             table_stride=4, type=1, n_pages=8, n_kv_heads=2, head_dim=64, page_size=16, n_seqs=3, max_pages=4)
    d.update(kw)
    return PagedKvDesc(**d)


def _append(L, desc, **kw):
    a = dict(q=4096, k=4096, v=4096, in_type=0, ldq=256, ldk=128, ldv=128, n_heads=4, cu_new=None, n_tokens=3,
             q_norm=None, k_norm=None, eps=1e-6, rope=None, rope_len=0, q_out=4096, ldqo=256, stream=None)
    a.update(kw)
    return L.lib.abra_paged_append(None if desc is None else C.byref(desc), *a.values())


def _attend(L, desc, **kw):
    a = dict(q=4096, ldq=256, n_heads=4, n_q=1, scale=0.125, out=4096, out_type=1, ldo=256, lse=None, flags=0,
             workspace=4096, workspace_bytes=1 << 40, stream=None)
    a.update(kw)
    return L.lib.abra_paged_attention(None if desc is None else C.byref(desc), *a.values())


def _evict(L, desc, **kw):
    a = dict(budget=16, n_sink=0, n_recent=0, new_lens=8192, workspace=4096, workspace_bytes=1 << 40, stream=None)
    a.update(kw)
    return L.lib.abra_paged_evict(None if desc is None else C.byref(desc), *a.values())


BAD_CACHES = [
    (dict(k=0), "INVALID"), (dict(v=0), "INVALID"), (dict(table=0), "INVALID"), (dict(lens=0), "INVALID"),
    (dict(k=4104), "INVALID"), (dict(v=4098), "INVALID"), (dict(acc=4098), "INVALID"), (dict(lens=4097), "INVALID"),
    (dict(k_page_stride=2047), "INVALID"), (dict(v_slot_stride=-64), "INVALID"), (dict(k_head_stride=4), "INVALID"),
    (dict(table_stride=3), "INVALID"), (dict(n_pages=0), "INVALID"), (dict(n_kv_heads=0), "INVALID"),
    (dict(page_size=0), "INVALID"), (dict(n_seqs=-1), "INVALID"), (dict(max_pages=0), "INVALID"),
    (dict(head_dim=80), "UNSUPPORTED"), (dict(head_dim=0), "UNSUPPORTED"), (dict(type=0), "UNSUPPORTED"),
    (dict(type=12), "UNSUPPORTED"), (dict(max_pages=1 << 28, table_stride=1 << 28), "UNSUPPORTED"),
]


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_every_call_refuses_a_bad_cache(change, code):
    from abra_b200 import _lib as L

    want = getattr(L, "ABRA_E_" + code)
    for call in (_append, _attend, _evict):
        assert call(L, _desc(**change)) == want
        assert L.last_error()
    assert L.lib.abra_paged_attention_workspace(C.byref(_desc(**change)), 4, 1, 0) == want
    assert L.lib.abra_paged_evict_workspace(C.byref(_desc(**change)), 16) == want


def test_null_cache():
    from abra_b200 import _lib as L

    for call in (_append, _attend, _evict):
        assert call(L, None) == L.ABRA_E_INVALID


@pytest.mark.parametrize("change,code", [
    (dict(in_type=12), "UNSUPPORTED"), (dict(n_tokens=-1), "INVALID"), (dict(n_tokens=4), "INVALID"),
    (dict(k=None), "INVALID"), (dict(v=None), "INVALID"), (dict(q=None), "INVALID"), (dict(q_out=None), "INVALID"),
    (dict(n_heads=0), "INVALID"), (dict(ldk=120), "INVALID"), (dict(ldv=127), "INVALID"), (dict(ldq=248), "INVALID"),
    (dict(ldqo=248), "INVALID"), (dict(ldq=257), "INVALID"), (dict(k=4100), "INVALID"), (dict(q_out=4104), "INVALID"),
    (dict(q_norm=4100), "INVALID"), (dict(rope=4098, rope_len=8), "INVALID"), (dict(rope=4096, rope_len=0), "INVALID"),
    (dict(cu_new=4097), "INVALID"),
])
def test_append_refusals(change, code):
    from abra_b200 import _lib as L

    assert _append(L, _desc(), **change) == getattr(L, "ABRA_E_" + code), L.last_error()


@pytest.mark.parametrize("change,code", [
    (dict(n_heads=3), "INVALID"), (dict(n_heads=0), "INVALID"), (dict(n_q=0), "INVALID"), (dict(n_q=5000), "INVALID"),
    (dict(flags=2), "INVALID"), (dict(out_type=30), "UNSUPPORTED"), (dict(q=None), "INVALID"),
    (dict(out=None), "INVALID"), (dict(workspace=None), "INVALID"), (dict(workspace=4112), "INVALID"),
    (dict(workspace_bytes=8), "INVALID"), (dict(ldq=248), "INVALID"), (dict(ldo=260), "INVALID"),
    (dict(q=4104), "INVALID"), (dict(out=4100), "INVALID"), (dict(lse=4098), "INVALID"),
])
def test_attention_refusals(change, code):
    from abra_b200 import _lib as L

    assert _attend(L, _desc(), **change) == getattr(L, "ABRA_E_" + code), L.last_error()


def test_accumulation_needs_acc():
    from abra_b200 import _lib as L

    assert _attend(L, _desc(acc=0), flags=1) == L.ABRA_E_INVALID
    assert L.lib.abra_paged_attention_workspace(C.byref(_desc(acc=0)), 4, 1, 1) == L.ABRA_E_INVALID


@pytest.mark.parametrize("change,code", [
    (dict(budget=0), "INVALID"), (dict(n_sink=-1), "INVALID"), (dict(n_recent=-1), "INVALID"),
    (dict(n_sink=9, n_recent=8), "INVALID"), (dict(n_sink=2**31 - 1, n_recent=2**31 - 1), "INVALID"),
    (dict(new_lens=None), "INVALID"), (dict(new_lens=4096), "INVALID"), (dict(new_lens=4104), "INVALID"),
    (dict(workspace=None), "INVALID"), (dict(workspace=4104), "INVALID"), (dict(workspace_bytes=0), "INVALID"),
])
def test_evict_refusals(change, code):
    from abra_b200 import _lib as L

    assert _evict(L, _desc(), **change) == getattr(L, "ABRA_E_" + code), L.last_error()


def test_evict_needs_weights_and_positions():
    from abra_b200 import _lib as L

    assert _evict(L, _desc(acc=0)) == L.ABRA_E_INVALID
    assert _evict(L, _desc(pos=0)) == L.ABRA_E_INVALID


def test_nothing_to_do_is_no_error():
    """No sequences, no tokens: success without a launch (there is no GPU here)."""
    from abra_b200 import _lib as L

    empty = _desc(n_seqs=0)
    assert _append(L, empty, n_tokens=0) == L.ABRA_OK
    assert _attend(L, empty) == L.ABRA_OK
    assert _evict(L, empty) == L.ABRA_OK
    assert _append(L, empty, n_tokens=3) == L.ABRA_E_INVALID


def test_python_refuses_tensors_off_the_gpu_and_of_other_shapes():
    import abra_b200 as A

    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        A.PagedKV(k, k, table, lens)
    with pytest.raises(ValueError, match="n_pages"):
        A.PagedKV(k, k[:3], table, lens)
    with pytest.raises(ValueError, match="float16"):
        A.PagedKV(k.float(), k.float(), table, lens)


def test_row_strides_of_views():
    from abra_b200.paged import _rows

    x = torch.zeros(6, 400)
    assert _rows(x[:, 8:136], "x", 128, -1) == (6, 400)
    assert _rows(x[:, 8:136].unflatten(1, (2, 64)), "x", 128, -1) == (6, 400)
    assert _rows(x[:, :384].view(6, 3, 128), "x", 384, -1) == (6, 400)
    assert _rows(torch.zeros(2, 3, 4, 64), "x", 256, -1) == (6, 256)
    assert _rows(torch.zeros(1, 1, 4, 64), "x", 256, -1) == (1, 256)
    assert _rows(x[:0, :128], "x", 128, -1)[0] == 0
    for bad in (x[:, :256:2], torch.zeros(4, 2, 300)[:, :, :128].transpose(0, 1)[:, :, :64], x[:, :100]):
        with pytest.raises(ValueError):
            _rows(bad, "x", 128, -1)
