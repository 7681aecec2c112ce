"""Which buffers of the paged calls may share memory (checked before any launch, no GPU)."""
from __future__ import annotations

import pytest

from test_paged import _append, _attend, _desc

# The cache of _desc has three sequences; four heads of 64 make rows of 256 elements.
Q = 1 << 20


@pytest.mark.parametrize("what", [
    dict(out=Q),  # the same rows
    dict(out=Q + 16),  # eight elements on
    dict(out=Q - 16),
    dict(out=Q + 2 * 2 * 256 + 496),  # the last sequence's last eight elements
    dict(out=Q - 2 * 2 * 256 - 496),
    dict(out=Q, out_type=0),  # fp32 over it
    dict(out=Q - 2048, out_type=0),  # its third row there
    dict(out=Q + 3 * 512 - 16, out_type=0),
    dict(out=Q + 512, ldq=512, ldo=256),  # between the rows at first, over the second one then
    dict(out=Q + 496, ldq=512, ldo=512),  # a column too far to the left
    dict(out=Q + 528, ldq=512, ldo=512),  # and to the right, into the next row
    dict(out=Q - 528, ldq=512, ldo=512),
    dict(out=Q + 512, ldq=512, ldo=256, out_type=0),  # columns too wide for what is left of the rows
])
def test_results_over_queries_are_refused(what):
    from abra_b200 import _lib as L

    assert _attend(L, _desc(), q=Q, workspace_bytes=256, **what) == L.ABRA_E_INVALID
    assert "share" in L.last_error()


@pytest.mark.parametrize("what", [
    dict(out=Q + 3 * 512), dict(out=Q - 3 * 512), dict(out=Q + 3 * 512, out_type=0), dict(out=Q - 3 * 1024, out_type=0),
    dict(out=Q + 512, ldq=512, ldo=512),  # columns of the same rows, behind the queries
    dict(out=Q - 512, ldq=512, ldo=512),  # in front of them
    dict(out=Q + 512, ldq=1024, ldo=512, out_type=0),
    dict(out=Q - 4096 + 1024, ldq=1024, ldo=512, out_type=0),  # one row earlier
])
def test_other_memory_is_not(what):
    """The call ends at the next check, of a workspace that is too small."""
    from abra_b200 import _lib as L

    assert _attend(L, _desc(), q=Q, workspace_bytes=256, **what) == L.ABRA_E_INVALID
    assert "workspace" in L.last_error()


@pytest.mark.parametrize("what", [
    dict(q=Q, q_out=Q),  # fp32 queries under 16-bit ones
    dict(q=Q, q_out=Q + 1024),
    dict(q=Q, q_out=Q + 16, in_type=1),
    dict(q=Q, q_out=Q, in_type=1, ldq=512),  # other rows from the second one on
    dict(k=Q, q_out=Q), dict(v=Q, q_out=Q + 1024), dict(k=Q, q_out=Q - 1024 + 16, in_type=30),
    # a fused row of 4 + 2 + 2 heads in fp32, its queries' place half taken by theirs in 16 bits
    dict(q=Q, k=Q + 1024, v=Q + 1536, ldq=512, ldk=512, ldv=512, q_out=Q + 512, ldqo=1024),
    dict(q=Q, k=Q + 1024, v=Q + 1536, ldq=512, ldk=512, ldv=512, q_out=Q + 1024, ldqo=1024),
])
def test_append_over_its_tokens_is_refused(what):
    from abra_b200 import _lib as L

    a = {"q": 1 << 24, "k": 1 << 25, "v": 1 << 26, "rope": 4096, "rope_len": 0, **what}
    assert _append(L, _desc(), n_heads=4, **a) == L.ABRA_E_INVALID
    assert "share" in L.last_error()


@pytest.mark.parametrize("what", [
    dict(q=Q, q_out=Q + 3 * 1024), dict(q=Q, q_out=Q, in_type=1), dict(q=Q, q_out=Q, in_type=30, ldq=512, ldqo=512),
    # behind the fused row's heads, and in its queries' place
    dict(q=Q, k=Q + 1024, v=Q + 1536, ldq=640, ldk=640, ldv=640, q_out=Q + 2048, ldqo=1280),
    dict(q=Q, k=Q + 512, v=Q + 768, ldq=512, ldk=512, ldv=512, q_out=Q, ldqo=512, in_type=1),
])
def test_append_beside_its_tokens_is_not(what):
    """The call ends at the next check, of a rotation table without rows."""
    from abra_b200 import _lib as L

    a = {"q": 1 << 24, "k": 1 << 25, "v": 1 << 26, "rope": 4096, "rope_len": 0, **what}
    assert _append(L, _desc(), n_heads=4, **a) == L.ABRA_E_INVALID
    assert "rope" in L.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_append_in_the_queries_place(dev, dtype):
    """16-bit queries turned where they lie in the fused rows, as beside them."""
    import numpy as np
    import torch

    import abra_b200 as A
    import paged_reference as R
    from test_paged_gpu import _kv, _no_error

    rng = np.random.default_rng(3)
    hq, hkv, d, n = 12, 2, 96, 150
    c = R.make_cache(rng, [n + 7], hkv, d, 16, dtype)
    rows = torch.from_numpy(rng.standard_normal((n, (hq + 2 * hkv) * d))).to(R.DTYPE[dtype]).to(dev)
    norm = torch.rand(d, device=dev) + 0.5
    angle = torch.rand(n + 7, d // 2, device=dev)
    rope = torch.stack([angle.cos(), angle.sin()], -1)
    got = {}
    for place in ("beside", "own"):
        cd = R.to_dev(c, dev)
        mine = rows.clone()
        q, k, v = mine.split((hq * d, hkv * d, hkv * d), 1)
        out = A.paged_append(_kv(cd), k, v, q=q, q_out=q if place == "own" else None, q_norm=norm, k_norm=norm, rope=rope)
        _no_error()
        got[place] = (out.reshape(n, hq * d).clone(), cd["k"].nan_to_num(), cd["v"].nan_to_num(), mine[:, hq * d :])
    for a, b in zip(got["beside"], got["own"]):
        assert torch.equal(a, b)
