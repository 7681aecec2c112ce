"""Which buffers of the paged calls may share memory (checked before any launch, no GPU)."""
from __future__ import annotations

import pytest

from test_paged import _attend, _desc

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
