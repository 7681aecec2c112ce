"""Paged append with offsets of new tokens that do not fit the call, and with
positions beyond the rotation's table."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as R
from test_paged_gpu import _kv, _no_error

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 4, 2, 64, 16


def _append(dev, lens, cu, n, rope=None, next_pos=None, error=16):
    """(cache, its tensors after the call, tokens, queries) of n tokens with these offsets."""
    import abra_b200 as A

    rng = np.random.default_rng(n)
    c = R.make_cache(rng, lens, HKV, D, PAGE, "f16")
    cd = R.to_dev(c, dev)
    x = torch.from_numpy(rng.standard_normal((n, (HQ + 2 * HKV) * D))).half().to(dev)
    q, k, v = x.split((HQ * D, HKV * D, HKV * D), 1)
    kv = _kv(cd, acc=cd["acc"], pos=cd["pos"], next_pos=None if next_pos is None else torch.tensor(next_pos, dtype=torch.int32, device=dev))
    out = A.paged_append(kv, k, v, q=q, cu_new=torch.tensor(cu, dtype=torch.int32, device=dev), rope=rope)
    torch.cuda.synchronize()
    assert A.device_error() == error
    return c, {a: t.cpu() if isinstance(t, torch.Tensor) else t for a, t in cd.items()}, x.cpu().view(n, -1, D), out.cpu()


def _check(c, after, x, stored):
    """The tokens of `stored`, {(sequence, slot): token}, are in the cache and nothing else is."""
    want = {a: c[a].clone() for a in ("k", "v", "acc", "pos")}
    for (b, t), i in stored.items():
        pg, off = int(c["table"][b, t // PAGE]), t % PAGE
        want["k"][pg, :, off], want["v"][pg, :, off] = x[i, HQ : HQ + HKV], x[i, HQ + HKV :]
        want["acc"][pg, :, off], want["pos"][pg, :, off] = 0.0, t
    for a, w in want.items():
        bits = torch.int16 if w.element_size() == 2 else torch.int32
        assert torch.equal(after[a].contiguous().view(bits), w.contiguous().view(bits)), a


@pytest.mark.parametrize("cu,n,stored", [
    ([0, 3, 3, 5], 5, {(0, 37): 0, (0, 38): 1, (0, 39): 2, (2, 18): 3, (2, 19): 4}),  # as it should be
    ([5, 8, 8, 10], 5, {}),  # a piece of a longer list, its tokens counted from there
    ([2, 3, 3, 5], 5, {(0, 39): 2, (2, 18): 3, (2, 19): 4}),  # two tokens of nobody's in front
    ([0, 3, 3, 4], 5, {(0, 37): 0, (0, 38): 1, (0, 39): 2, (2, 19): 3}),  # and one behind
    ([0, 3, 3, 9], 5, {(0, 37): 0, (0, 38): 1, (0, 39): 2}),  # more tokens than there are
    ([0, 5, 5, 8], 5, {(0, 35 + i): i for i in range(5)}),  # a sequence beyond them
    ([-2, 3, 3, 5], 5, {(0, 37): 0, (0, 38): 1, (0, 39): 2, (2, 18): 3, (2, 19): 4}),
    ([0, 3, 2, 5], 5, None),  # falling: only that it is reported
])
def test_offsets_that_do_not_fit_the_tokens(dev, cu, n, stored):
    good = cu == [0, 3, 3, 5]
    c, after, x, out = _append(dev, [40, 1, 20], cu, n, error=0 if good else 16)
    assert torch.equal(out, x[:, :HQ])
    if stored is not None:
        _check(c, after, x, stored)


def test_offsets_of_hundreds_of_sequences(dev):
    """One falling offset among hundreds, in front of tokens that are not its
    own, and thousands of tokens, several a CTA."""
    rng = np.random.default_rng(1)
    new = rng.integers(1, 9, 600)
    cu = np.concatenate([[0], np.cumsum(new)])
    lens = [int(m) + 5 for m in new]
    n = int(cu[-1])
    stored = {(b, 5 + i): int(cu[b]) + i for b in range(600) for i in range(new[b])}
    c, after, x, _ = _append(dev, lens, cu.tolist(), n, error=0)
    _check(c, after, x, stored)
    bad = cu.copy()
    bad[400] = bad[399] - 1
    _append(dev, lens, bad.tolist(), n)
    _append(dev, lens, (cu + 1).tolist(), n)


def test_positions_beyond_the_rotation(dev):
    """Reported; the token is stored, its query and key as they are without a
    rotation."""
    angle = torch.rand(30, D // 2, device=dev)
    rope = torch.stack([angle.cos(), angle.sin()], -1)
    c, after, x, out = _append(dev, [40, 12, 20], [0, 2, 3, 5], 5, rope=rope, next_pos=[31, 12, 0])
    turned = [True, False, True, False, False]  # positions 29, 30, 11, -2, -1
    for i, (b, t, at) in enumerate([(0, 38, 29), (0, 39, 30), (1, 11, 11), (2, 18, -2), (2, 19, -1)]):
        pg, off = int(c["table"][b, t // PAGE]), t % PAGE
        assert torch.equal(after["v"][pg, :, off], x[i, HQ + HKV :]) and (after["pos"][pg, :, off] == at).all()
        assert torch.equal(out[i], x[i, :HQ]) != turned[i]
        assert torch.equal(after["k"][pg, :, off], x[i, HQ : HQ + HKV]) != turned[i]
