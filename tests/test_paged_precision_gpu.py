"""What the paged attention's weights keep of their precision: weights far below
a row's largest one, and the second of the two 16-bit values that they are the
sum of, seen in fp32 results."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as R
from test_paged_gpu import EPS32, _kv, _no_error

pytestmark = pytest.mark.gpu

# A weight goes into the products as two values of the cache's type, each off by
# half a unit in its last place: the square of one value's.  fp16 values end at
# 2^-24, of which half may be lost, where the row's largest weight is 2^11 or more.
FLOOR = {"f16": 2.0**-25 / 2.0**11, "bf16": 0.0}
ROWS = [(4, 1), (2, 3), (24, 1), (4, 4), (8, 8)]  # heads of one kv head, queries: two of the narrow kernel, three of the wide


def _bounds(c, q, scale, dtype, fp32):
    """The exact result, its log-sum-exp, and bounds of both.  The queries have one
    element that is not zero, so a score is one exact product; scaling it (its
    factor rounded too) and subtracting the row's reference are three roundings of
    a magnitude of M log2 units, the exponential is good to four units of 2^-24.
    Twice that for the denominator's share, two roundings of 16 slots' sums and 64
    for the joins, half a unit of the result."""
    want, lse64, _, mag, dot = R.attention(c, q, scale)
    n = c["lens"].double().numpy()[:, None, None]
    assert (lse64 > -np.inf).all()
    worst = 1.4427 * abs(scale) * dot + 64.0
    ds = 3 * EPS32 * worst * 0.6932 + 4 * EPS32
    sums = (n / 8 + 64) * 2 * EPS32
    size = np.zeros(want.shape)  # sum |v| over the row's sum of exp(s - its largest)
    for b in range(q.shape[0]):
        for j in range(q.shape[1]):
            m = int(c["lens"][b]) - (q.shape[1] - 1 - j)
            k, v = (R.rows(c, c[x], b, m).double().numpy() for x in ("k", "v"))
            for h in range(q.shape[2]):
                g = h // (q.shape[2] // k.shape[0])
                top = (scale * (k[g] @ q[b, j, h].double().numpy())).max()
                size[b, j, h] = np.abs(v[g]).sum(0) / np.exp(lse64[b, j, h] - top)
    tol = mag * (2 * ds + R.UNIT[dtype] ** 2 + sums)[..., None] + FLOOR[dtype] * size
    tol += (EPS32 if fp32 else R.UNIT[dtype]) * np.abs(want) + (2.0**-25 if not fp32 and dtype == "f16" else 2.0**-126)
    return want, tol, lse64, ds + sums + 2 * EPS32 * np.abs(lse64)


def _check(c, q, scale, out, lse, dtype):
    want, tol, lse64, lse_tol = _bounds(c, q, scale, dtype, out.dtype == torch.float32)
    got = out.cpu().double().numpy()
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    if lse is not None:
        assert (np.abs(lse.cpu().double().numpy() - lse64) <= lse_tol).all()


def _few_bits(rng, shape, dtype):
    """Queries with one element that is not zero, another for each head."""
    q = torch.zeros(*shape)
    at = torch.arange(shape[2]) % shape[3]
    q[..., torch.arange(shape[2]), at] = torch.from_numpy(rng.choice([-3.0, -1.5, 1.0, 2.5], shape[:3])).float()
    return q.to(R.DTYPE[dtype])


def _attend(dev, c, q, scale, dtype):
    import abra_b200 as A

    kv = _kv(R.to_dev(c, dev))
    lse = torch.empty(q.shape[:3], device=dev)
    out32 = torch.empty(q.shape, device=dev)
    A.paged_attention(kv, q.to(dev), scale, out=out32, lse=lse)
    out = A.paged_attention(kv, q.to(dev), scale)
    _no_error()
    _check(c, q, scale, out32, lse, dtype)
    _check(c, q, scale, out, None, dtype)
    assert torch.equal(out32.to(q.dtype), out)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,n_q", ROWS)
@pytest.mark.parametrize("gap", [14.0, 16.0, 18.0, 20.0])
@pytest.mark.parametrize("where", ["first", "last"])
def test_a_sink_over_everything_else(dev, dtype, hq, n_q, gap, where):
    """One slot with a value of zero `gap` nats above thousands of others: the
    result is theirs alone, e^-gap of their size each."""
    rng = np.random.default_rng(int(gap) + hq)
    lens, d = [300, 2000, 8192], 64
    c = R.make_cache(rng, lens, 1, d, 16, dtype)
    for b, n in enumerate(lens):
        t = np.arange(n)
        pg, off = c["table"][b].long()[t // 16], torch.from_numpy(t % 16)
        sink = 0 if where == "first" else n - n_q
        score = -gap - rng.integers(0, 4, n) / 4.0
        score[sink] = 0.0
        v = 1.0 + rng.standard_normal((n, d))
        v[sink] = 0.0
        c["k"][pg, 0, off, 0] = torch.from_numpy(score).to(R.DTYPE[dtype])
        c["v"][pg, 0, off] = torch.from_numpy(v).to(R.DTYPE[dtype])
    q = torch.zeros(len(lens), n_q, hq, d)
    q[..., 0] = torch.tensor([1.0, 0.875, 0.5, 0.25]).repeat(16)[:hq]
    _attend(dev, c, q.to(R.DTYPE[dtype]), 1.0, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,n_q", ROWS)
def test_both_parts_of_the_weights(dev, dtype, hq, n_q):
    """Ordinary scores.  The bounds are those of weights of two 16-bit values:
    the definition with weights of one, which leave out the second, is beyond them."""
    rng = np.random.default_rng(hq * n_q)
    lens, d = [n_q + 2, 100, 700], 64
    c = R.make_cache(rng, lens, 1, d, 16, dtype)
    q = _few_bits(rng, (len(lens), n_q, hq, d), dtype)
    _attend(dev, c, q, 0.75, dtype)
    want, tol, _, _ = _bounds(c, q, 0.75, dtype, True)
    for b, n in enumerate(lens):
        k, v = (R.rows(c, c[x], b, n).double() for x in ("k", "v"))
        s = 0.75 * torch.einsum("qhd,td->qht", q[b].double(), k[0])
        s += torch.where(torch.arange(n) < n - n_q + 1 + torch.arange(n_q)[:, None], 0.0, -torch.inf)[:, None]
        w = (s - s.amax(-1, keepdim=True)).exp()
        one = (w.to(R.DTYPE[dtype]).double() @ v[0]) / w.sum(-1, keepdim=True)
        assert (np.abs(one.numpy() - want[b]) > tol[b]).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,n_q", ROWS)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_values_at_the_end_of_their_type(dev, dtype, hq, n_q, sign):
    """Thousands of values near the largest, or the lowest, of the type: their
    mean is one too, though their sum is far beyond fp32 in bf16."""
    rng = np.random.default_rng(hq + n_q)
    lens, d = [50, 6000], 64
    c = R.make_cache(rng, lens, 1, d, 16, dtype)
    most = float(torch.finfo(R.DTYPE[dtype]).max)
    c["v"] = torch.from_numpy(sign * most * rng.uniform(0.5, 0.9, c["v"].shape)).to(R.DTYPE[dtype])
    q = _few_bits(rng, (len(lens), n_q, hq, d), dtype)
    _attend(dev, c, q, 1.0, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,n_q", ROWS)
def test_scores_beyond_single_units(dev, dtype, hq, n_q):
    """Scores around 2^27, 2^28 log2 units, which fp32 holds in steps of 16 or
    32: which slot is the largest is lost, but the result stays among the values
    (up to the roundings) and no weight leaves the type's range."""
    import abra_b200 as A

    rng = np.random.default_rng(hq)
    n, d = 1000, 64
    c = R.make_cache(rng, [n], 1, d, 16, dtype)
    t = np.arange(n)
    pg, off = c["table"][0].long()[t // 16], torch.from_numpy(t % 16)
    c["k"][pg, 0, off] = 0.0
    c["k"][pg, 0, off, 0] = 4096.0
    c["k"][pg, 0, off, 1] = torch.from_numpy(np.sort(rng.integers(0, 128, n)).astype(np.float64)).to(R.DTYPE[dtype])
    q = torch.zeros(1, n_q, hq, d)
    q[..., 0] = 32768.0
    q[..., 1] = torch.tensor([1.0, 2.0, 0.5, -1.0]).repeat(16)[:hq]
    out = torch.empty(q.shape, device=dev)
    for scale in (1.0, 2.0):
        A.paged_attention(_kv(R.to_dev(c, dev)), q.to(R.DTYPE[dtype]).to(dev), scale, out=out)
        _no_error()
        v = c["v"][pg, 0, off].double()
        slack = 2.0**-15 * v.abs().amax(0)  # a row's weights and its sum of them, 1,000 slots
        got = out.cpu().double()
        assert torch.isfinite(got).all()
        assert (got <= v.amax(0) + slack).all() and (got >= v.amin(0) - slack).all()
