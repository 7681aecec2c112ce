"""The paged operators in their place: the example's decoder against the
library's own decode model on the same weights, and with a bounded cache."""
from __future__ import annotations

import ctypes as C
import importlib.util
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("paged_serving", ROOT / "examples" / "paged_serving.py")
    mod = importlib.util.module_from_spec(spec)
    sys.modules["paged_serving"] = mod  # its dataclass looks itself up
    spec.loader.exec_module(mod)
    return mod


def _model(ex, shape, weights):
    """The decode model (contiguous cache, fp32 queries) with these weights."""
    from abra_b200 import _lib
    from abra_b200.model import DecodeModel

    m = DecodeModel(n_layers=shape.layers, hidden=shape.hidden, n_heads=shape.heads, n_kv_heads=shape.kv_heads,
                    head_dim=shape.head_dim, ffn=shape.ffn, vocab=shape.vocab, max_ctx=512, rope_theta=shape.theta,
                    eps=shape.eps)
    slots = {"attn_norm": 0, "attn_q": 1, "attn_q_norm": 2, "attn_k_norm": 3, "attn_output": 4, "ffn_norm": 5,
             "ffn_gate": 6, "ffn_up": 7, "ffn_down": 8, "attn_k": 9, "attn_v": 10}
    for name, w in weights.items():
        layer, slot = (-1, 1 if name == "token_embd" else 2)
        if name.startswith("blk."):
            _, layer, what = name.split(".")
            layer, slot = int(layer), slots[what]
        rc = _lib.lib.abra_model_load_tensor(m.handle, layer, slot, 0 if w.dtype == np.float32 else 12,
                                             w.ctypes.data, C.c_uint64(w.nbytes))
        assert rc == 0, _lib.lib.abra_model_last_error()
    return m


def _exact(ex, shape, weights, tokens):
    """Logits of every position in 64 bits from the dequantized weights, no
    activation quantized, nothing rounded."""

    def mat(name, n, k):
        return torch.from_numpy(ex.dequantize(weights[name], n, k)).double()

    def norm(x, w):
        return x / ((x * x).mean(-1, keepdim=True) + shape.eps).sqrt() * torch.from_numpy(w).double()

    s, n, hd = shape, len(tokens), shape.head_dim
    embed = mat("token_embd", s.vocab, s.hidden)
    x = embed[torch.as_tensor(tokens)]
    angle = torch.arange(n).double()[:, None] * s.theta ** (-2.0 * torch.arange(hd // 2).double() / hd)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotate(y):
        z = torch.complex(y[..., : hd // 2], y[..., hd // 2 :]) * turn
        return torch.cat([z.real, z.imag], -1)

    mask = torch.full((n, n), -torch.inf, dtype=torch.float64).triu(1)
    for i in range(s.layers):
        b = f"blk.{i}."
        h = norm(x, weights[b + "attn_norm"])
        q = (h @ mat(b + "attn_q", s.heads * hd, s.hidden).T).view(n, s.heads, hd)
        k = (h @ mat(b + "attn_k", s.kv_heads * hd, s.hidden).T).view(n, s.kv_heads, hd)
        v = (h @ mat(b + "attn_v", s.kv_heads * hd, s.hidden).T).view(n, s.kv_heads, hd)
        q, k = rotate(norm(q, weights[b + "attn_q_norm"])), rotate(norm(k, weights[b + "attn_k_norm"]))
        g = s.heads // s.kv_heads
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        p = (torch.einsum("qhd,khd->hqk", q, k) * hd**-0.5 + mask).softmax(-1)
        a = torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1)
        x = x + a @ mat(b + "attn_output", s.hidden, s.heads * hd).T
        h = norm(x, weights[b + "ffn_norm"])
        h = torch.nn.functional.silu(h @ mat(b + "ffn_gate", s.ffn, s.hidden).T) * (h @ mat(b + "ffn_up", s.ffn, s.hidden).T)
        x = x + h @ mat(b + "ffn_down", s.hidden, s.ffn).T
    return norm(x, weights["output_norm"]) @ embed.T


def test_decoder_is_as_exact_as_the_decode_model(dev, ex):
    """Three conversations of different lengths over shared pages, token by
    token, against the exact model in 64 bits.  The library's decode model, run
    on each alone, has the same sources of error -- activations in 8 bits before
    every product, keys and values in fp16 -- so over all logits together the
    two are off by the same amount up to chance; the paged one's queries, fp16
    instead of fp32, add what is far below an 8-bit step.  A quarter more is
    allowed, which no error of the operators' own would stay in."""
    import abra_b200 as A

    shape = ex.Shape()
    weights = ex.random_weights(shape, 3)
    d = ex.PagedDecoder(shape, weights, n_pages=64, page=16)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, shape.vocab, n) for n in (3, 70, 37)]
    logits = [d.feed(d.add(), p).cpu() for p in prompts]
    forced = rng.integers(0, shape.vocab, (3, 6))
    for i in range(forced.shape[1]):  # the same next tokens for both
        got = d.forward(torch.as_tensor(forced[:, i : i + 1], device=dev), 0)[:, 0].cpu()
        logits = [torch.cat([a.view(-1, shape.vocab), g[None]]) for a, g in zip(logits, got)]
    torch.cuda.synchronize()
    assert A.device_error() == 0
    paged = model = size = 0.0
    with _model(ex, shape, weights) as m:
        for b, p in enumerate(prompts):
            tokens = np.concatenate([p, forced[b]])
            exact = _exact(ex, shape, weights, tokens)[len(p) - 1 :]
            m.reset(tokens)
            m.step(len(p) - 1)
            for i in range(forced.shape[1] + 1):
                m.step(1)
                m.sync()
                model += float((torch.from_numpy(m.logits()).double() - exact[i]).square().sum())
                paged += float((logits[b][i].double() - exact[i]).square().sum())
                size += float(exact[i].square().sum())
    paged, model = (paged / size) ** 0.5, (model / size) ** 0.5
    assert paged <= 1.25 * model, (paged, model)
    assert model < 0.1, model  # and the 8-bit steps leave the logits recognisable


def test_bounded_conversations(dev, ex):
    """With a budget the cache stays bounded, pages come back, and while a
    conversation is within it nothing changes."""
    import abra_b200 as A

    shape = ex.Shape()
    weights = ex.random_weights(shape, 4)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, shape.vocab, n) for n in (20, 150)]
    free = ex.PagedDecoder(shape, weights, n_pages=64)
    cut = ex.PagedDecoder(shape, weights, n_pages=64, budget=64, recent=16)
    for d in (free, cut):
        for p in prompts:
            d.first = d.feed(d.add(), p)
    t = torch.as_tensor(rng.integers(0, shape.vocab, (2, 1)), device=dev)
    a, b = free.forward(t, 0), cut.forward(t, 0)
    torch.cuda.synchronize()
    assert A.device_error() == 0
    assert torch.equal(a[0], b[0])  # 21 slots: never cut
    assert torch.isfinite(b).all() and not torch.equal(a[1], b[1])
    for _ in range(80):
        t = cut.forward(t, 0).argmax(-1)
        assert max(cut.lens) < 64 + 16
    torch.cuda.synchronize()
    assert A.device_error() == 0
    used = sum(-(-n // 16) for n in cut.lens)
    assert len(cut.free) >= 64 - used - 2 and sorted(cut.free + sum(cut.pages, [])) == list(range(64))
    # every layer and head kept the first four positions and the newest sixteen
    for pool in cut.pools:
        for s in range(2):
            slot = np.arange(cut.lens[s])
            pos = pool["pos"].cpu().numpy()[np.array(cut.pages[s])[slot // 16], :, slot % 16]
            for h in range(shape.kv_heads):
                assert len(set(pos[:, h])) == cut.lens[s]
                assert {0, 1, 2, 3} <= set(pos[:, h])
                assert set(range(cut.seen[s] - 16, cut.seen[s])) <= set(pos[:, h])
