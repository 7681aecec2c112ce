"""Serving several conversations of different lengths from one paged cache.

A small Qwen3-shaped decoder with Q4_K weights, put together from the
library's operators: the Q4_K x Q8_1 products, RMSNorm and quantization of the
decode path, and the paged cache's append, attention and eviction.  Prompts are
fed eight tokens at a time, then all conversations decode together, one token
each a step; a conversation that outgrows its budget keeps its first tokens,
its newest ones and those that attention has looked at most, and hands back the
pages it no longer needs.

    python examples/paged_serving.py        # needs a GPU and the built library
"""
from __future__ import annotations

import sys
from dataclasses import dataclass
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import abra_b200 as A  # noqa: E402
from abra_b200._lib import lib  # noqa: E402

COLUMNS = 8  # activation columns of one Q4_K product


@dataclass
class Shape:
    layers: int = 2
    hidden: int = 512
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 128
    ffn: int = 1024
    vocab: int = 2048
    theta: float = 1.0e6
    eps: float = 1.0e-6


def quantize(w: np.ndarray) -> np.ndarray:
    """Rows of a matrix as Q4_K blocks (bytes)."""
    w = np.ascontiguousarray(w, dtype=np.float32)
    out = np.empty(A.q4k_nbytes(*w.shape), dtype=np.uint8)
    lib.quantize_row_q4_K_upstream_cpu(w.ctypes.data, out.ctypes.data, w.size)
    return out


def dequantize(blocks: np.ndarray, n: int, k: int) -> np.ndarray:
    out = np.empty((n, k), dtype=np.float32)
    lib.dequantize_row_q4_K_upstream_cpu(blocks.ctypes.data, out.ctypes.data, out.size)
    return out


def random_weights(s: Shape, seed: int = 0) -> dict[str, np.ndarray]:
    """Seeded weights under their GGUF names: Q4_K matrices, fp32 norms."""
    r = np.random.default_rng(seed)

    def matrix(n, k):
        return quantize(r.standard_normal((n, k)) / np.sqrt(k))

    def norm(n):
        return r.uniform(0.8, 1.2, n).astype(np.float32)

    w = {"token_embd": matrix(s.vocab, s.hidden), "output_norm": norm(s.hidden)}
    for i in range(s.layers):
        w |= {f"blk.{i}.attn_norm": norm(s.hidden), f"blk.{i}.ffn_norm": norm(s.hidden),
              f"blk.{i}.attn_q": matrix(s.heads * s.head_dim, s.hidden),
              f"blk.{i}.attn_k": matrix(s.kv_heads * s.head_dim, s.hidden),
              f"blk.{i}.attn_v": matrix(s.kv_heads * s.head_dim, s.hidden),
              f"blk.{i}.attn_q_norm": norm(s.head_dim), f"blk.{i}.attn_k_norm": norm(s.head_dim),
              f"blk.{i}.attn_output": matrix(s.hidden, s.heads * s.head_dim),
              f"blk.{i}.ffn_gate": matrix(s.ffn, s.hidden), f"blk.{i}.ffn_up": matrix(s.ffn, s.hidden),
              f"blk.{i}.ffn_down": matrix(s.hidden, s.ffn)}
    return w


class PagedDecoder:
    """Up to eight conversations over a pool of pages shared by all of them;
    every layer has pools of its own and all layers share the page tables.

    budget: slots a conversation keeps (None: all); a conversation is cut when
    it is a page over it."""

    def __init__(self, shape: Shape, weights: dict[str, np.ndarray], n_pages: int, page: int = 16,
                 max_len: int = 4096, budget: int | None = None, sink: int = 4, recent: int = 64,
                 dtype=torch.float16, device="cuda"):
        s = self.shape = shape
        dev = self.device = torch.device(device)

        def up(name):
            return torch.from_numpy(weights[name]).to(dev)

        self.embed = torch.from_numpy(dequantize(weights["token_embd"], s.vocab, s.hidden)).to(dev)
        self.output, self.output_norm = up("token_embd"), up("output_norm")
        self.layers = []
        for i in range(s.layers):
            b = f"blk.{i}."
            qkv = torch.cat([up(b + "attn_q"), up(b + "attn_k"), up(b + "attn_v")])  # rows one after another
            self.layers.append({"qkv": qkv} | {
                n: up(b + n) for n in ("attn_norm", "ffn_norm", "attn_q_norm", "attn_k_norm", "attn_output", "ffn_gate",
                                       "ffn_up", "ffn_down")})
        angle = torch.arange(max_len).double()[:, None] * s.theta ** (
            -2.0 * torch.arange(s.head_dim // 2).double() / s.head_dim)
        self.rope = torch.stack([angle.cos(), angle.sin()], -1).float().to(dev)
        self.page, self.budget, self.sink, self.recent = page, budget, sink, recent
        pool = (n_pages, s.kv_heads, page, s.head_dim)
        self.pools = [{"k": torch.zeros(pool, dtype=dtype, device=dev), "v": torch.zeros(pool, dtype=dtype, device=dev),
                       "acc": torch.zeros(pool[:3], device=dev), "pos": torch.zeros(pool[:3], dtype=torch.int32, device=dev)}
                      for _ in range(s.layers)]
        self.free = list(range(n_pages))
        width = -(-(max_len if budget is None else budget + page + COLUMNS) // page) + 1
        self.table = torch.zeros(COLUMNS, width, dtype=torch.int32, device=dev)
        # cached slots and next positions of each conversation, here and on the device
        self.pages: list[list[int]] = []
        self.lens, self.seen = [], []
        self.state = torch.zeros(2, COLUMNS, dtype=torch.int32, device=dev)
        self.workspace: dict = {}

    def add(self) -> int:
        """A new, empty conversation."""
        if len(self.pages) == COLUMNS:
            raise ValueError(f"at most {COLUMNS} conversations")
        self.pages.append([])
        self.lens.append(0)
        self.seen.append(0)
        return len(self.pages) - 1

    def _grow(self, lo: int, hi: int, n: int) -> None:
        """Pages for n more slots of each of the conversations; the lengths count
        them.  All or, with an error, none."""
        if max(self.seen[lo:hi]) + n > len(self.rope):
            raise ValueError(f"a conversation would be longer than max_len ({len(self.rope)})")
        need = [-(-(self.lens[b] + n) // self.page) - len(self.pages[b]) for b in range(lo, hi)]
        if sum(max(0, x) for x in need) > len(self.free):
            raise RuntimeError("the pool of pages is used up")
        for b, more in zip(range(lo, hi), need):
            self.lens[b] += n
            self.seen[b] += n
            for _ in range(more):
                self.pages[b].append(self.free.pop())
                self.table[b, len(self.pages[b]) - 1] = self.pages[b][-1]

    def _handles(self, lo: int, hi: int) -> list[A.PagedKV]:
        """The layers' caches of conversations lo .. hi - 1."""
        return [A.PagedKV(p["k"], p["v"], self.table[lo:hi], self.state[0, lo:hi], next_pos=self.state[1, lo:hi],
                          pos=p["pos"], acc=p["acc"]) for p in self.pools]

    def _publish(self) -> None:
        n = len(self.lens)
        self.state[:, :n] = torch.tensor([self.lens, self.seen], dtype=torch.int32)

    def forward(self, tokens: torch.Tensor, lo: int) -> torch.Tensor:
        """The next tokens [n, m] of conversations lo .. lo + n - 1 (n * m <= 8),
        appended to their caches; logits [n, m, vocab]."""
        s, (n, m) = self.shape, tokens.shape
        cols = n * m
        self._grow(lo, lo + n, m)
        self._publish()
        caches = self._handles(lo, lo + n)
        dev, hd = self.device, s.heads * s.head_dim
        wide = max(hd, s.ffn, s.hidden)
        xq = torch.empty(A.q8_1_nbytes(wide, cols), dtype=torch.uint8, device=dev)
        x = self.embed[tokens.reshape(-1)]
        q16 = torch.empty(n, m, s.heads, s.head_dim, dtype=caches[0].dtype, device=dev)
        att = torch.empty(n, m, s.heads, s.head_dim, device=dev)  # fp32, as the next product's quantizer wants it
        key = (n, m)
        if key not in self.workspace:
            self.workspace[key] = A.paged_attention_workspace(caches[0], s.heads, m, accumulate=True)
        qkv = torch.empty(cols, hd + 2 * s.kv_heads * s.head_dim, device=dev)
        y, h = torch.empty(cols, s.hidden, device=dev), torch.empty(cols, s.ffn, device=dev)
        for w, kv in zip(self.layers, caches):
            A.rmsnorm_quantize_q8_1(x, w["attn_norm"], s.eps, xq, s.hidden, ncols=cols)
            A.mmvq(w["qkv"], xq, qkv, qkv.shape[1], s.hidden, ncols=cols)
            q, k, v = qkv.split((hd, s.kv_heads * s.head_dim, s.kv_heads * s.head_dim), 1)
            A.paged_append(kv, k, v, q=q, q_out=q16, q_norm=w["attn_q_norm"], k_norm=w["attn_k_norm"], eps=s.eps,
                           rope=self.rope)
            A.paged_attention(kv, q16, s.head_dim**-0.5, out=att, accumulate=True, workspace=self.workspace[key])
            A.launch_quantize_f32_to_q8_1(att, xq, hd, ncols=cols)
            A.mmvq(w["attn_output"], xq, y, s.hidden, hd, ncols=cols)
            x += y
            A.rmsnorm_quantize_q8_1(x, w["ffn_norm"], s.eps, xq, s.hidden, ncols=cols)
            A.mmvq_swiglu(w["ffn_gate"], w["ffn_up"], xq, h, s.ffn, s.hidden, ncols=cols)
            A.launch_quantize_f32_to_q8_1(h, xq, s.ffn, ncols=cols)
            A.mmvq(w["ffn_down"], xq, y, s.hidden, s.ffn, ncols=cols)
            x += y
        A.rmsnorm_quantize_q8_1(x, self.output_norm, s.eps, xq, s.hidden, ncols=cols)
        logits = torch.empty(n, m, s.vocab, device=dev)
        A.mmvq(self.output, xq, logits, s.vocab, s.hidden, ncols=cols)
        self._trim(caches, lo, lo + n)
        return logits

    def _trim(self, caches, lo: int, hi: int) -> None:
        """Cuts the conversations that are a page over the budget to it."""
        if self.budget is None or max(self.lens[lo:hi]) < self.budget + self.page:
            return
        for kv in caches:  # all layers by the same lengths, each by its own weights
            A.paged_evict(kv, self.budget, self.sink, self.recent)
        for b in range(lo, hi):
            self.lens[b] = min(self.lens[b], self.budget)
            while len(self.pages[b]) * self.page >= self.lens[b] + self.page:
                self.free.append(self.pages[b].pop())
        self._publish()

    def feed(self, b: int, prompt) -> torch.Tensor:
        """A prompt into conversation b, eight tokens at a time; the logits
        after its last token."""
        t = torch.as_tensor(np.asarray(prompt), dtype=torch.long, device=self.device)
        for at in range(0, len(t), COLUMNS):
            logits = self.forward(t[None, at : at + COLUMNS], b)
        return logits[0, -1]


def main() -> None:
    shape = Shape()
    d = PagedDecoder(shape, random_weights(shape), n_pages=128, budget=128, recent=32)
    r = np.random.default_rng(1)
    picks = []
    for n in (5, 60, 203, 17):  # conversations of different lengths
        b = d.add()
        picks.append(d.feed(b, r.integers(0, shape.vocab, n)).argmax())
        print(f"conversation {b}: prompt of {n} tokens, {d.lens[b]} slots kept, {len(d.pages[b])} pages")
    tokens = torch.stack(picks)[:, None]
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    steps = 100
    start.record()
    out = [tokens]
    for _ in range(steps):
        tokens = d.forward(tokens, 0).argmax(-1)
        out.append(tokens)
    end.record()
    torch.cuda.synchronize()
    print(f"{steps} steps of {len(picks)} conversations: {start.elapsed_time(end) / steps:.3f} ms a step, "
          f"slots {d.lens}, {len(d.free)} pages free")
    for b, row in enumerate(torch.cat(out, 1).tolist()):
        print(f"conversation {b}: {row[:12]} ...")
    assert A.device_error() == 0


if __name__ == "__main__":
    main()
