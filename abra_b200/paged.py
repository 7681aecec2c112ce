"""Paged key-value cache for many sequences: append, attention, eviction.

The decode model (abra_b200.model) keeps one contiguous cache per layer, as
the reference's runtime does.  A serving program with many sequences of
different lengths keeps its cache in pages instead and calls, per layer and
step,

    paged_append     norm and rotate the new tokens' heads, store keys and values
    paged_attention  the newest token(s) of every sequence over its pages
    paged_evict      cut long sequences to a budget of slots by accumulated weight

Buffers are torch CUDA tensors; every call is asynchronous on ``stream``
(default: torch's current stream) and allocates nothing when its outputs and
workspace are given.  Bad arguments raise ValueError before any launch.
Lengths, page numbers and offsets of new tokens live on the device: one outside
its range sets bit 4 of :func:`abra_b200.device_error`.  Results share no memory
with what a call reads, except where it says so.

    kv = PagedKV(k, v, table, lens, pos=pos, acc=acc)
    lens += 1                                   # the step's token
    paged_append(kv, k_new, v_new, q=q, q_out=q16, rope=rope)
    paged_attention(kv, q16, scale, out=o, accumulate=True, workspace=ws)
    paged_evict(kv, budget, n_sink=4, n_recent=256, new_lens=cut)
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import lib
from .q4k import stream_handle

ABRA_GGML_F32, ABRA_GGML_F16, ABRA_GGML_BF16 = 0, 1, 30
ABRA_PAGED_ACCUMULATE = 1


class PagedKvDesc(C.Structure):
    """abra_paged_kv of include/abra_b200.h."""

    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("acc", C.c_void_p), ("pos", C.c_void_p),
                ("table", C.c_void_p), ("lens", C.c_void_p), ("next_pos", C.c_void_p),
                ("k_page_stride", C.c_int64), ("k_head_stride", C.c_int64), ("k_slot_stride", C.c_int64),
                ("v_page_stride", C.c_int64), ("v_head_stride", C.c_int64), ("v_slot_stride", C.c_int64),
                ("table_stride", C.c_int64), ("type", C.c_int32), ("n_pages", C.c_int32),
                ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32), ("page_size", C.c_int32),
                ("n_seqs", C.c_int32), ("max_pages", C.c_int32)]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _rows(t, name: str, width: int, index: int) -> tuple[int, int]:
    """(rows, row stride) of a tensor [..., heads, head_dim] or [..., width]
    whose rows of ``width`` elements are contiguous and evenly spaced, on
    device ``index`` (-1: the CPU)."""
    if t.get_device() != index:
        raise ValueError(f"{name} must be on the cache's device")
    shape = t.shape
    if len(shape) == 2 and shape[1] == width and t.stride(1) == 1:
        return shape[0], t.stride(0) if shape[0] > 1 else width
    n = t.numel() // width if width else 0
    if t.is_contiguous() and n * width == t.numel() and shape[-1] <= width:
        inner, i = 1, len(shape)
        while i > 0 and inner < width:
            i -= 1
            inner *= shape[i]
        if inner == width:
            return n, width
    stride = t.stride()
    n, inner, i = 1, 1, len(shape)
    while i > 0 and inner < width:  # the trailing dimensions that make one row
        i -= 1
        _need(shape[i] == 1 or stride[i] == inner, f"the rows of {name} must be contiguous")
        inner *= shape[i]
    _need(inner == width, f"{name} must have rows of {width} elements (got shape {tuple(shape)})")
    ld = None
    while i > 0:  # the leading ones must step evenly from row to row
        i -= 1
        if shape[i] != 1:
            if ld is None:
                ld = stride[i]
            else:
                _need(stride[i] == ld * n, f"the rows of {name} must be evenly spaced")
        n *= shape[i]
    return n, width if ld is None else ld


class PagedKV:
    """One layer's paged cache over the caller's tensors.

    k, v: float16 or bfloat16 [n_pages, kv heads, page size, head_dim], any
    strides with contiguous rows (a [n_pages, page size, kv heads, head_dim]
    pool is passed permuted); table: int32 [n_seqs, max_pages], the pages of
    each sequence in order; lens: int32 [n_seqs], its slots, a step's new
    tokens counted already; next_pos: int32 [n_seqs], the position after its
    newest token (None: lens, while nothing has been evicted); pos (int32) and
    acc (float32): [n_pages, kv heads, page size], each slot's position and
    accumulated attention weight (eviction needs both).

    The calls go to the memory of these tensors, so they are filled in place
    (``kv.lens += 1``); another tensor needs another PagedKV.
    """

    _TENSORS = frozenset(("k", "v", "table", "lens", "next_pos", "pos", "acc"))

    def __setattr__(self, name, value):
        # an attribute put in a tensor's place would leave the calls with the old one's memory
        if name in self._TENSORS and getattr(self, name, value) is not value:
            raise AttributeError(f"PagedKV.{name} is filled in place; another tensor needs another PagedKV")
        super().__setattr__(name, value)

    def __init__(self, k, v, table, lens, next_pos=None, pos=None, acc=None):
        import torch

        _need(k.dim() == 4 and k.shape == v.shape, "k and v must be [n_pages, kv heads, page size, head_dim]")
        _need(k.dtype == v.dtype and k.dtype in (torch.float16, torch.bfloat16),
              "k and v must both be float16 or both bfloat16")
        dev = k.device
        _need(dev.type == "cuda", "the cache must be on a CUDA device")
        _need(table.dim() == 2 and lens.dim() == 1 and table.shape[0] == lens.shape[0],
              "table must be [n_seqs, max_pages] and lens [n_seqs]")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "rows of head_dim must be contiguous")
        _need(table.shape[1] == 1 or table.stride(1) == 1, "the table's rows must be contiguous")
        for name, t in (("v", v), ("table", table), ("lens", lens), ("next_pos", next_pos), ("pos", pos),
                        ("acc", acc)):
            _need(t is None or t.device == dev, f"{name} must be on the cache's device")
        for name, t in (("table", table), ("lens", lens), ("next_pos", next_pos), ("pos", pos)):
            _need(t is None or t.dtype == torch.int32, f"{name} must be int32")
        _need(acc is None or acc.dtype == torch.float32, "acc must be float32")
        _need(lens.is_contiguous(), "lens must be contiguous")
        _need(next_pos is None or (next_pos.shape == lens.shape and next_pos.is_contiguous()),
              "next_pos must be like lens")
        for name, t in (("pos", pos), ("acc", acc)):
            _need(t is None or (t.shape == k.shape[:3] and t.is_contiguous()),
                  f"{name} must be contiguous [n_pages, kv heads, page size]")
        self.k, self.v, self.table, self.lens = k, v, table, lens
        self.next_pos, self.pos, self.acc = next_pos, pos, acc
        self.device, self.dtype = dev, k.dtype
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.n_seqs, self.max_pages = table.shape

        def at(t):
            return 0 if t is None else t.data_ptr()

        self._types = {torch.float32: ABRA_GGML_F32, torch.float16: ABRA_GGML_F16,
                       torch.bfloat16: ABRA_GGML_BF16}
        self.desc = PagedKvDesc(
            at(k), at(v), at(acc), at(pos), at(table), at(lens), at(next_pos), *k.stride()[:3],
            *v.stride()[:3], max(table.stride(0), self.max_pages) if self.n_seqs < 2 else table.stride(0),
            self._types[k.dtype], self.n_pages, self.n_kv_heads, self.head_dim, self.page_size, self.n_seqs,
            self.max_pages)
        self._ref = C.byref(self.desc)
        self._index = k.get_device()
        # the current stream's handle without building a Stream object, where torch has it
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self._current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)

    def _stream(self, stream) -> int:
        """The stream of a call on this cache, whose device must be the current one."""
        if self._current_device() != self._index:
            raise ValueError(f"the cache is on device {self._index}, which is not the current one")
        if stream is None and self._raw_stream is not None:
            return self._raw_stream(self._index)
        return stream_handle(stream)


def _empty(kv: PagedKV, shape, dtype, stream):
    """Uninitialised memory for a call on ``stream``: of that stream's pool, so
    that neither what else ran on it before nor what takes it afterwards meets
    the call."""
    import torch

    if stream is None or stream_handle(stream) == stream_handle():
        return torch.empty(shape, dtype=dtype, device=kv.device)
    if isinstance(stream, int):  # 0, the default stream, is none that could be wrapped
        stream = torch.cuda.ExternalStream(stream, kv.device) if stream else torch.cuda.default_stream(kv.device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=kv.device)


def _vector(t, name: str, n: int, kv: PagedKV):
    if t is None:
        return 0
    if not (t.get_device() == kv._index and kv._types.get(t.dtype) == ABRA_GGML_F32 and t.numel() == n
            and t.is_contiguous()):
        raise ValueError(f"{name} must be {n} contiguous float32 values on the cache's device")
    return t.data_ptr()


def paged_append(kv: PagedKV, k, v, q=None, q_out=None, cu_new=None, q_norm=None, k_norm=None,
                 eps: float = 1e-6, rope=None, stream=None):
    """Store the new tokens' keys and values in the last slots of their
    sequences and return the queries in the cache's type (abra_paged_append).

    k, v: [n_tokens, kv heads * head_dim] (or split by heads), q: [n_tokens,
    heads * head_dim], all float32, float16 or bfloat16, rows at any stride (so
    slices of one fused projection will do), sequence after sequence.  cu_new:
    int32 [n_seqs + 1], the sequences' first tokens, from 0 to n_tokens (None:
    equally many each).  q_norm, k_norm: float32 [head_dim] RMSNorm weights; rope:
    float32 [length, head_dim / 2, 2], cos and sin of each position (a position
    beyond it is reported, its token not rotated).  q_out may be other columns of
    the tokens' rows, or q itself where that has 16 bits.
    """
    dev, hd, types = kv._index, kv.head_dim, kv._types
    kvw = kv.n_kv_heads * hd
    dtype = k.dtype
    n, ldk = _rows(k, "k", kvw, dev)
    nv, ldv = _rows(v, "v", kvw, dev)
    if nv != n or v.dtype != dtype or dtype not in types:
        raise ValueError("k and v must have the same rows and type, float32, float16 or bfloat16")
    heads = ldq = ldqo = qp = qop = 0
    if q is not None:
        width = q.shape[-1] if q.dim() == 2 else q.shape[-2] * q.shape[-1]
        heads = width // hd
        nq, ldq = _rows(q, "q", width, dev)
        if heads * hd != width or nq != n or q.dtype != dtype:
            raise ValueError("q must be whole heads with the rows and the type of k and v")
        if q_out is None:
            q_out = _empty(kv, (n, heads, hd), kv.dtype, stream)
        no, ldqo = _rows(q_out, "q_out", width, dev)
        if no != n or q_out.dtype != kv.dtype:
            raise ValueError("q_out must have q's rows and the cache's type")
        qp, qop = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    cu = 0
    if cu_new is not None:
        if not (cu_new.get_device() == dev and cu_new.dtype == kv.lens.dtype and cu_new.is_contiguous()
                and cu_new.numel() == kv.n_seqs + 1):
            raise ValueError("cu_new must be contiguous int32 [n_seqs + 1]")
        cu = cu_new.data_ptr()
    rope_len = 0
    if rope is not None:
        if rope.dim() != 3 or rope.shape[2] != 2:
            raise ValueError("rope must be [length, head_dim / 2, 2]")
        rope_len = rope.shape[0]
    rc = lib.abra_paged_append(
        kv._ref, qp, k.data_ptr(), v.data_ptr(), types[dtype], ldq, ldk, ldv, heads, cu, n,
        _vector(q_norm, "q_norm", hd, kv), _vector(k_norm, "k_norm", hd, kv), eps,
        _vector(rope, "rope", rope_len * hd, kv), rope_len, qop, ldqo, kv._stream(stream))
    if rc:
        _lib.check(rc, "abra_paged_append")
    return q_out


def _bytes(workspace, kv: PagedKV) -> tuple[int, int]:
    if workspace.get_device() != kv._index or not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous on the cache's device")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _size(n: int, func: str) -> int:
    if n < 0:
        _lib.check(int(n), func)
    return n


def paged_attention_workspace(kv: PagedKV, n_heads: int, n_q: int = 1, accumulate: bool = False, stream=None):
    """A workspace for :func:`paged_attention` with these arguments
    (uninitialised bytes, allocated on ``stream``).  One serves any number of
    calls that follow one another, all layers' among them; calls on several
    streams need one each."""
    import torch

    n = lib.abra_paged_attention_workspace(kv._ref, n_heads, n_q, ABRA_PAGED_ACCUMULATE if accumulate else 0)
    return _empty(kv, _size(n, "abra_paged_attention_workspace"), torch.uint8, stream)


def paged_attention(kv: PagedKV, q, scale: float, out=None, lse=None, accumulate: bool = False,
                    workspace=None, stream=None):
    """Attention of each sequence's newest n_q tokens over its cached slots
    (abra_paged_attention): q [n_seqs, n_q, heads, head_dim] (or [n_seqs,
    heads, head_dim] for one token) in the cache's type; query j sees the slots
    before lens - n_q + j + 1; up to 4,096 of them, though the work is that of all
    slots for each.  Returns out, of q's shape and the cache's type unless a
    float32 ``out`` is given (it may be other columns of q's rows).  lse: float32 [n_seqs, n_q, heads], log
    of the softmax's denominator.  accumulate: add every slot's weight to
    kv.acc."""
    dev, hd, shape = kv._index, kv.head_dim, q.shape
    if len(shape) not in (3, 4) or shape[0] != kv.n_seqs or shape[-1] != hd or q.dtype != kv.dtype:
        raise ValueError("q must be [n_seqs, n_q, heads, head_dim] in the cache's type")
    heads, n_q = shape[-2], shape[1] if len(shape) == 4 else 1
    width = heads * hd
    _, ldq = _rows(q, "q", width, dev)
    if out is None:
        out = _empty(kv, shape, kv.dtype, stream)
    out_type = kv._types.get(out.dtype)
    if out.numel() != q.numel() or (out.dtype != kv.dtype and out_type != ABRA_GGML_F32):
        raise ValueError("out must be like q, in the cache's type or float32")
    _, ldo = _rows(out, "out", width, dev)
    flags = ABRA_PAGED_ACCUMULATE if accumulate else 0
    if workspace is None:
        workspace = paged_attention_workspace(kv, heads, n_q, accumulate, stream)
    rc = lib.abra_paged_attention(
        kv._ref, q.data_ptr(), ldq, heads, n_q, scale, out.data_ptr(), out_type, ldo,
        _vector(lse, "lse", kv.n_seqs * n_q * heads, kv), flags, *_bytes(workspace, kv), kv._stream(stream))
    if rc:
        _lib.check(rc, "abra_paged_attention")
    return out


def paged_evict_workspace(kv: PagedKV, budget: int, stream=None):
    """A workspace for :func:`paged_evict` with this budget (uninitialised
    bytes, allocated on ``stream``)."""
    import torch

    n = lib.abra_paged_evict_workspace(kv._ref, budget)
    return _empty(kv, _size(n, "abra_paged_evict_workspace"), torch.uint8, stream)


def paged_evict(kv: PagedKV, budget: int, n_sink: int = 0, n_recent: int = 0, new_lens=None,
                workspace=None, stream=None):
    """Cut every sequence to at most ``budget`` slots, each kv head by itself
    (abra_paged_evict): positions below n_sink, the n_recent newest positions
    and the largest accumulated weights stay; kept rows beyond the budget move
    into the evicted slots below it.  Returns new_lens, int32 [n_seqs]; kv.lens
    is not changed, so that every layer's cache can be cut before
    ``kv.lens.copy_(new_lens)``."""
    if new_lens is None:
        new_lens = _empty(kv, kv.n_seqs, kv.lens.dtype, stream)
    elif not (new_lens.get_device() == kv._index and new_lens.dtype == kv.lens.dtype
              and new_lens.is_contiguous() and new_lens.numel() == kv.n_seqs):
        raise ValueError("new_lens must be contiguous int32 [n_seqs] on the cache's device")
    if workspace is None:
        workspace = paged_evict_workspace(kv, budget, stream)
    rc = lib.abra_paged_evict(kv._ref, budget, n_sink, n_recent, new_lens.data_ptr(), *_bytes(workspace, kv),
                              kv._stream(stream))
    if rc:
        _lib.check(rc, "abra_paged_evict")
    return new_lens
