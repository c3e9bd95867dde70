"""Operators over a paged K/V cache that many sequences share, on torch tensors.

``PagedCache`` and ``PagedBatch`` describe a cache and a batch of sequences with new rows;
``append``, ``tree_attention``, ``tree_commit`` and ``beam_reorder`` are the cache's methods and
``beam_select`` stands alone. They are the device-pointer operators of
``include/potpori_b200.h`` (pp_paged_append and those after it), where their rules are written
down. Every call enqueues on the current stream of the cache's device and allocates its outputs
and work buffers from torch's allocator, so calls on several streams, and captured graphs, do not
share any. Tensors must be on the cache's device and, as with torch's own operators, stay valid
until the stream has passed them. Errors that only the device can see (a length or page outside
the table or the cache) gather in ``PagedCache.err``; ``check`` reads it.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import PP_E_INVALID, PPError, check

DTYPES = {torch.float32: _lib.PP_F32, torch.bfloat16: _lib.PP_BF16, torch.float16: _lib.PP_F16}


def _refuse(message: str):
    raise PPError(PP_E_INVALID, message)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ints(name: str, t: torch.Tensor, device: torch.device, shape: tuple) -> int:
    """Device pointer of a contiguous int32 tensor of `shape`."""
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != shape or not t.is_contiguous():
        _refuse(f"{name}: a contiguous int32 tensor of shape {shape} on {device} expected, got "
                f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


class PagedBatch:
    """Sequences with new rows: sequence b owns rows ``cu_rows[b]:cu_rows[b + 1]`` of a call's row
    tensors, which are the last of its ``lengths[b]`` cached positions; position s is row
    ``s % page_size`` of page ``page_table[b, s // page_size]``. All int32 on the device, so a
    captured graph replays with new contents. ``max_rows`` and ``max_length`` are the host's
    bounds."""

    def __init__(self, page_table: torch.Tensor, lengths: torch.Tensor, cu_rows: torch.Tensor,
                 max_rows: int, max_length: Optional[int] = None):
        if page_table.dim() != 2 or page_table.shape[1] == 0:
            _refuse("page_table: [batch, pages] expected")
        n, stride = page_table.shape
        if max_rows < 0 or (max_length is not None and max_length < 0):
            _refuse("max_rows and max_length must not be negative")
        dev = page_table.device
        self.page_table, self.lengths, self.cu_rows = page_table, lengths, cu_rows
        self.device, self.size, self.max_rows = dev, n, int(max_rows)
        self.max_length = max_length
        self._c = _lib.PagedBatchDesc(
            n, 0, max_rows, max_length or 0, stride, _ints("cu_rows", cu_rows, dev, (n + 1,)),
            _ints("lengths", lengths, dev, (n,)), _ints("page_table", page_table, dev, (n, stride)))

    def _desc(self, cache: "PagedCache", rows: int) -> _lib.PagedBatchDesc:
        if self.device != cache.device:
            _refuse(f"the batch is on {self.device}, the cache on {cache.device}")
        c = _lib.PagedBatchDesc.from_buffer_copy(self._c)
        c.rows = rows
        if self.max_length is None:
            c.max_len = min(self.page_table.shape[1] * cache.page_size, 0x7FFFFFFF)
        return c


class PagedCache:
    """K and V pools of one shape and one set of strides: ``[pages, page_size, heads, dim]``
    (layout "nhd") or ``[pages, heads, page_size, dim]`` ("hnd"), with a leading ``layers``
    dimension when 5-dimensional. Views qualify (K and V interleaved in one pool) as long as dim
    is contiguous and the other strides are multiples of 16 bytes."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, layout: str = "nhd"):
        if layout not in ("nhd", "hnd"):
            _refuse("layout must be 'nhd' or 'hnd'")
        if k.dim() not in (4, 5) or k.shape != v.shape or k.stride() != v.stride():
            _refuse("k and v: 4 or 5 dimensions of equal shapes and strides expected")
        if k.dtype != v.dtype or k.dtype not in DTYPES:
            _refuse("k and v must both be float32, bfloat16 or float16")
        if not k.is_cuda or k.device != v.device:
            _refuse("k and v must be on one CUDA device")
        if k.stride(-1) != 1:
            _refuse("the last dimension must be contiguous")
        self._L = _lib.load()
        self.k, self.v, self.layout = k, v, layout
        self.device, self.dtype = k.device, k.dtype
        self.layers = k.shape[0] if k.dim() == 5 else 1
        row, head = (-3, -2) if layout == "nhd" else (-2, -3)
        self.pages, self.page_size = k.shape[-4], k.shape[row]
        self.kv_heads, self.head_dim = k.shape[head], k.shape[-1]
        self.err = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._c = _lib.PagedCacheDesc(
            k.data_ptr(), v.data_ptr(), DTYPES[k.dtype], self.layers, self.pages, self.page_size,
            self.kv_heads, self.head_dim, k.stride(0) if k.dim() == 5 else 0, k.stride(-4),
            k.stride(row), k.stride(head), k.device.index)
        self._ref = ctypes.byref(self._c)
        self._err = self.err.data_ptr()

    def check(self) -> None:
        """Raises when a call on this cache met a length or a page outside the table or the
        cache (synchronises), and clears the mark."""
        bits = int(self.err.item())
        if bits:
            self.err.zero_()
            raise PPError(PP_E_INVALID, "a length or page table entry outside the table or the cache")

    def _rows(self, name: str, t: torch.Tensor, heads: Optional[int], rows: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> None:
        if (t.dim() != 3 or t.shape[2] != self.head_dim or (heads is not None and t.shape[1] != heads)
                or (rows is not None and t.shape[0] != rows)):
            _refuse(f"{name}: [{rows if rows is not None else 'rows'}, "
                    f"{heads if heads is not None else 'heads'}, {self.head_dim}] expected, got "
                    f"{tuple(t.shape)}")
        if t.device != self.device or t.dtype not in DTYPES or (dtype is not None and t.dtype != dtype):
            _refuse(f"{name}: {dtype or 'a floating type'} on {self.device} expected, got {t.dtype} on "
                    f"{t.device}")
        if (t.shape[2] > 1 and t.stride(2) != 1) or (t.shape[1] > 1 and t.stride(1) != self.head_dim):
            _refuse(f"{name}: the heads of a row must be adjacent")

    def append(self, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor,
               q: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
               positions: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
               k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
               layer: int = 0, out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Write the rows k, v [rows, kv_heads, dim] into the pages of their positions, k normed
        and rotated on the way; returns q [rows, heads, dim] normed and rotated likewise in the
        cache's type (None without q). inv_freq [rotary_dim / 2] float64 radians per position."""
        rows = k.shape[0]
        self._rows("k", k, self.kv_heads)
        self._rows("v", v, self.kv_heads, rows, k.dtype)
        a = _lib.AppendRows(k=k.data_ptr(), v=v.data_ptr(), dtype=DTYPES[k.dtype],
                            k_stride=k.stride(0), v_stride=v.stride(0), eps=eps, layer=layer,
                            interleaved=int(interleaved))
        if q is not None:
            self._rows("q", q, None, rows, k.dtype)
            if out is None:
                out = torch.empty(q.shape, dtype=self.dtype, device=self.device)
            elif out.shape != q.shape or out.dtype != self.dtype or not out.is_contiguous() or out.device != self.device:
                _refuse("out: a contiguous tensor of q's shape and the cache's type expected")
            a.q, a.q_out, a.n_heads, a.q_stride = q.data_ptr(), out.data_ptr(), q.shape[1], q.stride(0)
        elif out is not None:
            _refuse("out without q")
        if inv_freq is not None:
            if (inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous()
                    or inv_freq.device != self.device):
                _refuse("inv_freq: a contiguous float64 vector on the cache's device expected")
            a.inv_freq, a.rotary_dim = inv_freq.data_ptr(), 2 * inv_freq.numel()
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None:
                if (w.dtype != torch.float32 or tuple(w.shape) != (self.head_dim,) or not w.is_contiguous()
                        or w.device != self.device):
                    _refuse(f"{name}: a contiguous float32 [{self.head_dim}] on the cache's device expected")
                setattr(a, name, w.data_ptr())
        if positions is not None:
            a.positions = _ints("positions", positions, self.device, (rows,))
        if rows:
            check(self._L.pp_paged_append(self._ref, ctypes.byref(batch._desc(self, rows)), ctypes.byref(a),
                                          self._err, _stream(self.device)), None, "append")
        return out if q is not None else None

    def tree_attention(self, batch: PagedBatch, q: torch.Tensor, mask: Optional[torch.Tensor] = None,
                       scale: Optional[float] = None, layer: int = 0,
                       out: Optional[torch.Tensor] = None,
                       lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q [rows, heads, dim] (the cache's type) over the cache. Row i of a sequence
        sees its context and the nodes j whose bit j % 32 of mask[row, j // 32] (int32 words) is
        set; without a mask the rows are a chain. scale defaults to dim ** -0.5. lse, optional:
        [rows, heads] float32, receives the log of the softmax's sum."""
        self._rows("q", q, None, None, self.dtype)
        rows, heads = q.shape[0], q.shape[1]
        if out is None:
            out = torch.empty(q.shape, dtype=self.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != self.dtype or not out.is_contiguous() or out.device != self.device:
            _refuse("out: a contiguous tensor of q's shape and type expected")
        a = _lib.TreeQuery(q=q.data_ptr(), out=out.data_ptr(), q_stride=q.stride(0), n_heads=heads,
                           layer=layer, scale=self.head_dim ** -0.5 if scale is None else scale)
        if lse is not None:
            if (lse.dtype != torch.float32 or tuple(lse.shape) != (rows, heads) or not lse.is_contiguous()
                    or lse.device != self.device):
                _refuse("lse: a contiguous float32 [rows, heads] on the cache's device expected")
            a.lse = lse.data_ptr()
        if mask is not None:
            if mask.dim() != 2:
                _refuse("mask: [rows, words] expected")
            a.mask, a.mask_words = _ints("mask", mask, self.device, (rows, mask.shape[1])), mask.shape[1]
        if rows:
            b = batch._desc(self, rows)
            need = self._L.pp_tree_attention_work_bytes(self._ref, ctypes.byref(b), heads)
            if not need:
                check(PP_E_INVALID, None, "tree_attention")
            work = torch.empty(need, dtype=torch.uint8, device=self.device)
            check(self._L.pp_tree_attention(self._ref, ctypes.byref(b), ctypes.byref(a), work.data_ptr(),
                                            need, self._err, _stream(self.device)), None, "tree_attention")
        return out

    def tree_commit(self, batch: PagedBatch, tokens: torch.Tensor, parents: torch.Tensor,
                    picks: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """Accept every tree's longest path that the target's picks follow and move its K/V rows,
        in every layer, to the front of the tree's. tokens, parents, picks: [rows] int32. Returns
        (path [batch, max_rows], accepted, correction, lengths), int32."""
        n, rows, width = batch.size, tokens.shape[0], max(batch.max_rows, 1)
        ptr = [_ints(name, t, self.device, (rows,)) if rows else self._err
               for name, t in (("tokens", tokens), ("parents", parents), ("picks", picks))]
        out = torch.empty(n * (width + 3), dtype=torch.int32, device=self.device)
        path, accepted, correction, lengths = out.split((n * width, n, n, n))
        check(self._L.pp_tree_commit(self._ref, ctypes.byref(batch._desc(self, rows)), *ptr,
                                     path.data_ptr(), width, accepted.data_ptr(), correction.data_ptr(),
                                     lengths.data_ptr(), self._err, _stream(self.device)),
              None, "tree_commit")
        return path.view(n, width), accepted, correction, lengths

    def beam_reorder(self, page_table: torch.Tensor, lengths: torch.Tensor, beams: torch.Tensor,
                     spare: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """States of new beams j continuing old beams beams[g, j]: (page table [groups, new, pages],
        lengths [groups, new], taken [groups, new]). Full pages are shared; a part-full last page
        stays with its first child and is copied, every layer, into page spare[g, j] for each other
        (taken[g, j] = 1)."""
        if page_table.dim() != 3 or beams.dim() != 2:
            _refuse("page_table: [groups, beams, pages] and beams: [groups, new beams] expected")
        g, old, stride = page_table.shape
        new, dev = beams.shape[1], self.device
        ptr = [_ints("page_table", page_table, dev, (g, old, stride)), _ints("lengths", lengths, dev, (g, old)),
               _ints("beams", beams, dev, (g, new)), _ints("spare", spare, dev, (g, new))]
        out = torch.empty(g * new * (stride + 2), dtype=torch.int32, device=dev)
        table, length, taken = out.split((g * new * stride, g * new, g * new))
        check(self._L.pp_beam_reorder(self._ref, ptr[0], ptr[1], g, old, new, stride, ptr[2], ptr[3],
                                      table.data_ptr(), length.data_ptr(), taken.data_ptr(), self._err,
                                      _stream(dev)), None, "beam_reorder")
        return table.view(g, new, stride), length.view(g, new), taken.view(g, new)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int,
                finished: Optional[torch.Tensor] = None, pad: int = 0,
                err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The k best continuations of every group of beams: logits [groups, beams, vocab], scores
    [groups, beams] float32 running log-probabilities (-inf: not in use), finished [groups, beams]
    bool or uint8 (such a beam goes on only as token `pad`, its score unchanged). Returns scores
    float32, beams int32, tokens int32, each [groups, k], best first, ties to the lower beam and
    token; -inf, -1, -1 where candidates run out. err: int32 [1], gets bit 2 where a beam was left
    out for a NaN or +inf."""
    if logits.dim() != 3 or logits.dtype not in DTYPES or not logits.is_cuda:
        _refuse("logits: [groups, beams, vocab] float32, bfloat16 or float16 on a CUDA device expected")
    g, w, vocab = logits.shape
    dev = logits.device
    if (vocab > 1 and logits.stride(2) != 1) or (
            g > 1 and w > 1 and logits.stride(0) != w * logits.stride(1)):
        _refuse("logits: contiguous rows, evenly spaced, expected")
    row = logits.stride(1) if w > 1 else logits.stride(0) if g > 1 else vocab
    if scores.dtype != torch.float32 or tuple(scores.shape) != (g, w) or not scores.is_contiguous() or scores.device != dev:
        _refuse("scores: a contiguous float32 [groups, beams] on the logits' device expected")
    fin = None
    if finished is not None:
        if (finished.dtype not in (torch.bool, torch.uint8) or tuple(finished.shape) != (g, w)
                or not finished.is_contiguous() or finished.device != dev):
            _refuse("finished: a contiguous bool [groups, beams] on the logits' device expected")
        fin = finished.data_ptr()
    e = None if err is None else _ints("err", err, dev, (1,))
    if k < 1:
        _refuse("k must be positive")
    L = _lib.load()
    need = L.pp_beam_select_work_bytes(g, w, vocab, k)
    work = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    out = torch.empty((3, g, k), dtype=torch.int32, device=dev)
    best, beams, tokens = out.unbind(0)
    best = best.view(torch.float32)
    check(L.pp_beam_select(logits.data_ptr(), DTYPES[logits.dtype], row, scores.data_ptr(), fin, pad, g, w,
                           vocab, k, best.data_ptr(), beams.data_ptr(), tokens.data_ptr(), work.data_ptr(),
                           need, e, dev.index, _stream(dev)), None, "beam_select")
    return best, beams, tokens
