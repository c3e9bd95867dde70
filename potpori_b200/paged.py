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

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import PACK_APPEND, PACK_BATCH, PACK_QUERY, PP_E_INVALID, PPError, check

DTYPES = {torch.float32: _lib.PP_F32, torch.bfloat16: _lib.PP_BF16, torch.float16: _lib.PP_F16}


def _refuse(message: str):
    raise PPError(PP_E_INVALID, message)


# The current stream's handle by device index, without building a Stream object where this torch
# can say it.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _pointer(name: str, t: torch.Tensor, index: int, dtype: torch.dtype, shape: tuple) -> int:
    """Device pointer of a contiguous tensor of this type and shape on device `index`."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        _refuse(f"{name}: a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{index} expected, got "
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
        if not 0 <= max_rows < 1 << 31 or not 0 <= (max_length or 0) < 1 << 31:
            _refuse("max_rows and max_length must not be negative")
        self.index = page_table.get_device()
        if self.index < 0:
            _refuse("the batch's tensors must be on a CUDA device")
        self.page_table, self.lengths, self.cu_rows = page_table, lengths, cu_rows
        self.size, self.width, self.max_rows, self.max_length = n, stride, int(max_rows), max_length
        i32 = torch.int32
        self._ptr = (_pointer("cu_rows", cu_rows, self.index, i32, (n + 1,)),
                     _pointer("lengths", lengths, self.index, i32, (n,)),
                     _pointer("page_table", page_table, self.index, i32, (n, stride)))

    def _desc(self, cache: "PagedCache", rows: int) -> bytes:
        if self.index != cache.index:
            _refuse(f"the batch is on cuda:{self.index}, the cache on cuda:{cache.index}")
        most = self.max_length
        if most is None:
            most = min(self.width * cache.page_size, 0x7FFFFFFF)
        return PACK_BATCH.pack(self.size, rows, self.max_rows, most, self.width, *self._ptr)


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
        self.device, self.index, self.dtype = k.device, k.get_device(), k.dtype
        self.layers = k.shape[0] if k.dim() == 5 else 1
        row, head = (-3, -2) if layout == "nhd" else (-2, -3)
        self.pages, self.page_size = k.shape[-4], k.shape[row]
        self.kv_heads, self.head_dim = k.shape[head], k.shape[-1]
        self.err = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._c = bytes(_lib.PagedCacheDesc(
            k.data_ptr(), v.data_ptr(), DTYPES[k.dtype], self.layers, self.pages, self.page_size,
            self.kv_heads, self.head_dim, k.stride(0) if k.dim() == 5 else 0, k.stride(-4),
            k.stride(row), k.stride(head), self.index))
        self._err = self.err.data_ptr()

    def check(self) -> None:
        """Raises when a call on this cache met a length or a page outside the table or the
        cache, or a device wait that ran out (synchronises), and clears the mark."""
        bits = int(self.err.item())
        if bits:
            self.err.zero_()
            if bits & 4:
                raise PPError(_lib.PP_E_TIMEOUT, "a wait on the device expired: outputs are undefined")
            raise PPError(PP_E_INVALID, "a length or page table entry outside the table or the cache")

    def _rows(self, name: str, t: torch.Tensor, rows: int, heads: int, dtype: torch.dtype) -> int:
        """Row stride of t, [rows, heads, dim] with the heads of a row adjacent."""
        dim = self.head_dim
        if t.shape != (rows, heads, dim) or t.dtype is not dtype or t.get_device() != self.index:
            _refuse(f"{name}: {dtype} [{rows}, {heads}, {dim}] on {self.device} expected, got {t.dtype} "
                    f"{tuple(t.shape)} on {t.device}")
        row, head, one = t.stride()
        if one != 1 or (head != dim and heads > 1):
            _refuse(f"{name}: the heads of a row must be adjacent")
        return row

    def append(self, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor,
               q: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
               positions: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
               k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
               layer: int = 0, out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Write the rows k, v [rows, kv_heads, dim] into the pages of their positions, k normed
        and rotated on the way; returns q [rows, heads, dim] normed and rotated likewise in the
        cache's type (None without q). inv_freq [rotary_dim / 2] float64 radians per position."""
        rows, dtype, index = k.shape[0], k.dtype, self.index
        if dtype not in DTYPES:
            _refuse("k, v and q must be float32, bfloat16 or float16")
        k_stride = self._rows("k", k, rows, self.kv_heads, dtype)
        v_stride = self._rows("v", v, rows, self.kv_heads, dtype)
        qp = op = heads = q_stride = 0
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else 0
            q_stride = self._rows("q", q, rows, heads, dtype)
            if out is None:
                out = torch.empty((rows, heads, self.head_dim), dtype=self.dtype, device=self.device)
                op = out.data_ptr()
            else:
                op = _pointer("out", out, index, self.dtype, (rows, heads, self.head_dim))
            qp = q.data_ptr()
        elif out is not None:
            _refuse("out without q")
        fp = rotary = 0
        if inv_freq is not None:
            rotary = 2 * inv_freq.numel()
            fp = _pointer("inv_freq", inv_freq, index, torch.float64, (rotary // 2,))
        qn = 0 if q_norm is None else _pointer("q_norm", q_norm, index, torch.float32, (self.head_dim,))
        kn = 0 if k_norm is None else _pointer("k_norm", k_norm, index, torch.float32, (self.head_dim,))
        pos = 0 if positions is None else _pointer("positions", positions, index, torch.int32, (rows,))
        if not 0 <= layer < self.layers:
            _refuse("layer outside the cache")
        if rows:
            a = PACK_APPEND.pack(qp, k.data_ptr(), v.data_ptr(), op, DTYPES[dtype], heads, q_stride,
                                 k_stride, v_stride, pos, fp, rotary, bool(interleaved), qn, kn, eps, layer)
            st = self._L.pp_paged_append(self._c, batch._desc(self, rows), a, self._err, _stream(index))
            if st:
                check(st, None, "append")
        return out

    def tree_attention(self, batch: PagedBatch, q: torch.Tensor, mask: Optional[torch.Tensor] = None,
                       scale: Optional[float] = None, layer: int = 0,
                       out: Optional[torch.Tensor] = None,
                       lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q [rows, heads, dim] (the cache's type) over the cache. Row i of a sequence
        sees its context and the nodes j whose bit j % 32 of mask[row, j // 32] (int32 words) is
        set; without a mask the rows are a chain. scale defaults to dim ** -0.5. lse, optional:
        [rows, heads] float32, receives the log of the softmax's sum."""
        if q.dim() != 3:
            _refuse("q: [rows, heads, dim] expected")
        rows, heads, dim = q.shape
        index = self.index
        q_stride = self._rows("q", q, rows, heads, self.dtype)
        if out is None:
            out = torch.empty((rows, heads, dim), dtype=self.dtype, device=self.device)
            op = out.data_ptr()
        else:
            op = _pointer("out", out, index, self.dtype, (rows, heads, dim))
        lp = 0 if lse is None else _pointer("lse", lse, index, torch.float32, (rows, heads))
        mp = words = 0
        if mask is not None:
            words = mask.shape[1] if mask.dim() == 2 else 0
            mp = _pointer("mask", mask, index, torch.int32, (rows, words))
        if not 0 <= layer < self.layers:
            _refuse("layer outside the cache")
        if rows:
            L, b = self._L, batch._desc(self, rows)
            a = PACK_QUERY.pack(q.data_ptr(), op, lp, q_stride, heads, layer, mp, words,
                                dim ** -0.5 if scale is None else scale)
            need = L.pp_tree_attention_work_bytes(self._c, b, heads)
            if not need:
                check(PP_E_INVALID, None, "tree_attention")
            work = torch.empty(need, dtype=torch.uint8, device=self.device)
            st = L.pp_tree_attention(self._c, b, a, work.data_ptr(), need, self._err, _stream(index))
            if st:
                check(st, None, "tree_attention")
        return out

    def tree_commit(self, batch: PagedBatch, tokens: torch.Tensor, parents: torch.Tensor,
                    picks: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """Accept every tree's longest path that the target's picks follow and move its K/V rows,
        in every layer, to the front of the tree's. tokens, parents, picks: [rows] int32. Returns
        (path [batch, max_rows], accepted, correction, lengths), int32."""
        n, shape, width, i32, index = batch.size, tokens.shape, max(batch.max_rows, 1), torch.int32, self.index
        if len(shape) != 1:
            _refuse("tokens: [rows] expected")
        # A batch without rows has no arrays: any valid pointer stands in.
        tp = _pointer("tokens", tokens, index, i32, shape) or self._err
        pp = _pointer("parents", parents, index, i32, shape) or self._err
        kp = _pointer("picks", picks, index, i32, shape) or self._err
        out = torch.empty(n * (width + 3), dtype=i32, device=self.device)
        at = out.data_ptr()
        a, c, l = at + 4 * n * width, at + 4 * n * (width + 1), at + 4 * n * (width + 2)
        st = self._L.pp_tree_commit(self._c, batch._desc(self, shape[0]), tp, pp, kp, at, width, a, c, l,
                                    self._err, _stream(index))
        if st:
            check(st, None, "tree_commit")
        path, accepted, correction, lengths = out.split((n * width, n, n, n))
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
        new, index, i32 = beams.shape[1], self.index, torch.int32
        tp = _pointer("page_table", page_table, index, i32, (g, old, stride))
        lp = _pointer("lengths", lengths, index, i32, (g, old))
        bp = _pointer("beams", beams, index, i32, (g, new))
        sp = _pointer("spare", spare, index, i32, (g, new))
        out = torch.empty(g * new * (stride + 2), dtype=i32, device=self.device)
        at, n = out.data_ptr(), g * new
        st = self._L.pp_beam_reorder(self._c, tp, lp, g, old, new, stride, bp, sp, at, at + 4 * n * stride,
                                     at + 4 * n * (stride + 1), self._err, _stream(index))
        if st:
            check(st, None, "beam_reorder")
        table, length, taken = out.split((n * stride, n, n))
        return table.view(g, new, stride), length.view(g, new), taken.view(g, new)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int,
                finished: Optional[torch.Tensor] = None, pad: int = 0,
                err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The k best continuations of every group of beams: logits [groups, beams, vocab], scores
    [groups, beams] float32 running log-probabilities (-inf: not in use), finished [groups, beams]
    bool or uint8 (such a beam goes on only as token `pad`, its score unchanged). Returns scores
    float32, beams int32, tokens int32, each [groups, k], best first, ties to the lower beam and
    token; -inf, -1, -1 where candidates run out. err: int32 [1], gets value 2 where a beam was left
    out for a NaN or +inf."""
    index = logits.get_device()
    if logits.dim() != 3 or logits.dtype not in DTYPES or index < 0:
        _refuse("logits: [groups, beams, vocab] float32, bfloat16 or float16 on a CUDA device expected")
    g, w, vocab = logits.shape
    gs, ws, one = logits.stride()
    if (vocab > 1 and one != 1) or (g > 1 and w > 1 and gs != w * ws):
        _refuse("logits: contiguous rows, evenly spaced, expected")
    row = ws if w > 1 else gs if g > 1 else vocab
    sp = _pointer("scores", scores, index, torch.float32, (g, w))
    fin = None
    if finished is not None:
        fin = _pointer("finished", finished, index,
                       torch.uint8 if finished.dtype is torch.uint8 else torch.bool, (g, w))
    e = None if err is None else _pointer("err", err, index, torch.int32, (1,))
    if k < 1:
        _refuse("k must be positive")
    L = _lib.load()
    need = L.pp_beam_select_work_bytes(g, w, vocab, k)
    work = torch.empty(max(need, 16), dtype=torch.uint8, device=logits.device)
    out = torch.empty((3, g, k), dtype=torch.int32, device=logits.device)
    at = out.data_ptr()
    st = L.pp_beam_select(logits.data_ptr(), DTYPES[logits.dtype], row, sp, fin, pad, g, w, vocab, k, at,
                          at + 4 * g * k, at + 8 * g * k, work.data_ptr(), need, e, index, _stream(index))
    if st:
        check(st, None, "beam_select")
    best, beams, tokens = out.unbind(0)
    return best.view(torch.float32), beams, tokens
