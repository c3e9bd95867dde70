"""Operators over a paged K/V cache that many sequences share, on torch tensors.

``PagedCache`` and ``PagedBatch`` describe a cache and a batch of sequences with new rows;
``append``, ``tree_attention``, ``tree_commit`` and ``beam_reorder`` are the cache's methods and
``beam_select`` stands alone. They are the device-pointer operators of
``include/potpori_b200.h`` (pp_paged_append and those after it), where their rules are written
down; the methods themselves are in ``csrc/pp_torch.cpp``. Every call enqueues on the current
stream of the cache's device and allocates its outputs and work buffers from torch's allocator,
so calls on several streams, and captured graphs, do not share any. Tensors must be on the
cache's device and, as with torch's own operators, stay valid until the stream has passed them.
Errors that only the device can see (a length or page outside the table or the cache) gather in
``PagedCache.err``; ``check`` reads it.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import PP_E_INVALID, PP_E_NONFINITE, PP_E_TIMEOUT, PPError

_lib.load()  # the library that the binding calls; raises where it was never built
try:
    from . import _paged  # noqa: E402
    from ._paged import beam_select  # noqa: E402,F401
except ImportError as e:
    raise ImportError("potpori_b200/_paged.so is absent or was built for another torch or Python: run "
                      f"`python -m potpori_b200.build` where torch is installed ({e})") from e

DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class PagedBatch(_paged.Batch):
    """Sequences with new rows: sequence b owns rows ``cu_rows[b]:cu_rows[b + 1]`` of a call's row
    tensors, which are the last of its ``lengths[b]`` cached positions; position s is row
    ``s % page_size`` of page ``page_table[b, s // page_size]``. All int32 on the device, so a
    captured graph replays with new contents. ``max_rows`` and ``max_length`` are the host's
    bounds.

    PagedBatch(page_table, lengths, cu_rows, max_rows, max_length=None)"""


class PagedCache(_paged.Cache):
    """K and V pools of one shape and one set of strides: ``[pages, page_size, heads, dim]``
    (layout "nhd") or ``[pages, heads, page_size, dim]`` ("hnd"), with a leading ``layers``
    dimension when 5-dimensional. Views qualify (K and V interleaved in one pool) as long as dim
    is contiguous and the other strides are multiples of 16 bytes."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, layout: str = "nhd"):
        def refuse(message):
            raise PPError(PP_E_INVALID, message)

        if layout not in ("nhd", "hnd"):
            refuse("layout must be 'nhd' or 'hnd'")
        if k.dim() not in (4, 5) or k.shape != v.shape or k.stride() != v.stride():
            refuse("k and v: 4 or 5 dimensions of equal shapes and strides expected")
        if k.dtype != v.dtype or k.dtype not in DTYPES:
            refuse("k and v must both be float32, bfloat16 or float16")
        if not k.is_cuda or k.device != v.device:
            refuse("k and v must be on one CUDA device")
        if k.stride(-1) != 1:
            refuse("the last dimension must be contiguous")
        super().__init__(k, v, torch.zeros(1, dtype=torch.int32, device=k.device), layout == "nhd")
        row, head = (-3, -2) if layout == "nhd" else (-2, -3)
        self.layout, self.device, self.dtype = layout, k.device, k.dtype
        self.layers = k.shape[0] if k.dim() == 5 else 1
        self.pages, self.page_size = k.shape[-4], k.shape[row]
        self.kv_heads, self.head_dim = k.shape[head], k.shape[-1]

    def check(self) -> None:
        """Raises when a call on this cache met rows outside the row tensors, a length or a page
        outside the table or the cache, or a device wait that ran out, or a ``beam_select`` that
        was given ``err`` left a beam out (synchronises), and clears the marks. The first of
        timeout, bad descriptor and beam gives the status; the message names all."""
        bits = int(self.err.item())
        if bits:
            self.err.zero_()
            found = [(status, text) for bit, status, text in (
                (4, PP_E_TIMEOUT, "a wait on the device expired: outputs are undefined"),
                (1, PP_E_INVALID, "rows, a length or a page table entry outside the arrays, the table or the cache"),
                (2, PP_E_NONFINITE, "a beam was left out for a NaN or +inf")) if bits & bit]
            raise PPError(found[0][0], "; ".join(text for _, text in found))
