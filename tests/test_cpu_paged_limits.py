"""Limits of the paged operators that only very large arguments reach, on the host."""
import ctypes

from potpori_b200 import _lib

FAKE = 1 << 20  # an aligned address that the host checks never read


def test_tables_whose_positions_would_wrap():
    """Tiles are counted from a length in 32 bits: a table that allows lengths up to 2^31 is refused."""
    L = _lib.load()

    def need(table_stride, page_size):
        c = _lib.PagedCacheDesc(k=FAKE, v=FAKE, dtype=_lib.PP_BF16, layers=1, n_pages=64, page_size=page_size,
                                n_kv_heads=1, head_dim=64, layer_stride=0, page_stride=64 * page_size, row_stride=64,
                                head_stride=64, cuda_device=0)
        b = _lib.PagedBatchDesc(batch=1, rows=1, max_rows=1, max_len=100, table_stride=table_stride, cu_rows=FAKE,
                                kv_len=FAKE, page_table=FAKE)
        return L.pp_tree_attention_work_bytes(ctypes.byref(c), ctypes.byref(b), 1)

    assert need(2 ** 27 - 1, 16) == 0 and "2^31" in _lib.last_error(None)
    assert need(2 ** 27 - 255, 16) == 0
    assert need(2 ** 27 - 256, 16) > 0 and need(1000, 16) > 0
