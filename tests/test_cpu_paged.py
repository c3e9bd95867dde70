"""What the paged operators refuse before any device work, through the C ABI, and the Python
layer's checks: no GPU takes part."""
import ctypes

import pytest
import torch

from potpori_b200 import _lib
from potpori_b200._lib import PPError

FAKE = 1 << 20  # an aligned address that the host checks never read


def cache(**kw):
    d = dict(k=FAKE, v=FAKE, dtype=_lib.PP_BF16, layers=2, n_pages=64, page_size=16, n_kv_heads=2, head_dim=128,
             layer_stride=64 * 16 * 256, page_stride=16 * 256, row_stride=256, head_stride=128, cuda_device=0)
    d.update(kw)
    return _lib.PagedCacheDesc(**d)


def batch(**kw):
    d = dict(batch=3, rows=6, max_rows=2, max_len=100, table_stride=8, cu_rows=FAKE, kv_len=FAKE + 64, page_table=FAKE)
    d.update(kw)
    return _lib.PagedBatchDesc(**d)


def rows(**kw):
    d = dict(q=FAKE, k=FAKE, v=FAKE, q_out=FAKE + 4096, dtype=_lib.PP_F32, n_heads=4, q_stride=1024, k_stride=1024,
             v_stride=1024, inv_freq=FAKE, rotary_dim=128, eps=1e-6, layer=0)
    d.update(kw)
    return _lib.AppendRows(**d)


def query(**kw):
    d = dict(q=FAKE, out=FAKE + 4096, q_stride=512, n_heads=4, layer=0, scale=0.1)
    d.update(kw)
    return _lib.TreeQuery(**d)


def refused(status, *say):
    assert status in (_lib.PP_E_INVALID, _lib.PP_E_UNSUPPORTED)
    text = _lib.last_error(None)
    assert all(s in text for s in say), text


BAD_CACHES = [dict(k=None), dict(dtype=3), dict(layers=0), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0),
              dict(head_dim=0), dict(head_dim=100), dict(head_dim=264), dict(k=FAKE + 2), dict(page_stride=4097),
              dict(row_stride=64), dict(head_stride=-128), dict(head_stride=64), dict(n_pages=2 ** 31),
              dict(page_size=2 ** 21)]
BAD_BATCHES = [dict(batch=0), dict(batch=4097), dict(cu_rows=None), dict(kv_len=None), dict(page_table=None),
               dict(table_stride=0), dict(rows=2 ** 25)]


@pytest.mark.parametrize("bad", BAD_CACHES + BAD_BATCHES, ids=str)
def test_bad_descriptors_are_refused_by_every_operator(bad):
    L = _lib.load()
    of_cache = bad in BAD_CACHES
    c = cache(**bad) if of_cache else cache()
    b = batch() if of_cache else batch(**bad)
    p, r = ctypes.byref(c), ctypes.byref(b)
    refused(L.pp_paged_append(p, r, ctypes.byref(rows()), None, None))
    refused(L.pp_tree_attention(p, r, ctypes.byref(query()), FAKE, 1 << 40, None, None))
    assert L.pp_tree_attention_work_bytes(p, r, 4) == 0
    refused(L.pp_tree_commit(p, r, FAKE, FAKE, FAKE, FAKE, 8, FAKE, FAKE, FAKE + 8, None, None))
    if of_cache:
        refused(L.pp_beam_reorder(p, FAKE, FAKE, 1, 4, 4, 8, FAKE, FAKE, FAKE + 8, FAKE + 16, FAKE + 24, None, None))


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(dtype=3), dict(q=None), dict(q_out=None),
                                 dict(n_heads=0), dict(layer=2), dict(rotary_dim=0), dict(rotary_dim=7),
                                 dict(rotary_dim=130), dict(k_stride=100), dict(v_stride=100), dict(q_stride=100),
                                 dict(k=FAKE + 2), dict(q_out=FAKE + 1), dict(q_out=FAKE)], ids=str)
def test_append_refusals(bad):
    refused(_lib.load().pp_paged_append(ctypes.byref(cache()), ctypes.byref(batch()), ctypes.byref(rows(**bad)), None,
                                        None))


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(n_heads=0), dict(n_heads=5), dict(layer=2),
                                 dict(q=FAKE + 8), dict(out=FAKE + 8), dict(q_stride=500), dict(q_stride=256),
                                 dict(mask=FAKE), dict(mask=FAKE, mask_words=40000), dict(out=FAKE)], ids=str)
def test_attention_refusals(bad):
    L = _lib.load()
    c, b = cache(), batch()
    refused(L.pp_tree_attention(ctypes.byref(c), ctypes.byref(b), ctypes.byref(query(**bad)), FAKE, 1 << 40, None,
                                None))


def test_work_and_commit_and_beam_refusals():
    L = _lib.load()
    c, b = ctypes.byref(cache()), ctypes.byref(batch())
    assert L.pp_tree_attention(c, b, None, FAKE, 1 << 40, None, None) == _lib.PP_E_INVALID
    refused(L.pp_tree_commit(c, b, None, FAKE, FAKE, FAKE, 8, FAKE, FAKE, FAKE, None, None))
    refused(L.pp_tree_commit(c, b, FAKE, FAKE, FAKE, FAKE, 1, FAKE, FAKE, FAKE, None, None), "path_stride")
    refused(L.pp_tree_commit(c, b, FAKE, FAKE, FAKE, FAKE, 8, FAKE, FAKE, FAKE + 64, None, None), "kv_len")
    refused(L.pp_tree_commit(c, ctypes.byref(batch(max_rows=1025)), FAKE, FAKE, FAKE, FAKE, 2000, FAKE, FAKE, FAKE,
                             None, None), "1024")
    ok = dict(logits=FAKE, dtype=_lib.PP_F32, stride=1000, scores=FAKE, fin=None, pad=0, groups=2, beams=4, vocab=1000,
              k=4, s=FAKE, b=FAKE, t=FAKE, work=FAKE, n=1 << 30, err=None, dev=0, stream=None)
    for bad in (dict(logits=None), dict(dtype=3), dict(stride=999), dict(scores=None), dict(groups=0), dict(beams=0),
                dict(beams=65), dict(k=0), dict(k=65), dict(vocab=0), dict(vocab=2 ** 25, stride=2 ** 25),
                dict(groups=20000), dict(logits=FAKE + 2), dict(work=None), dict(work=FAKE + 8), dict(n=10),
                dict(s=None), dict(b=None), dict(t=None)):
        refused(L.pp_beam_select(*{**ok, **bad}.values()))
    order = dict(c=c, t=FAKE, l=FAKE + 8, g=1, old=4, new=4, stride=8, beams=FAKE + 16, spare=FAKE, nt=FAKE + 24,
                 nl=FAKE + 32, taken=FAKE + 40, err=None, stream=None)
    for bad in (dict(t=None), dict(l=None), dict(g=0), dict(old=0), dict(new=0), dict(stride=0), dict(beams=None),
                dict(spare=None), dict(nt=None), dict(nl=None), dict(taken=None), dict(nt=FAKE), dict(nl=FAKE + 8),
                dict(nl=FAKE + 16), dict(taken=FAKE + 16), dict(g=70000)):
        refused(L.pp_beam_reorder(*{**order, **bad}.values()))


def test_outputs_that_are_inputs_are_refused():
    """Other CTAs of the call still read them."""
    L = _lib.load()
    c, b = ctypes.byref(cache()), ctypes.byref(batch())
    ok = dict(c=c, b=b, tokens=FAKE + 1024, parents=FAKE + 2048, picks=FAKE + 4096, path=FAKE + 8192, stride=8,
              accepted=FAKE + 8200, correction=FAKE + 8208, lengths=FAKE + 8216, err=None, stream=None)
    for bad in (dict(path=FAKE + 1024), dict(accepted=FAKE + 2048), dict(correction=FAKE + 4096), dict(lengths=FAKE + 1024)):
        refused(L.pp_tree_commit(*{**ok, **bad}.values()), "inputs")
    refused(L.pp_beam_select(FAKE, _lib.PP_F32, 1000, FAKE, None, 0, 2, 4, 1000, 4, FAKE, FAKE + 64, FAKE + 128, FAKE,
                             1 << 30, None, 0, None), "scores")
    for out in ("k", "v"):
        r = rows()
        r.q_out = getattr(r, out)
        refused(L.pp_paged_append(c, b, ctypes.byref(r), None, None), "q_out")
    order = dict(c=c, t=FAKE, l=FAKE + 8, g=1, old=4, new=4, stride=8, beams=FAKE + 16, spare=FAKE + 48, nt=FAKE + 24,
                 nl=FAKE + 32, taken=FAKE + 40, err=None, stream=None)
    for bad in (dict(taken=FAKE + 48), dict(nl=FAKE + 48), dict(nt=FAKE + 8)):
        refused(L.pp_beam_reorder(*{**order, **bad}.values()), "inputs")


def test_work_bytes():
    L = _lib.load()
    small = L.pp_tree_attention_work_bytes(ctypes.byref(cache()), ctypes.byref(batch(batch=1, rows=1, max_len=10)), 4)
    large = L.pp_tree_attention_work_bytes(ctypes.byref(cache()), ctypes.byref(batch(rows=60, max_rows=20, max_len=10 ** 6)), 4)
    assert 0 < small < large < 64 << 20
    assert L.pp_beam_select_work_bytes(1, 1, 1, 1) > 0


def test_shards_refuse_f16_parameters():
    """PP_F16 is the paged operators' only; a shard's loader knows F32 and BF16."""
    assert _lib.PP_F16 == 2 and _lib.load().pp_shard_set_tensor(None, b"x", _lib.PP_F16, None, 0) == _lib.PP_E_INVALID


def test_python_layer_refuses_host_tensors():
    from potpori_b200.paged import PagedBatch, PagedCache, beam_select

    k = torch.zeros(4, 16, 2, 64)
    for args in ((k, k), (k, k, "xyz"), (k, k.half()), (k, torch.zeros(4, 16, 2, 128)), (k[0], k[0])):
        with pytest.raises(PPError):
            PagedCache(*args)
    t, n, cu = (torch.zeros(s, dtype=torch.int32) for s in ((2, 3), (2,), (3,)))
    for args in ((t, n, n, 1), (t[0], n, cu, 1), (t, n.long(), cu, 1), (t, n, cu, -1), (t[:, ::2], n, cu, 1)):
        with pytest.raises(PPError):
            PagedBatch(*args)
    with pytest.raises(PPError):
        beam_select(torch.zeros(1, 2, 3), torch.zeros(1, 2), 1)
