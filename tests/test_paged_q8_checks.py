"""Refusals of the entries for int8 pages, windows over pages and stored rows, through the C ABI and without a GPU:
arguments are checked before the context, so a bad argument gives its own status and good ones with an unknown context
give RQ_ERR_HANDLE. Nothing is run."""
import ctypes as C

import pytest
import torch

import raster_amd.paged as paged
from raster_amd import _lib, attention
from raster_amd._lib import (RQ_BF16, RQ_ERR_DTYPE, RQ_ERR_HANDLE, RQ_ERR_NULL, RQ_ERR_SHAPE, RQ_F16, RQ_F32, RQ_I8,
                             RQ_OK)

CTX = C.c_void_p(0x1234)  # never dereferenced
P = 0x10000  # an aligned address, never dereferenced


def pages(**kw):
    a = dict(dtype=RQ_I8, kpages=P, vpages=P, pages=8, page_size=32, n_kv=2, head_dim=64, table=P, table_stride=4)
    a.update(kw)
    return _lib.Pages(*a.values())


def attend(pg, **kw):
    a = dict(ks=P, vs=P, ss=4, window=0, sinks=0, dtype=RQ_F32, q=P, qs=256, k=P, kst=128, v=P, vst=128, lens=P, batch=3,
             n_q=4, max_len=100, theta=1e4, scale=0.1, out=P, os=256, work=P, wb=1 << 40)
    a.update(kw)
    return _lib.lib().rq_paged_attention_window(CTX, C.byref(pg) if pg else None, *a.values(), None)


def append(pg, **kw):
    a = dict(ks=P, vs=P, ss=4, dtype=RQ_F32, q=P, qs=256, k=P, kst=128, v=P, vst=128, cu=P, past=P, batch=3, rows=9, n_q=4,
             theta=1e4, qo=P, qos=256, ko=P, kos=128)
    a.update(kw)
    return _lib.lib().rq_pages_append_q8(CTX, C.byref(pg) if pg else None, *a.values(), None)


def rows(pg, **kw):
    a = dict(ks=P, vs=P, ss=4, dtype=RQ_F32, cu=P, batch=3, rows=9, ko=P, kos=128, vo=P, vos=128)
    a.update(kw)
    return _lib.lib().rq_pages_rows(CTX, C.byref(pg) if pg else None, *a.values(), None)


@pytest.mark.parametrize("call", [attend, append, rows], ids=["attend", "append", "rows"])
def test_pages_and_scales(call):
    assert call(pages()) == RQ_ERR_HANDLE and call(pages(), dtype=RQ_BF16) == RQ_ERR_HANDLE
    assert call(pages(), ss=5) == RQ_ERR_HANDLE
    assert call(None) == RQ_ERR_NULL
    for kw in (dict(ks=None), dict(vs=None)):
        assert call(pages(), **kw) == RQ_ERR_NULL, kw
    for kw in (dict(ks=P + 2), dict(vs=P + 1), dict(ss=3), dict(ss=0), dict(ss=-4), dict(ss=2 ** 50)):
        assert call(pages(), **kw) == RQ_ERR_SHAPE, kw
    for kw in (dict(dtype=RQ_F16), dict(dtype=9)):
        assert call(pages(**kw)) == RQ_ERR_DTYPE, kw
    assert call(pages(), dtype=RQ_I8) == RQ_ERR_DTYPE and call(pages(), dtype=RQ_F16) == RQ_ERR_DTYPE
    for kw in (dict(page_size=8), dict(page_size=24), dict(pages=0), dict(head_dim=60), dict(head_dim=264),
               dict(n_kv=0), dict(kpages=P + 8), dict(vpages=P + 1), dict(table_stride=-1)):
        assert call(pages(**kw)) == RQ_ERR_SHAPE, kw
    assert call(pages(kpages=None)) == RQ_ERR_NULL and call(pages(table=None)) == RQ_ERR_NULL
    if call is not append:  # other pages have no scales
        assert call(pages(dtype=RQ_F32), ks=None, vs=None) == RQ_ERR_HANDLE
        assert call(pages(dtype=RQ_F32)) == RQ_ERR_DTYPE
        assert call(pages(dtype=RQ_F32), ks=None) == RQ_ERR_DTYPE
    else:
        assert call(pages(dtype=RQ_F32), ks=None, vs=None) == RQ_ERR_DTYPE


def test_attention_arguments():
    for kw in (dict(window=-1), dict(window=3, sinks=-1), dict(n_q=3), dict(batch=-1), dict(max_len=-1), dict(scale=0.0),
               dict(theta=-1.0), dict(qs=255), dict(os=8), dict(q=P + 4), dict(lens=P + 1)):
        assert attend(pages(), **kw) == RQ_ERR_SHAPE, kw
    for kw in (dict(k=None), dict(v=None), dict(q=None), dict(out=None), dict(lens=None)):
        assert attend(pages(), **kw) == RQ_ERR_NULL, kw
    for kw in (dict(k=None, v=None), dict(window=5, sinks=2), dict(window=2 ** 62, sinks=2 ** 62), dict(theta=0.0)):
        assert attend(pages(), **kw) == RQ_ERR_HANDLE, kw
        assert attend(pages(dtype=RQ_BF16), ks=None, vs=None, **kw) == RQ_ERR_HANDLE, kw
    assert attend(pages(), batch=0, q=None) == RQ_OK
    assert attend(pages(dtype=RQ_F32), ks=None, vs=None, dtype=RQ_BF16) == RQ_ERR_DTYPE  # as without a window
    n = C.c_size_t()
    work = _lib.lib().rq_paged_attention_window_work
    for bad, status in ((dict(cache=RQ_F16), RQ_ERR_DTYPE), (dict(window=-1), RQ_ERR_SHAPE), (dict(sinks=-1), RQ_ERR_SHAPE),
                        (dict(batch=-1), RQ_ERR_SHAPE), (dict(n_q=3), RQ_ERR_SHAPE), ({}, RQ_ERR_HANDLE)):
        a = dict(cache=RQ_I8, batch=3, n_q=4, n_kv=2, hd=64, max_len=100, window=0, sinks=0) | bad
        assert work(CTX, *a.values(), C.byref(n)) == status, bad
    assert work(CTX, RQ_I8, 3, 4, 2, 64, 100, 0, 0, None) == RQ_ERR_NULL


def test_append_and_rows_arguments():
    for kw in (dict(rows=-1), dict(batch=-1), dict(rows=2 ** 24), dict(qos=8), dict(kst=120), dict(cu=P + 2),
               dict(past=P + 3), dict(n_q=5)):
        assert append(pages(), **kw) == RQ_ERR_SHAPE, kw
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(qo=None), dict(cu=None), dict(past=None)):
        assert append(pages(), **kw) == RQ_ERR_NULL, kw
    assert append(pages(), ko=None) == RQ_ERR_HANDLE and append(pages(), rows=0, q=None) == RQ_OK
    for kw in (dict(rows=-1), dict(batch=-2), dict(rows=2 ** 24), dict(kos=120), dict(vos=0), dict(cu=P + 1), dict(ko=P + 4)):
        assert rows(pages(), **kw) == RQ_ERR_SHAPE, kw
    for kw in (dict(ko=None), dict(vo=None), dict(cu=None)):
        assert rows(pages(), **kw) == RQ_ERR_NULL, kw
    assert rows(pages(), batch=0, ko=None) == RQ_OK and rows(pages(), rows=0, ko=None) == RQ_OK
    # the old entries take no int8 pages
    L = _lib.lib()
    pg = pages()
    assert L.rq_paged_attention(CTX, C.byref(pg), RQ_F32, P, 256, P, 128, P, 128, P, 3, 4, 100, 1e4, 0.1, P, 256, P, 1 << 40,
                                None) == RQ_ERR_DTYPE
    assert L.rq_pages_append(CTX, C.byref(pg), RQ_F32, P, 256, P, 128, P, 128, P, P, 3, 9, 4, 1e4, P, 256, P, 128,
                             None) == RQ_ERR_DTYPE


def test_python_scales():
    """attention._scales, on CPU tensors that say they are on device 0."""

    class Ctx:
        device = -1  # (get_device() of a CPU tensor)

    pg = pages(pages=6)
    good = torch.zeros(6, 2, 2)
    strided = torch.zeros(6, 9)[:, :4].unflatten(1, (2, 2))
    assert attention._scales(Ctx, pg, good, good)[2] == 4 and attention._scales(Ctx, pg, strided, strided)[2] == 9
    assert attention._scales(Ctx, pages(dtype=RQ_F32), None, None) == (None, None, 0)
    for k, v in ((None, None), (good, None), (good, good.double()), (good[:5], good), (good, good.transpose(1, 2).contiguous().transpose(1, 2)),
                 (good, strided), (torch.zeros(6, 4, 2)[:, ::2], good)):
        with pytest.raises(ValueError):
            attention._scales(Ctx, pg, k, v)
    with pytest.raises(ValueError):
        attention._scales(Ctx, pages(dtype=RQ_F32), good, good)
    one = pages(pages=1, page_size=16, n_kv=1)
    assert attention._scales(Ctx, one, torch.zeros(1, 1, 1), torch.zeros(1, 1, 1))[2] == 1


def test_copies_take_the_scales_along(monkeypatch):
    done = []
    monkeypatch.setattr(paged, "pages_copy", lambda ctx, data, src, dst: done.append((data, src, dst)))
    c = object.__new__(paged.PagedCache)
    c.ctx, c.data = None, "pages"
    c._copy([1], [2])
    c.scales = "scales"
    c._copy([3], [4])
    assert done == [("pages", [1], [2]), ("pages", [3], [4]), ("scales", [3], [4])]
