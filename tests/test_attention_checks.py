"""Refusals of the prompt-attention and paged-cache entries, through the C ABI and
without a GPU: arguments are checked before the context, so a bad argument gives its
own status and good ones with an unknown context give RQ_ERR_HANDLE. Nothing is run."""
import ctypes as C

import pytest

from raster_amd import _lib
from raster_amd._lib import RQ_BF16, RQ_ERR_DTYPE, RQ_ERR_HANDLE, RQ_ERR_NULL, RQ_ERR_SHAPE, RQ_F16, RQ_F32, RQ_OK

CTX = C.c_void_p(0x1234)  # never dereferenced
P = 0x10000  # an aligned address, never dereferenced


def prompt(**kw):
    a = dict(dtype=RQ_BF16, batch=2, rows_q=10, rows_k=10, n_q=4, n_kv=2, head_dim=64, cu_q=P, cu_k=None, causal=1,
             scale=0.125)
    a.update(kw)
    return _lib.Prompt(*a.values())


def fwd(p, **kw):
    a = dict(q=P, qs=256, k=P, ks=128, v=P, vs=128, out=P, os=256, lse=None)
    a.update(kw)
    return _lib.lib().rq_prompt_attention(CTX, C.byref(p) if p else None, *a.values(), None)


def test_prompt_attention():
    assert fwd(prompt()) == RQ_ERR_HANDLE and fwd(prompt(), lse=P) == RQ_ERR_HANDLE
    assert fwd(prompt(cu_k=P, rows_k=99)) == RQ_ERR_HANDLE
    assert fwd(None) == RQ_ERR_NULL
    for kw in (dict(dtype=RQ_F16), dict(dtype=7)):
        assert fwd(prompt(**kw)) == RQ_ERR_DTYPE
    for kw in (dict(n_q=3), dict(n_q=0), dict(n_kv=0), dict(n_kv=-2), dict(head_dim=0), dict(head_dim=60),
               dict(head_dim=264), dict(batch=-1), dict(rows_q=-1), dict(rows_k=-1), dict(rows_k=11),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(rows_q=2 ** 31, rows_k=2 ** 31), dict(batch=2 ** 31), dict(n_q=65536, n_kv=1)):
        assert fwd(prompt(**kw)) == RQ_ERR_SHAPE, kw
    assert fwd(prompt(cu_q=None)) == RQ_ERR_NULL
    for name in ("q", "k", "v", "out"):
        assert fwd(prompt(), **{name: None}) == RQ_ERR_NULL
        assert fwd(prompt(), **{name: P + 8}) == RQ_ERR_SHAPE
        assert name in _lib.lib().rq_last_error().decode()
    for kw in (dict(qs=255), dict(qs=260), dict(ks=120), dict(vs=2 ** 22 + 8), dict(os=0), dict(os=-256)):
        assert fwd(prompt(), **kw) == RQ_ERR_SHAPE, kw
    assert fwd(prompt(), lse=P + 2) == RQ_ERR_SHAPE
    # nothing to do: no pointer is asked for
    assert fwd(prompt(rows_q=0, rows_k=0), q=None, k=None, v=None, out=None) == RQ_OK
    assert fwd(prompt(batch=0), q=None) == RQ_OK
    assert fwd(prompt(rows_k=0, cu_k=P), k=None, v=None) == RQ_ERR_HANDLE  # no keys: zeros are written


def bwd(p, **kw):
    a = dict(do=P, dos=256, q=P, qs=256, k=P, ks=128, v=P, vs=128, out=P, os=256, lse=P, dq=P, dqs=256, dk=P, dks=128,
             dv=P, dvs=128, work=P, wb=1 << 20)
    a.update(kw)
    return _lib.lib().rq_prompt_attention_bwd(CTX, C.byref(p), *a.values(), None)


def test_prompt_attention_bwd():
    assert bwd(prompt()) == RQ_ERR_HANDLE
    for name in ("do", "q", "k", "v", "out", "dq", "dk", "dv", "lse", "work"):
        assert bwd(prompt(), **{name: None}) == RQ_ERR_NULL, name
        assert bwd(prompt(), **{name: P + (2 if name == "lse" else 8)}) == RQ_ERR_SHAPE, name
    for name in ("dos", "qs", "ks", "vs", "os", "dqs", "dks", "dvs"):
        assert bwd(prompt(), **{name: 64}) == RQ_ERR_SHAPE, name
    assert bwd(prompt(scale=0.0)) == RQ_ERR_SHAPE
    n = C.c_size_t()
    p = prompt()
    assert _lib.lib().rq_prompt_attention_bwd_work(C.byref(p), C.byref(n)) == RQ_OK and n.value >= 160
    assert bwd(prompt(), wb=n.value - 1) == RQ_ERR_SHAPE and bwd(prompt(), wb=n.value) == RQ_ERR_HANDLE
    assert _lib.lib().rq_prompt_attention_bwd_work(C.byref(p), None) == RQ_ERR_NULL
    assert _lib.lib().rq_prompt_attention_bwd_work(None, C.byref(n)) == RQ_ERR_NULL


def pages(**kw):
    a = dict(dtype=RQ_BF16, kpages=P, vpages=P, pages=8, page_size=16, n_kv=2, head_dim=64, table=P, table_stride=4)
    a.update(kw)
    return _lib.Pages(*a.values())


def paged(g, **kw):
    a = dict(dtype=RQ_BF16, q=P, qs=256, k=P, ks=128, v=P, vs=128, lens=P, batch=2, n_q=4, max_len=64, theta=1e4,
             scale=0.125, out=P, os=256, work=P, wb=1 << 20)
    a.update(kw)
    return _lib.lib().rq_paged_attention(CTX, C.byref(g) if g else None, *a.values(), None)


def append(g, **kw):
    a = dict(dtype=RQ_BF16, q=P, qs=256, k=P, ks=128, v=P, vs=128, cu=P, past=P, batch=2, rows=5, n_q=4, theta=1e4,
             qo=P, qos=256, ko=P, kos=128)
    a.update(kw)
    return _lib.lib().rq_pages_append(CTX, C.byref(g) if g else None, *a.values(), None)


@pytest.mark.parametrize("call", [paged, append])
def test_paged_entries(call):
    assert call(pages()) == RQ_ERR_HANDLE and call(pages(), theta=0.0) == RQ_ERR_HANDLE
    assert call(pages(), dtype=RQ_F32) == RQ_ERR_HANDLE and call(pages(dtype=RQ_F32), dtype=RQ_F32) == RQ_ERR_HANDLE
    assert call(None) == RQ_ERR_NULL
    assert call(pages(dtype=RQ_F32)) == RQ_ERR_DTYPE and call(pages(dtype=RQ_F16)) == RQ_ERR_DTYPE
    assert call(pages(), dtype=RQ_F16) == RQ_ERR_DTYPE
    for kw in (dict(page_size=8), dict(page_size=24), dict(page_size=0), dict(page_size=1 << 17), dict(pages=0),
               dict(pages=2 ** 31), dict(table_stride=-1), dict(n_kv=3), dict(head_dim=12), dict(head_dim=512)):
        assert call(pages(**kw)) == RQ_ERR_SHAPE, kw
    for kw in (dict(kpages=None), dict(vpages=None), dict(table=None)):
        assert call(pages(**kw)) == RQ_ERR_NULL, kw
    for kw in (dict(kpages=P + 4), dict(vpages=P + 8), dict(table=P + 1)):
        assert call(pages(**kw)) == RQ_ERR_SHAPE, kw
    for kw in (dict(q=None), dict(qs=64), dict(q=P + 2), dict(batch=-1), dict(theta=-1.0), dict(theta=float("nan")),
               dict(n_q=5)):
        assert call(pages(), **kw) in (RQ_ERR_SHAPE, RQ_ERR_NULL), kw
    assert call(pages(), batch=0) == RQ_OK and call(pages(table=None), batch=0) == RQ_OK
    assert call(pages(table=None, table_stride=0)) == RQ_ERR_HANDLE  # no row has a page


def test_paged_attention_only():
    assert paged(pages(), k=None, v=None) == RQ_ERR_HANDLE
    assert paged(pages(), k=None) == RQ_ERR_NULL and paged(pages(), v=None) == RQ_ERR_NULL
    assert paged(pages(), lens=None) == RQ_ERR_NULL and paged(pages(), out=None) == RQ_ERR_NULL
    for kw in (dict(scale=0.0), dict(scale=float("nan")), dict(max_len=-1), dict(max_len=2 ** 31), dict(os=8),
               dict(lens=P + 1)):
        assert paged(pages(), **kw) == RQ_ERR_SHAPE, kw
    n = C.c_size_t()
    L = _lib.lib()
    assert L.rq_paged_attention_work(CTX, 2, 4, 2, 64, 64, C.byref(n)) == RQ_ERR_HANDLE
    assert L.rq_paged_attention_work(CTX, 2, 4, 3, 64, 64, C.byref(n)) == RQ_ERR_SHAPE
    assert L.rq_paged_attention_work(CTX, 2, 4, 2, 64, 64, None) == RQ_ERR_NULL


def test_append_only():
    assert append(pages(), ko=None) == RQ_ERR_HANDLE and append(pages(), rows=0, q=None) == RQ_OK
    for kw in (dict(cu=None), dict(past=None), dict(qo=None), dict(k=None), dict(v=None)):
        assert append(pages(), **kw) == RQ_ERR_NULL, kw
    for kw in (dict(rows=-1), dict(qos=8), dict(kos=8), dict(ko=P + 4)):
        assert append(pages(), **kw) == RQ_ERR_SHAPE, kw


def copy(src, dst, **kw):
    a = dict(base=P, planes=2, plane_bytes=8 * 64, pages=8, page_bytes=64)
    a.update(kw)
    arr = C.c_int32 * max(1, len(src))
    n = a.pop("n", len(src))
    return _lib.lib().rq_pages_copy(CTX, *a.values(), a.pop("s", arr(*src)), arr(*dst), n, None)


def test_pages_copy():
    assert copy([0, 1], [2, 3]) == RQ_ERR_HANDLE and copy([0, 0], [2, 3]) == RQ_ERR_HANDLE
    for src, dst in (([0], [8]), ([0], [-1]), ([8], [0]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]),
                     ([3], [3]), (list(range(9)), list(range(9)))):
        assert copy(src, dst) == RQ_ERR_SHAPE, (src, dst)
    for kw in (dict(page_bytes=24), dict(page_bytes=0), dict(plane_bytes=8 * 64 - 16), dict(plane_bytes=8 * 64 + 4),
               dict(pages=0), dict(pages=9), dict(planes=-1), dict(n=-1), dict(base=P + 8)):
        assert copy([0], [2], **kw) == RQ_ERR_SHAPE, kw
    assert copy([0], [2], base=None) == RQ_ERR_NULL
    assert copy([], []) == RQ_OK and copy([0], [2], planes=0) == RQ_OK


def test_launches_of_2_32_threads_are_refused():
    """HIP takes fewer than 2^32 threads a launch: RQ_ERR_SHAPE before it is asked."""
    def said(status):
        return status == RQ_ERR_SHAPE and "one launch" in _lib.lib().rq_last_error().decode()

    assert said(fwd(prompt(rows_q=2 ** 28, rows_k=2 ** 28)))  # 4 heads x (2^23 + 2) tiles of 32
    assert fwd(prompt(rows_q=2 ** 26, rows_k=2 ** 26)) == RQ_ERR_HANDLE
    assert fwd(prompt(rows_k=2 ** 30, cu_k=P)) == RQ_ERR_HANDLE  # keys take no workgroup
    assert said(fwd(prompt(batch=2 ** 24)))
    assert said(bwd(prompt(rows_q=2 ** 26, rows_k=2 ** 26), wb=2 ** 40))  # 16 threads a row and head
    assert said(bwd(prompt(rows_q=2 ** 25, rows_k=2 ** 30, cu_k=P), wb=2 ** 40))  # 2^24 tiles of 64 keys x 2 heads
    assert bwd(prompt(rows_q=2 ** 25, rows_k=2 ** 25), wb=2 ** 40) == RQ_ERR_HANDLE
    # 12 parts of the keys' gradient: slots count for each of them
    assert said(bwd(prompt(batch=2 ** 20, rows_q=2 ** 25, rows_k=64, n_q=8, n_kv=1, cu_k=P), qs=512, dos=512, os=512,
                    dqs=512, wb=2 ** 40))
    assert said(append(pages(), rows=2 ** 24)) and append(pages(), rows=2 ** 24 - 1) == RQ_ERR_HANDLE
    big = dict(plane_bytes=2 ** 33, pages=8, page_bytes=2 ** 30)
    assert said(copy([0], [2], planes=256, **big)) and copy([0], [2], planes=255, **big) == RQ_ERR_HANDLE


def test_paged_sizes_whose_products_overflow():
    """Batch times heads past one launch is refused before anything is planned with it: max_len times the groups
    would not fit 64 bits, and the bytes asked for would be anything."""
    n, L = C.c_size_t(), _lib.lib()

    def work(batch, n_q, n_kv, max_len):
        return L.rq_paged_attention_work(CTX, batch, n_q, n_kv, 64, max_len, C.byref(n))

    for a in ((2 ** 30, 65535, 65535, 2 ** 30), (2 ** 30, 16, 1, 2 ** 30), (2 ** 24, 1, 1, 16), (2 ** 20, 32, 1, 16)):
        assert work(*a) == RQ_ERR_SHAPE and "one launch" in L.rq_last_error().decode(), a
    assert work(2 ** 24 - 1, 1, 1, 2 ** 30) == RQ_ERR_HANDLE
    wide = dict(q=P, qs=65528 * 64, os=65528 * 64, n_q=65528)
    assert paged(pages(n_kv=1), batch=2 ** 30, max_len=2 ** 30, **wide) == RQ_ERR_SHAPE
    assert paged(pages(n_kv=1), batch=255, ks=64, vs=64, **wide) == RQ_ERR_HANDLE
