"""Refusals of the windowed prompt-attention entries, through the C ABI and without a GPU: arguments are checked
before the context, so a bad argument gives its own status and good ones with an unknown context give RQ_ERR_HANDLE."""
import ctypes as C

import pytest
import torch

from raster_amd import _lib, attention
from raster_amd._lib import RQ_BF16, RQ_ERR_HANDLE, RQ_ERR_NULL, RQ_ERR_SHAPE, RQ_OK

CTX = C.c_void_p(0x1234)  # never dereferenced
P = 0x10000  # an aligned address, never dereferenced


def prompt(**kw):
    a = dict(dtype=RQ_BF16, batch=2, rows_q=1000, rows_k=1000, n_q=4, n_kv=2, head_dim=64, cu_q=P, cu_k=None, causal=1,
             scale=0.125)
    a.update(kw)
    return _lib.Prompt(*a.values())


def fwd(p, window, sinks, **kw):
    a = dict(q=P, qs=256, k=P, ks=128, v=P, vs=128, out=P, os=256, lse=None)
    a.update(kw)
    return _lib.lib().rq_prompt_attention_window(CTX, C.byref(p) if p else None, window, sinks, *a.values(), None)


def bwd(p, window, sinks, **kw):
    a = dict(do=P, dos=256, q=P, qs=256, k=P, ks=128, v=P, vs=128, out=P, os=256, lse=P, dq=P, dqs=256, dk=P, dks=128,
             dv=P, dvs=128, work=P, wb=1 << 40)
    a.update(kw)
    return _lib.lib().rq_prompt_attention_window_bwd(CTX, C.byref(p), window, sinks, *a.values(), None)


def work(p, window, sinks):
    n = C.c_size_t()
    status = _lib.lib().rq_prompt_attention_window_bwd_work(C.byref(p), window, sinks, C.byref(n))
    return status, n.value


@pytest.mark.parametrize("call", [fwd, bwd, lambda p, w, z: work(p, w, z)[0]], ids=["fwd", "bwd", "work"])
def test_window_and_sinks(call):
    good = RQ_ERR_HANDLE if call in (fwd, bwd) else RQ_OK
    for w, z in ((0, 0), (1, 0), (64, 4), (0, 9), (2 ** 62, 2 ** 62), (2 ** 63 - 1, 1), (999, 1), (999, 0)):
        assert call(prompt(), w, z) == good, (w, z)
    for w, z in ((-1, 0), (5, -1), (0, -1), (-2 ** 62, 3)):
        assert call(prompt(), w, z) == RQ_ERR_SHAPE, (w, z)
    assert call(prompt(causal=0), 5, 0) == RQ_ERR_SHAPE
    assert "causal" in _lib.lib().rq_last_error().decode()
    assert call(prompt(causal=0), 0, 0) == good
    assert call(prompt(scale=0.0), 5, 0) == RQ_ERR_SHAPE


def test_work_size():
    p = prompt()
    need = work(p, 64, 4)[1]
    assert bwd(p, 64, 4, wb=need) == RQ_ERR_HANDLE and bwd(p, 64, 4, wb=need - 1) == RQ_ERR_SHAPE
    assert bwd(p, 64, 4, work=None) == RQ_ERR_NULL
    # a window that leaves nothing out asks for what the call without one does
    n = C.c_size_t()
    assert _lib.lib().rq_prompt_attention_bwd_work(C.byref(p), C.byref(n)) == RQ_OK
    assert work(p, 996, 4)[1] == n.value == work(p, 0, 0)[1]
    assert _lib.lib().rq_prompt_attention_window_bwd_work(C.byref(p), 5, 0, None) == RQ_ERR_NULL


def test_nothing_to_do():
    assert fwd(prompt(rows_q=0, rows_k=0), 5, 1, q=None) == RQ_OK
    assert bwd(prompt(batch=0), 5, 1, q=None) == RQ_OK


def test_python_arguments():
    for kw in (dict(window=-1), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            attention._window(kw.get("window"), kw.get("sinks", 0))
    assert attention._window(None, 3) == (0, 3) and attention._window(7, 0) == (7, 0)
    assert attention._window(None, 0) == attention._window(0, 0) == ()
    assert attention._window(2 ** 80, 2 ** 90) == (1 << 40, 1 << 40)
    with pytest.raises(ValueError):  # (a CPU tensor is refused before anything is called)
        x = torch.zeros(4, 64)
        attention.prompt_attention(type("C", (), {"device": 0, "handle": None})(), x, x, x,
                                   torch.zeros(2, dtype=torch.int32), 1, 1, 64, 0.1, window=3)


@pytest.mark.parametrize("window,sinks", [(64, 4), (1000, 500)])
def test_work_does_not_grow_with_the_sequences(window, sinks):
    """The sinks' partial sums are of chunks of 256 queries or more, and of at most two for each of so many, whatever the
    sequences: 64 keys' dK and dV in f32, for each 64 sinks and KV head."""
    rows = 400000
    for batch in (1, 7, 1000, 1563, 5000, 100000, 10 ** 7):
        p = prompt(batch=batch, rows_q=rows, rows_k=rows, n_q=16, n_kv=16, head_dim=128)
        more = work(p, window, sinks)[1] - work(p, window, 0)[1]
        assert more <= (rows // 128 + 1) * -(-sinks // 64) * 16 * 2 * 64 * 128 * 4, batch


@pytest.mark.parametrize("sinks", [0, 4, 500])
def test_many_sequences_with_sinks_are_taken(sinks):
    """Launches of fewer than 2^24 workgroups for 100000 sequences, with sinks as without."""
    for batch in (1, 1000, 100000):
        p = prompt(batch=batch, rows_q=400000, rows_k=400000, n_q=16, n_kv=16, head_dim=128)
        assert bwd(p, 64, sinks, **{s: 2048 for s in ("dos", "qs", "ks", "vs", "os", "dqs", "dks", "dvs")}) == RQ_ERR_HANDLE
