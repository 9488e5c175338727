"""Attention over prompts with a sliding window and sinks, and its gradient, against every head in 64 bits
(attn_ref.py states the tolerances: rounding counts, elementwise)."""
import ctypes as C

import pytest

from raster_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t

    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


@pytest.fixture(scope="module")
def ctx(torch):
    import raster_amd

    c = raster_amd.Context(0)
    yield c
    c.close()


def cu_of(torch, lens, start=0):
    return torch.tensor([start + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def rows(torch, g, n, width, dtype, pad=0):
    return torch.randn((n, width + pad), generator=g, device="cuda").to(dtype)[:, :width]


def heads(t, h, hd):
    return t[:, h * hd:(h + 1) * hd].double()


def seen(torch, a, b, window, sinks):
    at, j = torch.arange(a, device="cuda")[:, None] + b - a, torch.arange(b, device="cuda")
    return (j <= at) & ((at - j < window) | (j < sinks))


def check_forward(torch, q, k, v, out, lse, lq, lk, nq, nkv, hd, scale, window, sinks, start=0):
    import attn_ref as ref

    half = ref.HALF[q.dtype]
    a0 = b0 = start
    for a, b in zip(lq, lk):
        see = seen(torch, a, b, window, sinks)
        for h in range(nq):
            j = h // (nq // nkv)
            want, wlse, bound = ref.attend(heads(q[a0:a0 + a], h, hd), heads(k[b0:b0 + b], j, hd),
                                           heads(v[b0:b0 + b], j, hd), scale, see, half)
            got = heads(out[a0:a0 + a], h, hd)
            assert bool(((got - want).abs() <= bound).all()), (a, b, h, float(((got - want).abs() / bound).max()))
            if lse is not None:
                gl = lse[h, a0:a0 + a].double()
                dead = ~see.any(1)
                assert bool((gl[dead] == -torch.inf).all())
                assert bool(((gl - wlse)[~dead].abs() <= 1e-5 * (1 + wlse[~dead].abs())).all())
        a0, b0 = a0 + a, b0 + b


def check_gradient(torch, q, k, v, do, grads, lq, lk, nq, nkv, hd, scale, window, sinks):
    import attn_ref as ref

    dq, dk, dv = grads
    a0 = b0 = 0
    for a, b in zip(lq, lk):
        see = seen(torch, a, b, window, sinks)
        for j in range(nkv):
            kj, vj = heads(k[b0:b0 + b], j, hd), heads(v[b0:b0 + b], j, hd)
            wk, wv, bk, bv = (torch.zeros((b, hd), dtype=torch.float64, device="cuda") for _ in range(4))
            for h in range(j * (nq // nkv), (j + 1) * (nq // nkv)):
                (wq, dkh, dvh), (bq, bkh, bvh) = ref.attend_grad(
                    heads(q[a0:a0 + a], h, hd), kj, vj, heads(do[a0:a0 + a], h, hd), scale, see, ref.HALF[q.dtype])
                assert bool(((heads(dq[a0:a0 + a], h, hd) - wq).abs() <= bq).all()), (a, b, h, "dq")
                wk, wv, bk, bv = wk + dkh, wv + dvh, bk + bkh, bv + bvh
            assert bool(((heads(dk[b0:b0 + b], j, hd) - wk).abs() <= bk).all()), (a, b, j, "dk")
            assert bool(((heads(dv[b0:b0 + b], j, hd) - wv).abs() <= bv).all()), (a, b, j, "dv")
        a0, b0 = a0 + a, b0 + b


# type, heads, KV heads, head_dim, queries and keys of each sequence
CASES = [
    ("bf16", 4, 2, 128, [37, 1], [37, 1]),
    ("bf16", 8, 2, 128, [128, 1, 0, 129, 333], [128, 1, 0, 129, 333]),
    ("bf16", 8, 1, 64, [65, 200, 31], [65, 200, 31]),
    ("bf16", 3, 3, 80, [90, 17], [90, 17]),
    ("bf16", 2, 1, 200, [161], [161]),
    ("bf16", 2, 2, 128, [5, 64, 100], [300, 64, 40]),      # the end of a sequence; more queries than keys
    ("bf16", 2, 2, 128, [40, 0, 7], [0, 50, 3]),           # no keys, no queries
    ("bf16", 64, 8, 128, [300, 129, 90, 5], [300, 129, 90, 5]),  # grids that fill the CUs
    ("bf16", 96, 8, 128, [300, 129, 90, 5], [300, 129, 90, 5]),
    ("bf16", 128, 8, 64, [300, 129, 90], [300, 129, 90]),
    ("bf16", 16, 4, 256, [200, 70], [200, 70]),
    ("bf16", 128, 8, 200, [300, 0, 90], [310, 129, 90]),
    ("f32", 4, 2, 128, [33, 0, 130], [33, 0, 130]),
    ("f32", 6, 2, 64, [65, 200], [65, 200]),
    ("f32", 3, 3, 40, [77], [77]),
    ("f32", 2, 1, 256, [170, 9], [170, 9]),
    ("f32", 2, 2, 128, [5, 64, 100], [300, 64, 40]),
    ("bf16", 4, 2, 128, [700], [700]),
    ("bf16", 4, 2, 48, [700, 33], [700, 33]),
    ("f32", 128, 8, 40, [300, 129, 90], [300, 129, 90]),
    ("f32", 32, 8, 64, [300, 129, 90], [300, 129, 90]),
    ("f32", 64, 8, 128, [300, 129, 90], [300, 129, 90]),
    ("f32", 128, 8, 104, [300, 0, 90], [310, 129, 90]),
]
WINDOWS = [(1, 0), (7, 3), (32, 0), (33, 1), (64, 4), (100, 70), (250, 4), (300, 4)]


def data(torch, t, nq, nkv, hd, lq, lk, seed):
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[t]
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [rows(torch, g, sum(n), w * hd, dt, pad=8) for n, w in ((lq, nq), (lk, nkv), (lk, nkv), (lq, nq))]


@pytest.mark.parametrize("t,nq,nkv,hd,lq,lk", CASES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_window(torch, ctx, t, nq, nkv, hd, lq, lk, window, sinks):
    import raster_amd

    print(f"[gpu] window {t} {nq}/{nkv}x{hd} {lq} {lk} {window}+{sinks}", flush=True)
    q, k, v, do = data(torch, t, nq, nkv, hd, lq, lk, hd + sum(lq) + window)
    cu, cu_k, scale = cu_of(torch, lq), None if lq == lk else cu_of(torch, lk), hd ** -0.5
    lse = torch.empty((nq, sum(lq)), device="cuda")
    see = dict(window=window, sinks=sinks, cu_k=cu_k)
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, **see)
    check_forward(torch, q, k, v, out, lse, lq, lk, nq, nkv, hd, scale, window, sinks)
    grads = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, **see)
    check_gradient(torch, q, k, v, do, grads, lq, lk, nq, nkv, hd, scale, window, sinks)


def tile(ctx, t, nq, nkv, hd, lq, lk, window, sinks):
    p = _lib.Prompt({"f32": _lib.RQ_F32, "bf16": _lib.RQ_BF16}[t], len(lq), sum(lq), sum(lk), nq, nkv, hd, 0x10000,
                    0x10000, 1, 0.125)
    n = C.c_int(-1)
    _lib.call("rq_prompt_attention_window_tile", ctx.handle, C.byref(p), window, sinks, C.byref(n))
    return n.value


# bf16, more than 4096 queries a sequence
LONG = [
    (8, 2, 128, [4600], [4600], 300, 4),
    (6, 3, 72, [5000, 4000], [5000, 4700], 1111, 0),
    (4, 4, 128, [8300, 1, 4100], [8300, 1, 4100], 2049, 130),
    (4, 2, 104, [9000, 0], [8200, 77], 64, 1),      # more queries than keys
    (4, 4, 128, [4200], [9000], 4096, 4),
    (4, 4, 128, [4999], [0], 16, 1),
    (4, 2, 128, [6000], [6000], 1, 0),
    (6, 2, 128, [12500], [12500], 8192, 3),         # the kernel of 256 queries
    (6, 6, 72, [6100, 5000], [15000, 5000], 8200, 70),
]


@pytest.mark.parametrize("nq,nkv,hd,lq,lk,window,sinks", LONG)
def test_long_sequences(torch, ctx, nq, nkv, hd, lq, lk, window, sinks):
    import raster_amd

    print(f"[gpu] window long {nq}/{nkv}x{hd} {lq} {lk} {window}+{sinks}", flush=True)
    if window >= 8192:
        assert tile(ctx, "bf16", nq, nkv, hd, lq, lk, window, sinks) == 256
    q, k, v, do = data(torch, "bf16", nq, nkv, hd, lq, lk, sum(lq))
    cu, cu_k, scale = cu_of(torch, lq), None if lq == lk else cu_of(torch, lk), hd ** -0.5
    lse = torch.empty((nq, sum(lq)), device="cuda")
    see = dict(window=window, sinks=sinks, cu_k=cu_k)
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, **see)
    check_forward(torch, q, k, v, out, lse, lq, lk, nq, nkv, hd, scale, window, sinks)
    grads = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, **see)
    check_gradient(torch, q, k, v, do, grads, lq, lk, nq, nkv, hd, scale, window, sinks)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("lens,window,sinks", [([300, 129], 300, 0), ([300, 129], 200, 229), ([50], 10 ** 15, 4)])
def test_a_window_of_everything_is_none(torch, ctx, t, lens, window, sinks):
    """The same bits as without a window, from the same kernel where the sizes alone say so."""
    import raster_amd

    nq, nkv, hd = 4, 2, 128
    print(f"[gpu] window of everything {t} {lens} {window}+{sinks}", flush=True)
    q, k, v, do = data(torch, t, nq, nkv, hd, lens, lens, 3)
    cu, scale, got = cu_of(torch, lens), hd ** -0.5, []
    for see in ({}, dict(window=window, sinks=sinks), dict(window=0, sinks=sinks), dict(window=None)):
        lse = torch.empty((nq, sum(lens)), device="cuda")
        out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, **see)
        got.append([out, lse, *raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale,
                                                               **see)])
    for g in got[2:]:
        assert all(torch.equal(a, b) for a, b in zip(g, got[0]))
    if window + sinks >= sum(lens):
        assert all(torch.equal(a, b) for a, b in zip(got[1], got[0]))
    else:  # all of every sequence, which only the device knows: the other kernel, sums in the same order
        for a, b in zip(got[1], got[0]):
            assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.float().abs().max())


def test_gradient_against_differences(torch, ctx):
    """The derivative along a direction from two forward calls: sum of dout . out at
    +e and -e, f32, relative to the gradient's own product with the direction. The
    difference errs by e^2 of its third derivative (order 1) and by out's rounding over
    e, 1e-6 / e of the magnitude: 1e-3 at e = 1e-2."""
    import raster_amd

    nq, nkv, hd, lens, see = 4, 2, 64, [150, 3, 70], dict(window=20, sinks=2)
    print("[gpu] window gradient against differences", flush=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    n = sum(lens)
    q, do, uq = (torch.randn((n, nq * hd), generator=g, device="cuda") for _ in range(3))
    k, v, uk, uv = (torch.randn((n, nkv * hd), generator=g, device="cuda") for _ in range(4))
    cu, scale, lse = cu_of(torch, lens), hd ** -0.5, torch.empty((nq, n), device="cuda")

    def f(e):
        return float((raster_amd.prompt_attention(ctx, q + e * uq, k + e * uk, v + e * uv, cu, nq, nkv, hd, scale, **see)
                      .double() * do.double()).sum())

    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, **see)
    grads = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, **see)
    want = sum(float((a.double() * b.double()).sum()) for a, b in zip(grads, (uq, uk, uv)))
    size = sum(float((a.double() * b.double()).norm()) for a, b in zip(grads, (uq, uk, uv)))
    got = (f(1e-2) - f(-1e-2)) / 2e-2
    assert abs(got - want) <= 1e-3 * max(abs(want), size)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("n,window,sinks", [(700, 64, 4), (5000, 200, 1)])
def test_nan_far_outside_the_window(torch, ctx, t, n, window, sinks):
    """Keys and values of NaN reach no query that sees none of them and is 95 keys or more away from seeing one;
    queries and gradients of NaN no key as far from them."""
    import raster_amd

    nq, nkv, hd = 2, 1, 128
    print(f"[gpu] window NaN {t} {n}", flush=True)
    q, k, v, do = (x.clone() for x in data(torch, t, nq, nkv, hd, [n], [n], 8))
    cu, scale = cu_of(torch, [n]), hd ** -0.5

    def both():
        lse = torch.empty((nq, n), device="cuda")
        out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, window=window, sinks=sinks)
        return [out, *raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, window=window,
                                                      sinks=sinks)]

    clean = both()
    at = n // 2
    k[at], v[at] = float("nan"), float("inf")
    dirty = both()
    far = torch.ones(n, dtype=torch.bool, device="cuda")
    far[at - 94:at + window + 95] = False
    assert bool(torch.isnan(dirty[0][at:at + window]).all())
    assert torch.equal(clean[0][far], dirty[0][far]) and torch.equal(clean[1][far], dirty[1][far])


def test_rows_of_no_sequence_and_graphs(torch, ctx):
    """Rows before the first and behind the last sequence hold NaN and stay as they were; a captured forward and
    gradient, replayed with eager work between, give the eager bits."""
    import raster_amd

    nq, nkv, hd, lens, first, n = 8, 2, 128, [70, 0, 445], 3, 540
    see = dict(window=50, sinks=4)
    print("[gpu] window rows of no sequence, graphs", flush=True)
    mid = slice(first, first + sum(lens))
    for dt in ("bf16", "f32"):
        q, k, v, do = (x.clone() for x in data(torch, dt, nq, nkv, hd, [n], [n], 12))
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        keep[mid] = False
        for x in (q, k, v, do):
            x[keep] = float("nan")
        cu, scale = cu_of(torch, lens, first), hd ** -0.5
        out, lse = torch.full_like(q, 7.0), torch.full((nq, n), 7.0, device="cuda")
        grads = [torch.full_like(x, 7.0) for x in (q, k, v)]

        def call():
            raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, out=out, lse=lse, **see)
            raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, dq=grads[0],
                                            dk=grads[1], dv=grads[2], **see)

        call()
        check_forward(torch, q, k, v, out, lse, lens, lens, nq, nkv, hd, scale, 50, 4, start=first)
        for x in (out, *grads):
            assert bool((x[keep] == 7).all())
        assert bool((lse[:, keep] == 7).all())
        want = [x.clone() for x in (out, lse, *grads)]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call()
        for _ in range(3):
            for x in (out, lse, *grads):
                x[mid] = 5.0 if x is not lse else x[mid]
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip((out, lse, *grads), want))


@pytest.mark.parametrize("t,nq,nkv,hd,lens,window,sinks", [
    ("bf16", 16, 8, 64, [2100, 3, 1300, 0, 777], 100, 4),
    ("bf16", 8, 8, 128, [2500, 900], 256, 130),   # three tiles of sinks, the second sequence's window among them
    ("bf16", 8, 8, 200, [2600, 640], 300, 1),
    ("f32", 16, 8, 64, [2100, 30, 1500], 64, 64),
    ("f32", 8, 8, 104, [3000, 200], 70, 500),
    ("f32", 8, 8, 136, [3000, 100], 1, 2),
])
def test_gradient_of_sinks_by_chunks(torch, ctx, t, nq, nkv, hd, lens, window, sinks):
    """Grids thick enough that the first keys' gradients are summed by chunks of queries (the call asks for room for
    them); queries that are the end of longer sequences; the same bits on every run."""
    import raster_amd

    print(f"[gpu] window sinks by chunks {t} {nq}/{nkv}x{hd} {lens} {window}+{sinks}", flush=True)
    for lk in (lens, [n + 37 if n else 50 for n in lens]):
        def room(z):
            p = _lib.Prompt({"f32": _lib.RQ_F32, "bf16": _lib.RQ_BF16}[t], len(lens), sum(lens), sum(lk), nq, nkv, hd,
                            0x10000, 0x10000, 1, 0.125)
            n = C.c_size_t()
            _lib.call("rq_prompt_attention_window_bwd_work", C.byref(p), window, z, C.byref(n))
            return n.value

        assert room(sinks) > room(0)
        q, k, v, do = data(torch, t, nq, nkv, hd, lens, lk, sum(lens))
        cu, cu_k, scale = cu_of(torch, lens), None if lens == lk else cu_of(torch, lk), hd ** -0.5
        lse = torch.empty((nq, sum(lens)), device="cuda")
        see = dict(window=window, sinks=sinks, cu_k=cu_k)
        out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, **see)
        grads = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, **see)
        check_gradient(torch, q, k, v, do, grads, lens, lk, nq, nkv, hd, scale, window, sinks)
        again = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, **see)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_every_kernel_has_a_case(ctx):
    """The tiles that the cases here reach, by type and padded head size."""
    seen = {(t, 64 if hd <= 64 else 128 if hd <= 128 else 256, tile(ctx, t, nq, nkv, hd, lq, lk, w, z))
            for t, nq, nkv, hd, lq, lk in CASES for w, z in WINDOWS}
    seen |= {("bf16", 64 if hd <= 64 else 128, tile(ctx, "bf16", nq, nkv, hd, lq, lk, w, z))
             for nq, nkv, hd, lq, lk, w, z in LONG}
    want = {(t, w, n) for t in ("f32", "bf16") for w in (64, 128) for n in (32, 64, 128)}
    want |= {("bf16", 256, 64), ("bf16", 256, 128), ("f32", 256, 128), ("bf16", 128, 256)}
    assert want <= seen, want - seen


@pytest.mark.parametrize("t,nq,n,window,sinks", [(t, *c) for t in ("bf16", "f32") for c in (
    (2, 1500, 64, 4), (16, 1500, 64, 4), (2, 5000, 200, 1), (16, 5000, 200, 70))] + [("bf16", 6, 12500, 8192, 2)])
def test_nan_behind_the_sinks(torch, ctx, t, nq, n, window, sinks):
    """Keys and values of NaN in the sinks' own tile, but no sinks, reach no query whose window begins 320 rows after them;
    a query and a gradient of NaN reach the sinks and their window's keys, and no other 95 rows from those."""
    import raster_amd

    nkv, hd, at = nq // 2, 128, sinks + 7
    print(f"[gpu] window NaN behind the sinks {t} {nq} heads {n}", flush=True)
    q, k, v, do = (x.clone() for x in data(torch, t, nq, nkv, hd, [n], [n], 8))
    cu, scale = cu_of(torch, [n]), hd ** -0.5

    def both():
        lse = torch.empty((nq, n), device="cuda")
        out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, window=window, sinks=sinks)
        return [out, *raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, window=window,
                                                      sinks=sinks)]

    clean, kept = both(), (k[at].clone(), v[at].clone())
    k[at], v[at] = float("nan"), float("inf")
    dirty = both()
    far = at + window + 320
    assert bool(torch.isnan(dirty[0][at:at + window]).all())
    for a, b in zip(clean[:2], dirty[:2]):
        assert torch.equal(a[:at - 94], b[:at - 94]) if at > 94 else True
        assert torch.equal(a[far:], b[far:])
    k[at], v[at] = kept
    last = n - 10
    q[last], do[last] = float("nan"), float("inf")
    dirty = both()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[:sinks] = False
    keep[max(0, last - window + 1 - 94):] = False
    for a, b in zip(clean[2:], dirty[2:]):
        assert bool(torch.isnan(b[:sinks]).all()) and torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("hd", [64, 128, 200])
@pytest.mark.parametrize("window,sinks,lq,lk", [
    (2, 0, [700, 90], [700, 90]),
    (4, 1, [300, 65, 1000], [300, 65, 1000]),
    (8, 0, [600, 0, 5], [600, 30, 5]),
    (16, 16, [500], [500]),
    (60, 4, [333, 200], [333, 200]),
    (1, 63, [400], [400]),
    (20, 5, [100, 300, 40], [700, 200, 0]),  # the end of a sequence; more queries than keys; no keys
])
def test_gradient_of_few_keys(torch, ctx, hd, window, sinks, lq, lk):
    """bf16, no query sees more than 64 keys: dout . out is formed from the weights, not from the rounded out.

    Elementwise, with U = 2^-24 and H = 2^-8: a weight p is off by d p (attn_ref.py: scores and log-sum-exp), dout . V_j by
    hd U of its magnitudes (e), D = sum p_j (dout . V_j) by sum p_j (d |dout . V_j| + e) and 64 + 4 roundings of its terms.
    dS = p (dout . V_j - D) by d |dS|, p times the errors of both and of their difference, and as an operand by H and 2^-16
    (weights are handed over in 24 bits)."""
    import attn_ref as ref
    import raster_amd

    nq, nkv, scale = 4, 2, hd ** -0.5
    print(f"[gpu] window gradient of few keys x{hd} {lq} {lk} {window}+{sinks}", flush=True)
    q, k, v, do = data(torch, "bf16", nq, nkv, hd, lq, lk, hd + sum(lq) + window)
    cu, cu_k = cu_of(torch, lq), None if lq == lk else cu_of(torch, lk)
    lse = torch.empty((nq, sum(lq)), device="cuda")
    see = dict(window=window, sinks=sinks, cu_k=cu_k)
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, **see)
    dq, dk, _ = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, **see)
    U, H = 2.0 ** -24, 2.0 ** -8
    a0 = b0 = 0
    for a, b in zip(lq, lk):
        see = seen(torch, a, b, window, sinks)
        for j in range(nkv):
            kj, vj = heads(k[b0:b0 + b], j, hd), heads(v[b0:b0 + b], j, hd)
            wk, bk = (torch.zeros((b, hd), dtype=torch.float64, device="cuda") for _ in range(2))
            for h in range(j * (nq // nkv), (j + 1) * (nq // nkv)):
                qh, dh = heads(q[a0:a0 + a], h, hd), heads(do[a0:a0 + a], h, hd)
                x = (qh @ kj.T * scale).masked_fill(~see, -torch.inf)
                p = torch.where(see, torch.exp(x - torch.logsumexp(x, 1)[:, None].clamp(min=-1e300)), 0.0)
                dp, e = dh @ vj.T, hd * U * (dh.abs() @ vj.abs().T)
                delta = (p * dp).sum(1, keepdim=True)
                ds = p * (dp - delta)
                mag = (qh.abs() @ kj.abs().T * scale).masked_fill(~see, 0.0)
                d = 2 * (hd + 4) * U * ref._largest(mag) + 8 * U
                edelta = (p * ((d + 68 * U) * dp.abs() + e)).sum(1, keepdim=True)
                eds = (H + 2.0 ** -15 + d + U) * ds.abs() + p * (edelta + e)
                adds = (max(a, b) + 4) * U
                bq = H * (ds @ kj * scale).abs() + (eds + adds * ds.abs()) @ kj.abs() * scale + 1e-30
                off = (heads(dq[a0:a0 + a], h, hd) - ds @ kj * scale).abs()
                assert bool((off <= bq).all()), (a, b, h, "dq", float((off / bq).max()))
                wk += ds.T @ qh * scale
                bk += (eds + adds * ds.abs()).T @ qh.abs() * scale
            bk += H * wk.abs() + 1e-30
            off = (heads(dk[b0:b0 + b], j, hd) - wk).abs()
            assert bool((off <= bk).all()), (a, b, j, "dk", float((off / bk).max()))
        a0, b0 = a0 + a, b0 + b


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(3, 0), (40, 2), (1, 63)])
def test_nan_around_few_keys(torch, ctx, t, window, sinks):
    """As above where no query sees more than 64 keys."""
    test_nan_far_outside_the_window(torch, ctx, t, 700, window, sinks)
    if sinks:
        test_nan_behind_the_sinks(torch, ctx, t, 2, 1500, window, sinks)


@pytest.mark.parametrize("t,nq,nkv,hd,window,sinks", [("bf16", 4, 4, 128, 100, 4), ("bf16", 8, 4, 64, 40, 70),
                                                      ("f32", 4, 4, 64, 300, 130), ("f32", 2, 2, 128, 7, 9)])
@pytest.mark.parametrize("more", [0, 37])
def test_gradient_of_sinks_of_many_sequences(torch, ctx, t, nq, nkv, hd, window, sinks, more):
    """Long sequences among many short ones and ones of about a chunk of queries (256; of 300 keys 320)."""
    import raster_amd

    print(f"[gpu] window sinks of many {t} {nq}/{nkv}x{hd} {window}+{sinks}", flush=True)
    lens = [1, 0, 257, 3, 900, 255, 256, 1, 0, 0, 321, 319, 320, 2, 512, 513, 5, 640, 641, 1, 130, 2, 2, 700, 0]
    lk = [n + more for n in lens]
    q, k, v, do = data(torch, t, nq, nkv, hd, lens, lk, window)
    cu, cu_k, scale = cu_of(torch, lens), None if lens == lk else cu_of(torch, lk), hd ** -0.5
    lse = torch.empty((nq, sum(lens)), device="cuda")
    see = dict(window=window, sinks=sinks, cu_k=cu_k)
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, **see)
    nan = [torch.full_like(x, float("nan")) for x in (q, k, v)]
    grads = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, dq=nan[0], dk=nan[1],
                                            dv=nan[2], **see)
    check_gradient(torch, q, k, v, do, grads, lens, lk, nq, nkv, hd, scale, window, sinks)


def test_gradient_of_sinks_of_very_many_sequences(torch, ctx):
    """9000 sequences x 16 KV heads x 8 tiles of sinks, one workgroup for each where there are 16 for each otherwise: the
    long ones in the middle as by themselves, up to the order of sums; the rest, of one token each, have dq = dk = 0."""
    import raster_amd

    nq = nkv = 16
    hd, batch, see, scale = 8, 9000, dict(window=30, sinks=500), 0.3
    print("[gpu] window sinks of very many", flush=True)
    lens = [1] * batch
    lens[batch // 2], lens[batch // 2 + 1] = 1200, 600
    n, at = sum(lens), batch // 2
    q, k, v, do = data(torch, "f32", nq, nkv, hd, lens, lens, 4)

    def both(s, cu):
        x = [t[s] for t in (q, k, v, do)]
        lse = torch.empty((nq, x[0].shape[0]), device="cuda")
        out = raster_amd.prompt_attention(ctx, *x[:3], cu, nq, nkv, hd, scale, lse=lse, **see)
        return raster_amd.prompt_attention_bwd(ctx, x[3], *x[:3], out, lse, cu, nq, nkv, hd, scale, **see)

    many, alone = both(slice(0, n), cu_of(torch, lens)), both(slice(at, at + 1800), cu_of(torch, [1200, 600]))
    for a, b in zip(many, alone):
        assert bool(((a[at:at + 1800] - b).abs() <= 2.0 ** -16 * b.abs().max()).all())
    for a in many[:2]:
        assert float(a[:at].abs().max()) <= 1e-5 and float(a[at + 1800:].abs().max()) <= 1e-5
    assert torch.allclose(many[2][:at], do[:at], rtol=1e-6, atol=0)
