"""rq_prompt_attention and rq_prompt_attention_bwd against every head in 64 bits
(attn_ref.py states the tolerances: rounding counts, elementwise)."""
import pytest

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
    """[n, width] rows of a wider array when pad is given."""
    return torch.randn((n, width + pad), generator=g, device="cuda").to(dtype)[:, :width]


def heads(t, h, hd):
    return t[:, h * hd:(h + 1) * hd].double()


def check_forward(torch, q, k, v, out, lse, lq, lk, nq, nkv, hd, scale, is_causal, start=0):
    import attn_ref as ref

    half = ref.HALF[q.dtype]
    a0 = b0 = start
    for a, b in zip(lq, lk):
        see = ref.causal(a, b) if is_causal else torch.ones((a, b), dtype=torch.bool, device="cuda")
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


# type, heads, KV heads, head_dim, queries and keys of each sequence
CASES = [
    ("bf16", 4, 4, 128, [1], [1]),
    ("bf16", 4, 2, 128, [37], [37]),
    ("bf16", 8, 2, 128, [128, 1, 0, 129, 333], [128, 1, 0, 129, 333]),
    ("bf16", 8, 1, 64, [65, 200, 31], [65, 200, 31]),
    ("bf16", 3, 3, 80, [90, 17], [90, 17]),
    ("bf16", 2, 2, 8, [70], [70]),
    ("bf16", 4, 2, 256, [100, 33], [100, 33]),
    ("bf16", 2, 1, 200, [61], [61]),
    ("bf16", 2, 2, 128, [5, 64, 100], [300, 64, 40]),     # the end of a sequence; more queries than keys
    ("bf16", 2, 2, 128, [40, 0, 7], [0, 50, 3]),          # no keys, no queries
    ("bf16", 2, 2, 128, [1500], [1500]),
    ("bf16", 64, 8, 128, [300, 129, 40], [300, 129, 40]),  # grids that fill the CUs: keys not split
    ("bf16", 64, 8, 64, [300, 129, 90], [300, 129, 90]),
    ("bf16", 64, 8, 128, [300, 129, 90, 5], [300, 129, 90, 5]),
    ("bf16", 96, 8, 128, [300, 129, 90, 5], [300, 129, 90, 5]),
    ("bf16", 128, 8, 64, [300, 129, 90], [300, 129, 90]),
    ("bf16", 16, 4, 256, [200, 70], [200, 70]),
    ("bf16", 4, 4, 144, [5, 40], [300, 331]),
    ("bf16", 64, 8, 200, [300, 129, 90], [300, 129, 90]),
    ("bf16", 128, 8, 72, [300, 0, 90], [310, 129, 90]),
    ("f32", 64, 8, 104, [300, 0, 90], [310, 129, 90]),
    ("f32", 64, 8, 128, [300, 129, 90], [300, 129, 90]),
    ("f32", 128, 8, 40, [300, 129, 90], [300, 129, 90]),
    ("f32", 4, 4, 128, [1], [1]),
    ("f32", 4, 2, 128, [33, 0, 130], [33, 0, 130]),
    ("f32", 6, 2, 64, [65, 200], [65, 200]),
    ("f32", 3, 3, 40, [77], [77]),
    ("f32", 2, 1, 256, [70, 9], [70, 9]),
    ("f32", 2, 2, 128, [5, 64, 100], [300, 64, 40]),
]


@pytest.mark.parametrize("t,nq,nkv,hd,lq,lk", CASES)
@pytest.mark.parametrize("is_causal", [True, False], ids=["causal", "full"])
def test_forward(torch, ctx, t, nq, nkv, hd, lq, lk, is_causal):
    import raster_amd

    print(f"[gpu] prompt {t} {nq}/{nkv}x{hd} {lq} {lk} causal={is_causal}", flush=True)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[t]
    g = torch.Generator(device="cuda").manual_seed(hd + sum(lq))
    q, k, v = (rows(torch, g, sum(n), w * hd, dt) for n, w in ((lq, nq), (lk, nkv), (lk, nkv)))
    scale = hd ** -0.5
    lse = torch.empty((nq, sum(lq)), device="cuda")
    out = raster_amd.prompt_attention(ctx, q, k, v, cu_of(torch, lq), nq, nkv, hd, scale, causal=is_causal,
                                      cu_k=None if lq == lk else cu_of(torch, lk), lse=lse)
    check_forward(torch, q, k, v, out, lse, lq, lk, nq, nkv, hd, scale, is_causal)


@pytest.mark.parametrize("nq,nkv,hd,lq,lk", [(8, 2, 128, [4600], [4600]), (6, 6, 72, [5000, 4000], [5000, 4700])])
def test_long_sequences(torch, ctx, nq, nkv, hd, lq, lk):
    """The kernel of long sequences (bf16, more than 4096 queries each on average)."""
    import raster_amd

    print(f"[gpu] prompt long {nq}/{nkv}x{hd} {lq} {lk}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(sum(lq))
    q, k, v = (rows(torch, g, sum(n), w * hd, torch.bfloat16) for n, w in ((lq, nq), (lk, nkv), (lk, nkv)))
    scale, lse = hd ** -0.5, torch.empty((nq, sum(lq)), device="cuda")
    cu_k = None if lq == lk else cu_of(torch, lk)
    for is_causal in (True, False):
        out = raster_amd.prompt_attention(ctx, q, k, v, cu_of(torch, lq), nq, nkv, hd, scale, causal=is_causal,
                                          cu_k=cu_k, lse=lse)
        check_forward(torch, q, k, v, out, lse, lq, lk, nq, nkv, hd, scale, is_causal)


@pytest.mark.parametrize("t,nq,nkv,hd,lq,lk", [c for c in CASES if max(c[4]) <= 400])
@pytest.mark.parametrize("is_causal", [True, False], ids=["causal", "full"])
def test_gradient(torch, ctx, t, nq, nkv, hd, lq, lk, is_causal):
    import attn_ref as ref
    import raster_amd

    print(f"[gpu] prompt gradient {t} {nq}/{nkv}x{hd} {lq} {lk} causal={is_causal}", flush=True)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[t]
    g = torch.Generator(device="cuda").manual_seed(1 + hd + sum(lq))
    q, k, v, do = (rows(torch, g, sum(n), w * hd, dt) for n, w in ((lq, nq), (lk, nkv), (lk, nkv), (lq, nq)))
    scale = hd ** -0.5
    cu, cu_k = cu_of(torch, lq), None if lq == lk else cu_of(torch, lk)
    lse = torch.empty((nq, sum(lq)), device="cuda")
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, causal=is_causal, cu_k=cu_k, lse=lse)
    dq, dk, dv = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale,
                                                 causal=is_causal, cu_k=cu_k)
    a0 = b0 = 0
    for a, b in zip(lq, lk):
        see = ref.causal(a, b) if is_causal else torch.ones((a, b), dtype=torch.bool, device="cuda")
        for j in range(nkv):
            kj, vj = heads(k[b0:b0 + b], j, hd), heads(v[b0:b0 + b], j, hd)
            wk, wv, bk, bv = (torch.zeros((b, hd), dtype=torch.float64, device="cuda") for _ in range(4))
            for h in range(j * (nq // nkv), (j + 1) * (nq // nkv)):
                (wq, dkh, dvh), (bq, bkh, bvh) = ref.attend_grad(
                    heads(q[a0:a0 + a], h, hd), kj, vj, heads(do[a0:a0 + a], h, hd), scale, see, ref.HALF[dt])
                assert bool(((heads(dq[a0:a0 + a], h, hd) - wq).abs() <= bq).all()), (a, b, h, "dq")
                wk, wv, bk, bv = wk + dkh, wv + dvh, bk + bkh, bv + bvh
            assert bool(((heads(dk[b0:b0 + b], j, hd) - wk).abs() <= bk).all()), (a, b, j, "dk")
            assert bool(((heads(dv[b0:b0 + b], j, hd) - wv).abs() <= bv).all()), (a, b, j, "dv")
        a0, b0 = a0 + a, b0 + b


def test_gradient_against_differences(torch, ctx):
    """The derivative along a direction from two forward calls: sum of dout . out at
    +e and -e, f32, relative to the gradient's own product with the direction. The
    difference errs by e^2 of its third derivative (order 1) and by out's rounding over
    e, 1e-6 / e of the magnitude: 1e-3 at e = 1e-2."""
    import raster_amd

    nq, nkv, hd, lens = 4, 2, 64, [50, 3, 70]
    print("[gpu] prompt gradient against differences", flush=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    n = sum(lens)
    q, do, uq = (torch.randn((n, nq * hd), generator=g, device="cuda") for _ in range(3))
    k, v, uk, uv = (torch.randn((n, nkv * hd), generator=g, device="cuda") for _ in range(4))
    cu, scale, lse = cu_of(torch, lens), hd ** -0.5, torch.empty((nq, n), device="cuda")

    def f(e):
        return float((raster_amd.prompt_attention(ctx, q + e * uq, k + e * uk, v + e * uv, cu, nq, nkv, hd, scale)
                      .double() * do.double()).sum())

    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse)
    grads = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale)
    want = sum(float((a.double() * b.double()).sum()) for a, b in zip(grads, (uq, uk, uv)))
    size = sum(float((a.double() * b.double()).norm()) for a, b in zip(grads, (uq, uk, uv)))
    got = (f(1e-2) - f(-1e-2)) / 2e-2
    assert abs(got - want) <= 1e-3 * max(abs(want), size)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_strided_rows_and_rows_of_no_sequence(torch, ctx, t):
    """q, k, v and the outputs as columns of wider arrays; rows before the first and behind
    the last sequence hold NaN, are not read into any result and stay as they were."""
    import raster_amd

    nq, nkv, hd, lens = 4, 2, 128, [70, 0, 45]
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[t]
    print(f"[gpu] prompt strided {t}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(9)
    n, first = 3 + sum(lens) + 20, 3
    wide = (nq + 2 * nkv) * hd + 16
    buf = torch.randn((n, wide), generator=g, device="cuda").to(dt)
    buf[:first] = buf[first + sum(lens):] = float("nan")
    q, k, v = buf[:, :nq * hd], buf[:, nq * hd:(nq + nkv) * hd], buf[:, (nq + nkv) * hd:(nq + 2 * nkv) * hd]
    do = rows(torch, g, n, nq * hd, dt, pad=8)
    do[:first] = do[first + sum(lens):] = float("nan")
    cu, scale = cu_of(torch, lens, first), hd ** -0.5
    out = torch.full((n, nq * hd + 24), 7.0, dtype=dt, device="cuda")
    lse = torch.full((nq, n), 7.0, device="cuda")
    raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, out=out[:, 8:8 + nq * hd], lse=lse)
    mid = slice(first, first + sum(lens))
    check_forward(torch, q, k, v, out[:, 8:8 + nq * hd], lse, lens, lens, nq, nkv, hd, scale, True, start=first)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[mid] = False
    assert bool((out[keep] == 7).all()) and bool((out[:, :8] == 7).all()) and bool((out[:, 8 + nq * hd:] == 7).all())
    assert bool((lse[:, keep] == 7).all())
    d = torch.full((n, wide), 7.0, dtype=dt, device="cuda")
    dq, dk, dv = d[:, :nq * hd], d[:, nq * hd:(nq + nkv) * hd], d[:, (nq + nkv) * hd:(nq + 2 * nkv) * hd]
    raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out[:, 8:8 + nq * hd], lse, cu, nq, nkv, hd, scale, dq=dq,
                                    dk=dk, dv=dv)
    assert bool((d[keep] == 7).all()) and bool((d[:, -16:] == 7).all())
    # the same sequences by themselves, contiguous: the same bits
    a = [x[mid].contiguous() for x in (q, k, v, do)]
    cu0, lse0 = cu_of(torch, lens), torch.empty((nq, sum(lens)), device="cuda")
    o0 = raster_amd.prompt_attention(ctx, a[0], a[1], a[2], cu0, nq, nkv, hd, scale, lse=lse0)
    g0 = raster_amd.prompt_attention_bwd(ctx, a[3], a[0], a[1], a[2], o0, lse0, cu0, nq, nkv, hd, scale)
    assert torch.equal(o0, out[mid, 8:8 + nq * hd])
    assert all(torch.equal(x, y[mid]) for x, y in zip(g0, (dq, dk, dv)))


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_a_sequence_of_nan_stays_its_own(torch, ctx, t):
    """Sequences share tiles of memory but no values: NaN and inf in one reach no other."""
    import raster_amd

    nq, nkv, hd, lens = 2, 1, 64, [50, 20, 77]
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[t]
    print(f"[gpu] prompt NaN sequence {t}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(4)
    n = sum(lens)
    q, do = (rows(torch, g, n, nq * hd, dt) for _ in range(2))
    k, v = (rows(torch, g, n, nkv * hd, dt) for _ in range(2))
    cu, scale = cu_of(torch, lens), hd ** -0.5

    def both():
        lse = torch.empty((nq, n), device="cuda")
        out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse)
        return [out, *raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale)]

    clean = both()
    for x in (q, k, v, do):
        x[50:70:2], x[51:70:2] = float("nan"), float("inf")
    keep = [i for i in range(n) if not 50 <= i < 70]
    dirty = both()
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(clean, dirty))
    assert bool(torch.isnan(dirty[0][50:70]).all())


def test_infinite_scores(torch, ctx):
    """A key whose score is -inf is left out; a query all of whose scores are -inf gets
    zeros, a log-sum-exp of -inf and no gradient; a score of +inf makes its query NaN."""
    import raster_amd

    hd, n = 64, 40
    print("[gpu] prompt infinite scores", flush=True)
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v, do = (torch.randn((n, hd), generator=g, device="cuda") for _ in range(4))
    q[:, 0] = 1.0
    k[7, 0] = -float("inf")
    cu, lse = cu_of(torch, [n]), torch.empty((1, n), device="cuda")
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, 1, 1, hd, 0.125, causal=False, lse=lse)
    keep = [i for i in range(n) if i != 7]
    want = torch.softmax(q.double() @ k[keep].double().T * 0.125, 1) @ v[keep].double()
    assert float((out.double() - want).abs().max()) < 1e-5
    k[:, 0] = -float("inf")
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, 1, 1, hd, 0.125, lse=lse)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())
    k[:, 0] = 0.0
    k[3, 0] = float("inf")
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, 1, 1, hd, 0.125)
    assert bool(torch.isnan(out[3:]).all()) and bool(torch.isfinite(out[:3]).all())


def test_graph_replays_and_streams(torch, ctx):
    """Forward and gradient captured twice on one stream, the graphs replayed on two
    streams with eager work between: every replay gives the eager bits."""
    import raster_amd

    nq, nkv, hd = 4, 2, 128
    print("[gpu] prompt graphs", flush=True)
    scale = hd ** -0.5

    def data(seed, lens):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = sum(lens)
        return [rows(torch, g, n, w * hd, torch.bfloat16) for w in (nq, nkv, nkv, nq)] + [cu_of(torch, lens)]

    def call(d, stream=None):
        q, k, v, do, cu = d
        lse = torch.empty((nq, q.shape[0]), device="cuda")
        out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse, stream=stream)
        return [out, lse, *raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale,
                                                           stream=stream)]

    sets = [data(1, [100, 31]), data(2, [257])]
    eager = [[x.clone() for x in call(d)] for d in sets]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs, outs = [], []
    for d in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            outs.append(call(d))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        call(sets[0])
        torch.cuda.synchronize()
        for a, b in zip(eager, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    # another stream than the current one, new outputs
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    a = call(sets[1], stream=st)
    st.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, eager[1]))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch", [64, 65, 300, 5000])
def test_many_sequences(torch, ctx, dtype, batch):
    """More sequences than a wave has lanes, most of a few rows or none: one dense product
    with a mask of equal sequences is the reference."""
    import attn_ref as ref
    import raster_amd

    print(f"[gpu] prompt {dtype} {batch} sequences", flush=True)
    nq, nkv, hd, scale = 2, 1, 64, 0.125
    ty = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g = torch.Generator(device="cuda").manual_seed(batch)
    lens = torch.randint(0, 4, (batch,), generator=torch.Generator().manual_seed(batch))
    lens[torch.randperm(batch)[batch // 4:]] = 0
    lens[batch // 2] = 200
    lens[-1] = 33
    n = int(lens.sum())
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).int().cuda()
    owner = torch.repeat_interleave(torch.arange(batch), lens).cuda()
    see = (owner[:, None] == owner[None]) & ref.causal(n, n)
    q, k, v, do = (rows(torch, g, n, w * hd, ty) for w in (nq, nkv, nkv, nq))
    lse = torch.empty((nq, n), device="cuda")
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, lse=lse)
    dq, dk, dv = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale)
    half = ref.HALF[ty]
    sums = [0.0] * 4
    for h in range(nq):
        args = heads(q, h, hd), heads(k, 0, hd), heads(v, 0, hd)
        want, wlse, bound = ref.attend(*args, scale, see, half)
        assert bool(((heads(out, h, hd) - want).abs() <= bound).all())
        assert bool(((lse[h].double() - wlse).abs() <= 1e-5 * (1 + wlse.abs())).all())
        (wq, wk, wv), (bq, bk, bv) = ref.attend_grad(*args, heads(do, h, hd), scale, see, half)
        assert bool(((heads(dq, h, hd) - wq).abs() <= bq).all())
        sums = [a + b for a, b in zip(sums, (wk, wv, bk, bv))]
    for got, want, bound in ((dk, sums[0], sums[2]), (dv, sums[1], sums[3])):
        assert bool(((got.double() - want).abs() <= bound + half * want.abs()).all())


def test_rows_more_than_4_gib_apart(torch, ctx):
    """The widest stride, 2^22 elements, and offsets past 32 bits."""
    import raster_amd

    print("[gpu] prompt, 2^22 elements a row", flush=True)
    n, nq, nkv, hd, scale = 620, 2, 1, 64, 0.125
    wide = torch.empty((n, 2 ** 22), dtype=torch.bfloat16, device="cuda")  # 5 GiB, a few columns of it used
    g = torch.Generator(device="cuda").manual_seed(5)
    width = (nq + 2 * nkv) * hd
    wide[:, :width] = torch.randn((n, width), generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = wide[:, :nq * hd], wide[:, nq * hd:(nq + 1) * hd], wide[:, (nq + 1) * hd:width]
    near = [t.contiguous() for t in (q, k, v)]
    cu = cu_of(torch, [100, 520])
    lse = torch.empty((nq, n), device="cuda")
    want = raster_amd.prompt_attention(ctx, *near, cu, nq, nkv, hd, scale, lse=lse)
    assert torch.equal(raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale), want)
    do = torch.randn((n, nq * hd), generator=g, device="cuda").to(torch.bfloat16)
    grads = raster_amd.prompt_attention_bwd(ctx, do, *near, want, lse, cu, nq, nkv, hd, scale)
    far = raster_amd.prompt_attention_bwd(ctx, do, q, k, v, want, lse, cu, nq, nkv, hd, scale)
    assert all(torch.equal(a, b) for a, b in zip(grads, far))


@pytest.mark.parametrize("t,nq,nkv,hd,n", [("bf16", 2, 1, 128, 300), ("bf16", 64, 8, 128, 700), ("bf16", 2, 1, 128, 4500),
                                           ("f32", 2, 2, 64, 300), ("f32", 4, 1, 256, 300)])
def test_nan_in_masked_keys_and_values(torch, ctx, t, nq, nkv, hd, n):
    """A NaN in k reaches no query that does not see it; one in v none before its tile (64 keys at most)."""
    import raster_amd

    print(f"[gpu] masked NaN {t} {nq}/{nkv}x{hd} {n}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(n)
    ty = {"bf16": torch.bfloat16, "f32": torch.float32}[t]
    q, k, v = (rows(torch, g, n, w * hd, ty) for w in (nq, nkv, nkv))
    cu, scale, at = cu_of(torch, [n]), hd ** -0.5, 200
    want = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale)
    for x, first in ((k, at), (v, at // 64 * 64)):
        keep = x[at].clone()
        for bad in (float("nan"), float("inf")):
            x[at] = bad
            out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale)
            assert torch.equal(out[:first], want[:first])
            assert not bool(torch.isfinite(out[at:]).all(1).any())
        x[at] = keep
