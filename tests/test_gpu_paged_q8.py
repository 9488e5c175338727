"""Int8 pages: append, one-token attention and stored rows, against the block's arithmetic in plain torch
(q8_ref.py, bit for bit) and attention over the stored values in 64 bits (attn_ref.py states the tolerances)."""
import pytest

pytestmark = pytest.mark.gpu

THETA = 1e4


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


def new_rows(torch, seed, act, rows, nq, nkv, hd):
    ty = {"f32": torch.float32, "bf16": torch.bfloat16}[act]
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn((rows, (nq + 2 * nkv) * hd), generator=g, device="cuda").to(ty)
    return qkv.split([nq * hd, nkv * hd, nkv * hd], 1)


def near_codes(got, want, x, s):
    """Rotations may differ in an angle's last bit: the codes agree, or x / s is by the border (127 steps of 2^-21)."""
    off = got != want
    return bool(((got.double() - x.double() / s.double()).abs()[off] <= 0.5 + 127 * 2.0 ** -21).all())


def check_out(torch, ref, out, q, cache, lens, add, nq, nkv, hd, scale, window, sinks):
    """out's rows against attention over the cache as it is stored; q: the rotated queries, f64 [batch, nq, hd].

    Beside attn_ref's roundings two of the kernel's own: queries and weights are whole numbers of `step` = 1 / (2 M) of the
    largest of their head, or tile, M = 0x7F7F7C for f32 results and 0x7F7E for bf16 ones (the factors by a reciprocal of one unit in
    the last place: 2^-22 more). A query's element is off by at most step * max |q|, a score by that times the sum of |k|, a
    weight, relatively, by twice as much (its own score and the sum); a weight with its block's scale, w, by at most step * max w,
    and so element d of the result by that times the sum of the rows' |code| there."""
    half = ref.HALF[out.dtype]
    step = 0.5 / (0x7F7F7C if out.dtype == torch.float32 else 0x7F7E) * (1 + 2.0 ** -20)
    for b, m in enumerate(lens):
        if m < 0 or m + add == 0:
            assert bool((out[b] == 0).all())
            continue
        n = m + add
        keys, values = cache.values("k", b, n), cache.values("v", b, n)
        scales = cache.vs[cache._mine(b, n)].reshape(-1, nkv).double().repeat_interleave(16, 0)[:n]
        j = torch.arange(n, device="cuda")
        see = (((n - 1 - j < window) | (j < sinks)) if window else j >= 0)[None]
        for h in range(nq):
            g = h // (nq // nkv)
            qh, kh, vh = q[b, h:h + 1], keys[:, g], values[:, g]
            want, lse, bound = ref.attend(qh, kh, vh, scale, see, half, 2.0 ** -22)
            p = torch.where(see, torch.exp(qh @ kh.T * scale - lse[:, None]), 0.0)[0]
            off = step * qh.abs().max() * (kh.abs().sum(1) * see[0]).max() * scale
            codes = torch.where(scales[:, g:g + 1] > 0, vh / scales[:, g:g + 1], 0.0).abs() * see[0][:, None]
            extra = 2 * off * (p @ vh.abs()) + step * (p * scales[:, g]).max() * codes.sum(0)
            got = out[b, h * hd:(h + 1) * hd].double()
            assert bool(((got - want[0]).abs() <= bound[0] + extra).all()), (
                b, h, float(((got - want[0]).abs() / (bound[0] + extra)).max()))


# activations, heads, KV heads, head_dim, page, cached rows, window, sinks
CASES = [
    ("f32", 4, 4, 128, 16, [0], 0, 0),
    ("f32", 16, 16, 128, 16, [128, 0, 31, 32, 33, 15, 16, 17], 0, 0),
    ("f32", 8, 2, 64, 32, [7, 700, 255, 256, 257], 0, 0),
    ("f32", 6, 2, 40, 16, [100, 3], 0, 0),
    ("f32", 4, 1, 256, 16, [300, 40, 95], 0, 0),
    ("f32", 2, 2, 136, 16, [77], 0, 0),
    ("f32", 2, 1, 200, 32, [130, 4], 0, 0),
    ("f32", 5, 1, 8, 16, [130, 4], 0, 0),
    ("bf16", 32, 8, 128, 16, [2500, 77, 0, 1024, 4099], 0, 0),
    ("bf16", 64, 2, 64, 128, [300, 5000], 0, 0),  # 32 heads a KV head: the row is appended in a launch before
    ("bf16", 17, 1, 128, 16, [40, 0, 15, 16], 0, 0),
    ("f32", 40, 2, 104, 16, [47, 200], 30, 5),
    ("bf16", 3, 3, 80, 16, [90, 12], 0, 0),
    ("bf16", 2, 1, 248, 16, [400, 33], 0, 0),
    ("bf16", 8, 2, 128, 16, [1000, 0, 5, 16, 63, 64, 65, 300], 64, 4),
    ("f32", 8, 2, 64, 16, [1000, 0, 5, 16, 1999], 1, 0),
    ("f32", 4, 4, 128, 64, [1000, 100, 16, 40], 1, 1),
    ("bf16", 4, 2, 256, 16, [500, 17, 16], 17, 33),
    ("f32", 8, 8, 72, 32, [3000, 40], 1111, 16),
    # groups of 4, 5, 8 and 9 heads, where the digits stop fitting beside each other; few and many rows
    ("f32", 32, 8, 64, 16, [2500, 77, 0, 1024, 4099], 0, 0),
    ("f32", 40, 8, 64, 16, [2500, 77, 0, 1024, 4099], 0, 0),
    ("bf16", 64, 8, 128, 16, [2500, 77, 0, 1024, 4099], 0, 0),
    ("bf16", 36, 4, 128, 16, [2500, 77, 0, 1024], 0, 0),
    ("f32", 20, 4, 128, 32, [28000, 3, 64, 500, 27001, 0, 17, 900], 0, 0),
    ("bf16", 32, 4, 128, 32, [28000, 3, 64, 500, 27001, 0, 17, 900], 0, 0),
    ("bf16", 36, 4, 64, 32, [28000, 3, 64, 500, 27001, 0, 17, 900], 0, 0),
]


@pytest.mark.parametrize("act,nq,nkv,hd,page,lens,window,sinks", CASES)
@pytest.mark.parametrize("mode", ["append", "read", "no_rope"])
def test_attention(torch, ctx, act, nq, nkv, hd, page, lens, window, sinks, mode):
    import attn_ref as ref
    import q8_ref
    import raster_amd

    print(f"[gpu] q8 {act} {nq}/{nkv}x{hd} page={page} {lens} {window}+{sinks} {mode}", flush=True)
    add = mode != "read"
    lens = lens + [-1]
    n = len(lens)
    cache = q8_ref.Cache(hd + sum(lens), nkv, hd, [x + 1 for x in lens], page, lens, pad=3 if hd == 64 else 0)
    q, k, v = new_rows(torch, sum(lens), act, n, nq, nkv, hd)
    theta, scale = 0.0 if mode == "no_rope" else THETA, hd ** -0.5
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = cache.clone()
    out = raster_amd.paged_attention(ctx, q, k if add else None, v if add else None, cache.k, cache.v, cache.table, lt,
                                     nq, nkv, hd, theta, scale, max_len=max(lens) + 1, window=window, sinks=sinks,
                                     **cache.scales())
    pos = torch.tensor(lens, device="cuda")
    k32 = q8_ref.rope32(k.float().view(n, nkv, hd), pos, theta)
    if add:
        for b, m in enumerate(lens):
            if m >= 0:
                want.append("k", b, m, k32[b:b + 1])
                want.append("v", b, m, v[b:b + 1].float().view(1, nkv, hd))
    if theta and add:  # (an angle's last bit)
        for b, m in enumerate(lens):
            if m < 0:
                continue
            at = (int(cache.table[b, m // page]), m % page)
            s = cache.ks[at[0], at[1] // 16]
            assert bool(((s - want.ks[at[0], at[1] // 16]).abs() <= 2.0 ** -22 * s).all())
            codes = (c.k[at].view(nkv, hd) for c in (cache, want))
            assert near_codes(*codes, k32[b], s[:, None])
            want.k[at], want.ks[at[0], at[1] // 16] = cache.k[at], s
    assert cache.same(want)
    rq = ref.rope(q.double().view(n, nq, hd), pos, theta) if theta else q.double().view(n, nq, hd)
    check_out(torch, ref, out, rq, cache, lens, add, nq, nkv, hd, scale, window, sinks)


@pytest.mark.parametrize("act,nq,nkv,hd,page,lens,past", [
    ("f32", 4, 2, 128, 16, [37, 0, 1, 16, 15, 2], [0, 5, 15, 1000, 1, 15]),
    ("f32", 3, 1, 40, 32, [33, 2], [31, 5000]),
    ("bf16", 32, 8, 128, 16, [300, 1, 77], [0, 128, 5]),
    ("bf16", 2, 2, 8, 16, [5], [3]),
    ("bf16", 2, 1, 256, 64, [70, 17, 18], [0, 15, 30]),
    ("f32", 2, 1, 248, 16, [40], [9]),
    ("bf16", 4, 4, 64, 128, [200, 16], [100, 0]),
])
@pytest.mark.parametrize("theta", [0.0, THETA])
@pytest.mark.parametrize("in_place", [False, True])
def test_append(torch, ctx, act, nq, nkv, hd, page, lens, past, theta, in_place):
    import q8_ref
    import raster_amd

    print(f"[gpu] q8 append {act} {nq}/{nkv}x{hd} {lens} {past}", flush=True)
    n, tail = sum(lens), 3
    lens2, past2 = lens + [2], past + [-1]  # a sequence left out, and rows of none behind it
    cache = q8_ref.Cache(n, nkv, hd, [a + b for a, b in zip(lens, past)] + [1], page, past + [0],
                         pad=5 if in_place else 0)
    want = cache.clone()
    q, k, v = (x.contiguous() if not in_place else x for x in new_rows(torch, n, act, n + 2 + tail, nq, nkv, hd))
    cu = torch.tensor([sum(lens2[:i]) for i in range(len(lens2) + 1)], dtype=torch.int32, device="cuda")
    pt = torch.tensor(past2, dtype=torch.int32, device="cuda")
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    qo, ko = (q, k) if in_place else (torch.full_like(q, 7.0), torch.full_like(k, 7.0))
    raster_amd.pages_append(ctx, q, k, v, cache.k, cache.v, cache.table, cu, pt, nq, nkv, hd, theta, q_out=qo, k_out=ko,
                            **cache.scales())
    at = 0
    for b, (m, p0) in enumerate(zip(lens, past)):
        if m == 0:
            continue
        pos = torch.arange(p0, p0 + m, device="cuda")
        rows = slice(at, at + m)
        q32, k32 = (q8_ref.rope32(x[rows].float().view(m, -1, hd), pos, theta) for x in (q0, k0))
        for got, w in ((qo[rows], q32), (ko[rows], k32)):
            w = w.reshape(m, -1)
            tol = (2.0 ** -8 if act == "bf16" else 2.0 ** -22) * (w.abs() + 1)
            assert bool(((got.float() - w).abs() <= tol).all()) if theta else torch.equal(got, w.to(got.dtype))
        want.append("k", b, p0, k32)
        want.append("v", b, p0, v0[rows].float().view(m, nkv, hd))
        if theta:
            pages, r = cache.table[b].long()[pos // page], pos % page
            s = cache.ks[pages, r // 16]
            assert bool(((s - want.ks[pages, r // 16]).abs() <= 2.0 ** -22 * s).all())
            assert near_codes(cache.k[pages, r].view(m, nkv, hd), want.k[pages, r].view(m, nkv, hd), k32, s[..., None])
            want.k[pages, r], want.ks[pages, r // 16] = cache.k[pages, r], s
        at += m
    assert cache.same(want)
    assert torch.equal(qo[n:], q0[n:] if in_place else torch.full_like(qo[n:], 7.0))
    assert torch.equal(ko[n:], k0[n:] if in_place else torch.full_like(ko[n:], 7.0))
    assert torch.equal(v, v0)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("most", [127.0, 1.0, 3.7e5, 3e38, 1.28e-28, 1.26e-28, 1e-36, 3e-38, 2e-43])
def test_codes_where_two_are_as_near(torch, ctx, act, most):
    """Values halfway between two codes and the floats beside those, with scales up to the largest and down to
    denormal ones: the codes of the definition, bit for bit, from prompts and from single tokens."""
    import q8_ref
    import raster_amd

    print(f"[gpu] q8 ties {act} {most}", flush=True)
    dt = torch.float32 if act == "f32" else torch.bfloat16
    top = torch.tensor(most).to(dt).float()
    s = top * torch.tensor(1 / 127)
    x = (torch.arange(-127, 127) + 0.5) * s
    inf = torch.tensor(float("inf"))
    x = torch.stack([x, torch.nextafter(x, inf), torch.nextafter(x, -inf)]).flatten().to(dt).float()
    x = x[x.abs() <= top]
    x = torch.cat([top[None], x, torch.zeros(16 * 128)])[:16 * 128].view(16, 1, 128)
    codes, scales = torch.zeros((1, 16, 1, 128), dtype=torch.int8), torch.zeros((1, 1))
    q8_ref.put(codes, scales, 0, x)
    one = codes.clone()
    for single in (False, True):
        cache = q8_ref.Cache(1, 1, 128, [16], 16, [0])
        k = x.view(16, 128).to("cuda", dt)
        if single:
            for i in range(16):
                raster_amd.paged_attention(ctx, k[i:i + 1], k[i:i + 1], k[i:i + 1], cache.k, cache.v, cache.table,
                                           torch.tensor([i], dtype=torch.int32, device="cuda"), 1, 1, 128, 0.0, 0.1,
                                           max_len=16, **cache.scales())
        else:
            raster_amd.pages_append(ctx, k, k, k, cache.k, cache.v, cache.table,
                                    torch.tensor([0, 16], dtype=torch.int32, device="cuda"),
                                    torch.zeros(1, dtype=torch.int32, device="cuda"), 1, 1, 128, 0.0, **cache.scales())
        page = int(cache.table[0, 0])
        for pages, sc in ((cache.k, cache.ks), (cache.v, cache.vs)):
            assert float(sc[page, 0, 0]) == float(scales[0, 0])
            assert torch.equal(pages[page].cpu().view(16, 1, 128), one[0])


@pytest.mark.parametrize("act,nq", [("f32", 4), ("f32", 8), ("bf16", 8), ("bf16", 16)])
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_small_and_large_values(torch, ctx, act, nq, size):
    """Values far from 1. Weights times scales are whole numbers, 2^126 at most for 1: the largest of a tile has p = 1 and
    a scale of more than 1e-30 / 127 = 8e-33 (a block's largest of 1024 normal values is above 1), so 6.7e5 units at least, or
    0x7F7E for bf16 results. Each is off by half of one, which the row's code multiplies; 2^-7 of the sum of p |v|
    is more than all other roundings (bf16's 2^-8, the scores')."""
    import q8_ref
    import raster_amd

    print(f"[gpu] q8 size {size} {act} {nq}", flush=True)
    n, nkv, hd = 200, 2, 64
    cache = q8_ref.Cache(5, nkv, hd, [n], 16, [n])
    g = torch.Generator(device="cuda").manual_seed(2)
    cache.append("v", 0, 0, torch.randn((n, nkv, hd), generator=g, device="cuda") * size)
    dt = torch.float32 if act == "f32" else torch.bfloat16
    q = torch.randn((1, nq * hd), generator=g, device="cuda").to(dt)
    out = raster_amd.paged_attention(ctx, q, None, None, cache.k, cache.v, cache.table,
                                     torch.tensor([n], dtype=torch.int32, device="cuda"), nq, nkv, hd, 0.0, hd ** -0.5,
                                     max_len=n, **cache.scales())
    keys, values = cache.values("k", 0, n), cache.values("v", 0, n)
    for h in range(nq):
        kv = h // (nq // nkv)
        p = torch.softmax(keys[:, kv] @ q[0, h * hd:(h + 1) * hd].double() * hd ** -0.5, 0)
        want, most = p @ values[:, kv], p @ values[:, kv].abs()
        scales = cache.vs[cache._mine(0, n)].reshape(-1, nkv)[:, kv].double().repeat_interleave(16)[:n]
        off = 0.5 / (6.7e5 if act == "f32" else 0x7F7E) * (p * scales).max()
        bound = 2.0 ** -7 * most + off * (values[:, kv] / scales[:, None]).abs().sum(0)
        assert bool(((out[0, h * hd:(h + 1) * hd].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (40, 2, 64)])
def test_a_block_fills_row_by_row(torch, ctx, nq, nkv, hd):
    """33 tokens one by one, of rising and falling size: codes rounded anew, scales that only rise in a block and
    start anew with the next; the same bits when a step is repeated."""
    import attn_ref as ref
    import q8_ref
    import raster_amd

    print(f"[gpu] q8 row by row {nq}/{nkv}x{hd}", flush=True)
    cache = q8_ref.Cache(1, nkv, hd, [40, 50], 16, [0, 13])
    want = cache.clone()
    for step in range(33):
        lens = [step, 13 + step]
        q, k, v = (x * (0.3 + (7 * step) % 11) for x in new_rows(torch, step, "f32", 2, nq, nkv, hd))
        lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for b in range(2):
            for which, x in (("k", k), ("v", v)):
                want.append(which, b, lens[b], x[b:b + 1].reshape(1, nkv, hd))
        first = None
        for _ in range(2):
            out = raster_amd.paged_attention(ctx, q, k, v, cache.k, cache.v, cache.table, lt, nq, nkv, hd, 0.0, 0.05,
                                             **cache.scales())
            assert cache.same(want)
            first = out if first is None else first
            assert torch.equal(out, first)
        check_out(torch, ref, out, q.double().view(2, nq, hd), cache, lens, 1, nq, nkv, hd, 0.05, 0, 0)


def test_values_that_are_not_finite_and_zeros(torch, ctx):
    """A NaN or inf makes its block NaN until the block starts anew, hidden or not, and no other head; zeros stay zeros."""
    import q8_ref
    import raster_amd

    nq, nkv, hd = 4, 2, 64
    print("[gpu] q8 not finite", flush=True)
    cache = q8_ref.Cache(2, nkv, hd, [80, 80], 16, [20, 20])
    q, k, v = (x.contiguous() for x in new_rows(torch, 1, "f32", 2, nq, nkv, hd))
    k[0, 3], v[1, hd + 5] = float("nan"), float("inf")
    args = (nq, nkv, hd, THETA, 0.1)

    def step(lens, q, k, v, **kw):
        lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return raster_amd.paged_attention(ctx, q, k, v, cache.k, cache.v, cache.table, lt, *args, **cache.scales(), **kw)

    out = step([20, 20], q, k, v)
    bad = torch.isnan(out.view(2, nq, hd))
    assert bool(bad[0, :2].all()) and not bool(bad[0, 2:].any())  # KV head 0 of sequence 0
    assert bool(bad[1, 2:].all()) and not bool(bad[1, :2].any())
    assert bool(torch.isnan(cache.ks[int(cache.table[0, 1]), 0, 0])) and bool(torch.isfinite(cache.vs[int(cache.table[0, 1]), 0]).all())
    q, k, v = new_rows(torch, 2, "f32", 2, nq, nkv, hd)
    assert bool(torch.isnan(step([21, 21], q, k, v)).any())  # still the same block
    # rows 32 and on: a window that does not reach back to it
    for r in range(32, 52):
        out = step([r, r], *new_rows(torch, r, "f32", 2, nq, nkv, hd), window=1)
        assert bool(torch.isfinite(out).all())
    assert bool(torch.isfinite(step([52, 52], q, k, v, window=21)).all())
    assert bool(torch.isfinite(step([53, 53], q, k, v, window=22, sinks=3)).all())
    assert bool(torch.isnan(step([54, 54], q, k, v)).any())
    # written from the block's first row on, it is as good as new
    cu = torch.tensor([0, 16, 32], dtype=torch.int32, device="cuda")
    x = new_rows(torch, 4, "f32", 32, nq, nkv, hd)
    raster_amd.pages_append(ctx, *x, cache.k, cache.v, cache.table, cu,
                            torch.tensor([16, 16], dtype=torch.int32, device="cuda"), nq, nkv, hd, THETA, **cache.scales())
    assert bool(torch.isfinite(step([55, 55], q, k, v)).all())
    # zeros
    z = torch.zeros_like(k)
    out = step([64, 64], q, z, z)
    at = int(cache.table[0, 4])
    assert bool((cache.ks[at, 0] == 0).all()) and bool((cache.k[at, 0] == 0).all()) and bool(torch.isfinite(out).all())
    tiny = torch.full_like(k, 1e-44)  # max / 127 is 0 in f32
    step([65, 65], q, tiny, tiny)
    assert bool((cache.ks[at, 0] == 0).all()) and bool((cache.k[at, :2] == 0).all())
    step([66, 66], q, k, v)
    assert bool((cache.k[at, :2] == 0).all()) and bool((cache.k[at, 2] != 0).any())


def test_bad_pages_and_lengths(torch, ctx):
    import q8_ref
    import raster_amd

    print("[gpu] q8 bad pages", flush=True)
    for nq, nkv in ((4, 2), (40, 2)):
        hd, lens = 64, [40, 50, 60, 70]
        start = q8_ref.Cache(5, nkv, hd, [n + 1 for n in lens], 16, lens)
        q, k, v = new_rows(torch, 5, "f32", 4, nq, nkv, hd)
        lt = torch.tensor(lens, dtype=torch.int32, device="cuda")

        def call(c, table, lt, **kw):
            return raster_amd.paged_attention(ctx, q, k, v, c.k, c.v, table, lt, nq, nkv, hd, THETA, hd ** -0.5,
                                              **c.scales(), **kw)

        whole = start.clone()
        good = call(whole, start.table, lt)
        bad, far = start.table.clone(), lt.clone()
        bad[0, 1] = start.k.shape[0]  # read
        bad[1, 3] = -1                # appended (row 50 is in page 3)
        far[3] = 10 ** 6              # past the table
        c = start.clone()
        out = call(c, bad, far)
        for b in (0, 1, 3):
            assert bool(torch.isnan(out[b]).all())
        assert torch.equal(out[2], good[2])
        want = start.clone()  # sequences 0 and 2 wrote their blocks, nobody else anything
        for b in (0, 2):
            at = int(start.table[b, lens[b] // 16])
            want.k[at], want.v[at], want.ks[at], want.vs[at] = whole.k[at], whole.v[at], whole.ks[at], whole.vs[at]
        assert c.same(want)
        c = start.clone()
        out = call(c, start.table, lt, max_len=61)
        assert torch.equal(out[:3], good[:3]) and bool(torch.isnan(out[3]).all())
        at = int(start.table[3, 4])
        assert torch.equal(c.k[at], start.k[at]) and torch.equal(c.ks[at].nan_to_num(), start.ks[at].nan_to_num())
        # pages that the window has left are not looked up
        gone = start.table.clone()
        gone[2, 1:3] = -1
        a, b = (call(start.clone(), t, lt, window=10, sinks=2) for t in (start.table, gone))
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_append_without_a_page(torch, ctx):
    import q8_ref
    import raster_amd

    print("[gpu] q8 append without a page", flush=True)
    c = q8_ref.Cache(1, 2, 64, [40], 16, [0])
    c.table[0, 1] = 10 ** 6
    start = c.clone()
    q, k, v = new_rows(torch, 1, "f32", 70, 2, 2, 64)
    cu, past = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 70], [0]))
    qo, ko = raster_amd.pages_append(ctx, q, k, v, c.k, c.v, c.table, cu, past, 2, 2, 64, THETA, **c.scales())
    lost = torch.zeros(70, dtype=torch.bool, device="cuda")
    lost[16:32] = lost[48:] = True
    assert bool(torch.isnan(qo[lost]).all()) and bool(torch.isnan(ko[lost]).all()) and bool(torch.isfinite(qo[~lost]).all())
    wrote = [int(c.table[0, i]) for i in (0, 2)]
    keep = [i for i in range(c.k.shape[0]) if i not in wrote]
    assert torch.equal(c.k[keep], start.k[keep]) and bool(torch.isnan(c.ks[keep]).all())
    assert bool(torch.isfinite(c.ks[wrote]).all())


@pytest.mark.parametrize("cache", ["i8", "f32", "bf16"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("nkv,hd,page,lens", [(8, 128, 16, [37, 0, 200, 1]), (1, 8, 16, [5]), (3, 40, 32, [33, 100, 0]),
                                              (2, 256, 64, [130, 64])])
def test_rows(torch, ctx, cache, out, nkv, hd, page, lens):
    import q8_ref
    import raster_amd

    print(f"[gpu] rows {cache}->{out} {nkv}x{hd} {lens}", flush=True)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}
    c = q8_ref.Cache(sum(lens), nkv, hd, lens, page, lens, pad=1)
    kp, vp, sc = c.k, c.v, c.scales()
    if cache != "i8":
        g = torch.Generator(device="cuda").manual_seed(1)
        kp, vp = (torch.randn(c.k.shape, generator=g, device="cuda").to(dt[cache]) for _ in range(2))
        sc = {}
    first, n = 2, sum(lens)
    cu = torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    rows = first + n + 3
    wide = torch.full((rows, 2 * nkv * hd + 8), 7.0, dtype=dt[out], device="cuda")
    k, v = wide[:, :nkv * hd], wide[:, nkv * hd:2 * nkv * hd]
    table = c.table.clone()
    if len(lens) > 2:
        table[2, 1] = -1
    raster_amd.pages_rows(ctx, kp, vp, table, cu, rows, nkv, hd, k_out=k, v_out=v, **sc)
    at = first
    for b, m in enumerate(lens):
        if m == 0:
            continue
        mine = c.table[b, :-(-m // page)].long()
        for got, pages, which in ((k, kp, "k"), (v, vp, "v")):
            if cache == "i8":  # code * scale rounded to f32, then to the rows' type
                s = (c.ks if which == "k" else c.vs)[mine].repeat_interleave(16, 1).view(-1, nkv, 1)[:m]
                want = (pages[mine].view(-1, nkv, hd)[:m].float() * s).reshape(m, -1).to(dt[out])
            else:
                want = pages[mine].reshape(-1, nkv * hd)[:m].to(dt[out])
            if b == 2:
                want[page:2 * page] = float("nan")
            assert torch.equal(got[at:at + m].nan_to_num(9.0), want.nan_to_num(9.0))
        at += m
    assert bool((wide[:first] == 7).all()) and bool((wide[at:] == 7).all()) and bool((wide[:, 2 * nkv * hd:] == 7).all())
    k2, v2 = raster_amd.pages_rows(ctx, kp, vp, c.table, cu - first, n, nkv, hd, dt[out], **sc)
    assert k2.shape == (n, nkv * hd) and k2.dtype == dt[out] and v2.dtype == dt[out]


@pytest.mark.parametrize("batch", [65, 300, 5000])
def test_many_sequences(torch, ctx, batch):
    """Appended and read back, most sequences of a few rows or none."""
    import q8_ref
    import raster_amd

    print(f"[gpu] q8 {batch} sequences", flush=True)
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 3, (batch,), generator=gen)
    lens[batch // 3] = 40
    n = int(lens.sum())
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).int().cuda()
    table = torch.randperm(4 * batch, generator=gen).int().view(batch, 4).cuda()
    kp, vp = (torch.zeros((4 * batch, 16, 64), dtype=torch.int8, device="cuda") for _ in range(2))
    sc = dict(kscales=torch.zeros((4 * batch, 1, 1), device="cuda"), vscales=torch.zeros((4 * batch, 1, 1), device="cuda"))
    q, k, v = new_rows(torch, batch, "f32", n, 1, 1, 64)
    past = torch.zeros(batch, dtype=torch.int32, device="cuda")
    qo, ko = raster_amd.pages_append(ctx, q, k, v, kp, vp, table, cu, past, 1, 1, 64, 0.0, **sc)
    assert torch.equal(qo, q) and torch.equal(ko, k)
    k2, v2 = raster_amd.pages_rows(ctx, kp, vp, table, cu, n, 1, 64, **sc)
    owner = torch.repeat_interleave(torch.arange(batch), lens)
    block = torch.arange(n) - cu.cpu()[owner]
    block = owner * 4 + block // 16
    for x, y in ((k, k2), (v, v2)):
        top = torch.zeros(4 * batch).scatter_reduce(0, block, x.abs().amax(1).cpu(), "amax")[block]
        assert bool(((x - y).abs().amax(1).cpu() <= top / 127 * 0.5001).all())  # half a step, and f32's roundings


def test_graphs(torch, ctx):
    """Append, attention and rows captured, replayed on another stream between eager work."""
    import q8_ref
    import raster_amd

    nq, nkv, hd, lens = 8, 2, 128, [300, 2000]
    print("[gpu] q8 graphs", flush=True)
    c = q8_ref.Cache(8, nkv, hd, [n + 1 for n in lens], 16, lens)
    q, k, v = new_rows(torch, 1, "bf16", 2, nq, nkv, hd)
    pq, pk, pv = new_rows(torch, 2, "bf16", 50, nq, nkv, hd)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu, past = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 20, 50], [280, 1970]))
    rows = torch.tensor([0, 300, 2300], dtype=torch.int32, device="cuda")

    def call():
        got = raster_amd.pages_append(ctx, pq, pk, pv, c.k, c.v, c.table, cu, past, nq, nkv, hd, THETA, **c.scales())
        out = raster_amd.paged_attention(ctx, q, k, v, c.k, c.v, c.table, lt, nq, nkv, hd, THETA, hd ** -0.5,
                                         max_len=2001, **c.scales())
        return [*got, out, *raster_amd.pages_rows(ctx, c.k, c.v, c.table, rows, 2300, nkv, hd, **c.scales())]

    call()
    want = [x.clone() for x in call()]
    torch.cuda.synchronize()
    held, gr, s = c.clone(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(gr, stream=s):
        outs = call()
    other = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(other):
            gr.replay()
        torch.cuda.synchronize()
        again = call()
        torch.cuda.synchronize()
        for x, y, z in zip(outs, want, again):
            assert torch.equal(x, y) and torch.equal(z, y)
        assert c.same(held)


@pytest.mark.parametrize("batch,max_len", [(1, 2500), (30, 2500), (90, 2500), (130, 2500), (400, 1500)])
def test_a_graph_follows_the_lengths(torch, ctx, batch, max_len):
    """One captured call replayed over new lengths, ranges planned by waves, by workgroups or not at all: the
    eager call's bits."""
    import raster_amd

    print(f"[gpu] q8 graph over lengths {batch} {max_len}", flush=True)
    nq, nkv, hd, pages = 8, 2, 64, 400
    gen = torch.Generator(device="cuda").manual_seed(batch)
    kp, vp = (torch.randint(-127, 128, (pages, 16, nkv * hd), generator=gen, device="cuda", dtype=torch.int32)
              .to(torch.int8) for _ in range(2))
    ks, vs = (torch.rand((pages, 1, nkv), generator=gen, device="cuda") * 0.02 + 0.01 for _ in range(2))
    table = torch.randint(0, pages, (batch, (max_len + 15) // 16), generator=gen, device="cuda", dtype=torch.int32)
    q = torch.randn((batch, nq * hd), generator=gen, device="cuda")
    lens = torch.full((batch,), 40, dtype=torch.int32, device="cuda")

    def call():
        return raster_amd.paged_attention(ctx, q, None, None, kp, vp, table, lens, nq, nkv, hd, THETA, hd ** -0.5,
                                          max_len=max_len, kscales=ks, vscales=vs)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = call()
    for top in (max_len, 300, 0, max_len):
        lens.copy_(torch.randint(-1, top + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32))
        lens[batch // 2] = top
        graph.replay()
        got = out.clone()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and not bool(torch.isnan(want).any())
        assert bool((want[lens <= 0] == 0).all()) and (top == 0 or bool((want[batch // 2] != 0).any()))


def test_offsets_past_32_bits(torch, ctx):
    """Pages of 4.6 GiB of codes a plane, the last ones used."""
    import raster_amd

    print("[gpu] q8 offsets past 2^32", flush=True)
    nq, nkv, hd, total, used = 8, 8, 128, 300000, 64
    data = torch.empty((2, total, 16, nkv * hd), dtype=torch.int8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    small = torch.randint(-127, 128, (2, used, 16, nkv * hd), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    ssmall = torch.rand((2, used, 1, nkv), generator=g, device="cuda") + 0.01
    scales = torch.empty((2, total, 1, nkv), device="cuda")
    data[:, total - used:], scales[:, total - used:] = small, ssmall
    table = torch.randperm(used, generator=torch.Generator().manual_seed(3)).int().view(2, -1).cuda()
    lens = torch.tensor([300, 511], dtype=torch.int32, device="cuda")
    q, k, v = new_rows(torch, 3, "bf16", 2, nq, nkv, hd)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    outs = []
    for pages, sc, first in ((small, ssmall, 0), (data, scales, total - used)):
        s = dict(kscales=sc[0], vscales=sc[1])
        got = [raster_amd.paged_attention(ctx, q, k, v, pages[0], pages[1], table + first, lens, nq, nkv, hd, THETA,
                                          hd ** -0.5, **s)]
        raster_amd.pages_append(ctx, q, k, v, pages[0], pages[1], table + first, cu, lens - 100, nq, nkv, hd, THETA, **s)
        got += raster_amd.pages_rows(ctx, pages[0], pages[1], table + first, cu * 200, 400, nkv, hd, **s)
        outs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert torch.equal(data[:, total - used:], small) and torch.equal(scales[:, total - used:], ssmall)


@pytest.mark.parametrize("nq,nkv,hd,batch", [(4, 2, 64, 1500), (8, 4, 64, 2100), (20, 1, 40, 1030)])
@pytest.mark.parametrize("max_len", [2001, 4001])  # (sequences of up to 2048 rows stay whole where there are many)
def test_attention_of_many_sequences(torch, ctx, nq, nkv, hd, batch, max_len):
    """More sequences than one launch plans for, a few long ones among short and idle ones, q, k, v and out as columns of
    wider arrays: as in batches of 100, up to the ranges that long ones are cut into, and the same bits in the cache."""
    import raster_amd

    print(f"[gpu] q8 attention of {batch} sequences {nq}/{nkv}x{hd} {max_len}", flush=True)
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(-1, 40, (batch,), generator=gen)
    lens[[3, batch // 2, batch - 2]] = torch.tensor([1900, 700, 2000])
    need = (lens + 16) // 16
    first = torch.cat([torch.zeros(1, dtype=torch.long), need.cumsum(0)])
    table = torch.full((batch, 251), -1, dtype=torch.int32)
    order = torch.randperm(int(first[-1]), generator=gen).int()
    for b in range(batch):
        table[b, :need[b]] = order[first[b]:first[b + 1]]
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = [torch.randint(-127, 128, (int(first[-1]), 16, nkv * hd), generator=g, device="cuda", dtype=torch.int32)
             .to(torch.int8) for _ in range(2)]
    scales = [torch.rand((int(first[-1]), 1, nkv), generator=g, device="cuda") * 0.02 + 0.01 for _ in range(2)]
    wide = torch.randn((batch, (nq + 2 * nkv) * hd + 16), generator=g, device="cuda")
    q, k, v, _ = wide.split([nq * hd, nkv * hd, nkv * hd, 16], 1)
    table, lt = table.cuda(), lens.int().cuda()

    def call(at):
        p, s = [x.clone() for x in pages], [x.clone() for x in scales]
        out = torch.full((batch, nq * hd + 8), 7.0, device="cuda")
        for i in range(0, batch, at):
            j = slice(i, i + at)
            raster_amd.paged_attention(ctx, q[j], k[j], v[j], p[0], p[1], table[j], lt[j], nq, nkv, hd, THETA, hd ** -0.5,
                                       max_len=max_len, out=out[j, 4:-4] if nq * hd % 4 else out[j, 4:4 + nq * hd],
                                       kscales=s[0], vscales=s[1])
        return out, p + s

    a, b = call(batch), call(100)
    assert all(torch.equal(x, y) for x, y in zip(a[1], b[1]))
    assert bool((a[0][:, :4] == 7).all()) and bool((a[0][:, 4 + nq * hd:] == 7).all())
    x, y = a[0][:, 4:4 + nq * hd], b[0][:, 4:4 + nq * hd]
    assert bool((x[lens < 0] == 0).all())
    # weights are 23-bit shares of a tile's largest, sums in f32: a few 2^-23 of the row's largest value
    assert bool(((x - y).abs() <= 2.0 ** -19 * y.abs().amax(1, keepdim=True)).all())


def test_streams_and_threads(torch, ctx):
    """Calls on streams of their own from four threads over caches of their own: the bits of the same calls in turn."""
    import threading

    import q8_ref
    import raster_amd

    nq, nkv, hd, lens = 8, 2, 128, [300, 2000, 15]
    print("[gpu] q8 threads", flush=True)
    sets = []
    for i in range(4):
        c = q8_ref.Cache(i, nkv, hd, [n + 8 for n in lens], 16, lens)
        sets.append((c, c.clone(), [new_rows(torch, 10 * i + s, "f32", 3, nq, nkv, hd) for s in range(5)]))

    def steps(c, rows, stream):
        outs = []
        for s, (q, k, v) in enumerate(rows):
            lt = torch.tensor([n + s for n in lens], dtype=torch.int32).to("cuda", non_blocking=False)
            if stream is not None:
                stream.wait_stream(torch.cuda.default_stream())
            outs.append(raster_amd.paged_attention(ctx, q, k, v, c.k, c.v, c.table, lt, nq, nkv, hd, THETA, hd ** -0.5,
                                                   stream=stream, window=600 if s % 2 else 0, sinks=2, **c.scales()))
            if stream is not None:
                stream.synchronize()
        return outs

    want = [steps(c, rows, None) for c, _, rows in sets]
    torch.cuda.synchronize()
    got = [None] * 4

    def run(i):
        got[i] = steps(sets[i][1], sets[i][2], torch.cuda.Stream())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for (c, d, _), x, y in zip(sets, want, got):
        assert d.same(c) and all(torch.equal(p, r) for p, r in zip(x, y))


@pytest.mark.parametrize("act,nq", [("f32", 4), ("f32", 8), ("bf16", 8), ("bf16", 16), ("bf16", 40)])
@pytest.mark.parametrize("most", [8e37, 1e38, 3.3e38])
def test_queries_up_to_the_largest(torch, ctx, act, nq, most):
    """Queries whose largest element is past 2^126 over normal keys: scores so far apart that one key has all the weight.

    A score is off by step * max |q| times the sum of |k| (check_out) and by (hd + 4) 2^-24 of the products' magnitudes, or
    2^-22 of them. Where the best is ahead of the second by more than twice that and 1000, every other weight is below
    2^-1000, 0 in f32. The best one is 1 (f32: exp2 of its own difference, 0), with its block's scale a whole number of
    steps of the tile's largest scale; the sum of weights is 1, its join with other ranges exact: the row's values, off by
    step * the largest scale * |code|, a few 2^-24 and the result's rounding."""
    import attn_ref as ref
    import q8_ref
    import raster_amd

    print(f"[gpu] q8 queries {most} {act} {nq}", flush=True)
    nkv, hd, lens, scale = 2, 64, [200, 2500], 0.01
    cache = q8_ref.Cache(6, nkv, hd, lens, 16, lens)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn((2, nq, hd), generator=g, device="cuda")
    q = (q / q.abs().amax(2, keepdim=True) * most).to(torch.float32 if act == "f32" else torch.bfloat16)
    out = raster_amd.paged_attention(ctx, q.view(2, -1), None, None, cache.k, cache.v, cache.table,
                                     torch.tensor(lens, dtype=torch.int32, device="cuda"), nq, nkv, hd, 0.0, scale,
                                     max_len=2500, **cache.scales())
    half = ref.HALF[out.dtype]
    step = 0.5 / (0x7F7F7C if act == "f32" else 0x7F7E) * (1 + 2.0 ** -20)
    sure = 0
    for b, n in enumerate(lens):
        keys, values = cache.values("k", b, n), cache.values("v", b, n)
        scales = cache.vs[cache._mine(b, n)].reshape(-1, nkv).double()
        for h in range(nq):
            qh, kh, vh = q[b, h].double(), keys[:, h // (nq // nkv)], values[:, h // (nq // nkv)]
            top, at = (kh @ qh * scale).topk(2)
            off = step * qh.abs().max() * kh.abs().sum(1).max() * scale + 2.0 ** -22 * (kh.abs() @ qh.abs()).max() * scale
            got = out[b, h * hd:(h + 1) * hd].double()
            assert bool(torch.isfinite(got).all())
            if top[0] - top[1] <= 2 * off + 1000:
                continue
            sure += 1
            s = scales[:, h // (nq // nkv)]
            want, code = vh[at[0]], vh[at[0]].abs() / s[at[0] // 16]
            assert bool(((got - want).abs() <= (half + 2.0 ** -21) * want.abs() + step * s.max() * code).all()), (b, h)
    assert sure >= nq


def test_no_rows_allowed(torch, ctx):
    """max_len 0 allows no row: nothing is stored, whatever the heads a KV head; results are NaN, an idle slot's zeros."""
    import q8_ref
    import raster_amd

    for nq, nkv in ((4, 2), (40, 2)):
        print(f"[gpu] q8 max_len 0 {nq}/{nkv}", flush=True)
        lens = [40, 0, -1, 47]
        cache = q8_ref.Cache(5, nkv, 64, [n + 1 for n in lens], 16, lens)
        start = cache.clone()
        q, k, v = (9 * x for x in new_rows(torch, 5, "f32", 4, nq, nkv, 64))  # (larger than what is there: a scale would rise)
        out = raster_amd.paged_attention(ctx, q, k, v, cache.k, cache.v, cache.table,
                                         torch.tensor(lens, dtype=torch.int32, device="cuda"), nq, nkv, 64, THETA, 0.1,
                                         max_len=0, **cache.scales())
        assert cache.same(start)
        assert bool(torch.isnan(out[[0, 1, 3]]).all()) and bool((out[2] == 0).all())


@pytest.mark.parametrize("nq", [4, 8])
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_small_and_large_values_in_f32(torch, ctx, nq, size):
    """f32 results over values far from 1, by the roundings of f32 arithmetic. At 1e30 check_out's bounds scale with the
    values. At 1e-30 weights have 6.7e5 units only (test_small_and_large_values); beside those attend's bound."""
    import attn_ref as ref
    import q8_ref
    import raster_amd

    print(f"[gpu] q8 size in f32 {size} {nq}", flush=True)
    n, nkv, hd = 200, 2, 64
    cache = q8_ref.Cache(5, nkv, hd, [n], 16, [n])
    g = torch.Generator(device="cuda").manual_seed(2)
    cache.append("v", 0, 0, torch.randn((n, nkv, hd), generator=g, device="cuda") * size)
    q = torch.randn((1, nq * hd), generator=g, device="cuda")
    out = raster_amd.paged_attention(ctx, q, None, None, cache.k, cache.v, cache.table,
                                     torch.tensor([n], dtype=torch.int32, device="cuda"), nq, nkv, hd, 0.0, hd ** -0.5,
                                     max_len=n, **cache.scales())
    qd = q.double().view(1, nq, hd)
    if size > 1:
        check_out(torch, ref, out, qd, cache, [n], 0, nq, nkv, hd, hd ** -0.5, 0, 0)
        return
    keys, values = cache.values("k", 0, n), cache.values("v", 0, n)
    step = 0.5 / 0x7F7F7C * (1 + 2.0 ** -20)
    see = torch.ones((1, n), dtype=torch.bool, device="cuda")
    for h in range(nq):
        kv = h // (nq // nkv)
        qh, kh, vh = qd[0, h:h + 1], keys[:, kv], values[:, kv]
        scales = cache.vs[cache._mine(0, n)].reshape(-1, nkv)[:, kv].double().repeat_interleave(16)[:n]
        # (in units of the values, so that attend's 1e-30 for results of 0 counts for nothing)
        want, lse, bound = ref.attend(qh, kh, vh / size, hd ** -0.5, see, ref.HALF[torch.float32], 2.0 ** -22)
        p = torch.softmax(qh @ kh.T * hd ** -0.5, 1)[0]
        off = step * qh.abs().max() * kh.abs().sum(1).max() * hd ** -0.5
        units = 0.5 / 6.7e5 * (p * scales).max() / size * (vh / scales[:, None]).abs().sum(0)
        got = out[0, h * hd:(h + 1) * hd].double() / size
        assert bool(((got - want[0]).abs() <= bound[0] + 2 * off * (p @ vh.abs()) / size + units).all())
