"""rq_paged_attention, rq_pages_append and rq_pages_copy against 64 bits
(attn_ref.py states the tolerances)."""
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


def make(torch, seed, act, cache, nq, nkv, hd, need, page, rows):
    """A cache for sequences of `need` rows in shuffled pages (NaN where nothing is
    stored yet), and `rows` rows of q, k, v as columns of one array."""
    ty = {"f32": torch.float32, "bf16": torch.bfloat16}
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-n // page) for n in need]
    total = sum(pages) + 2
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(need), max(pages) + 1), 2 ** 30, dtype=torch.int32)
    for b, n in enumerate(pages):
        table[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    kp, vp = (torch.full((total, page, nkv * hd), float("nan"), dtype=ty[cache], device="cuda") for _ in range(2))
    qkv = torch.randn((rows, (nq + 2 * nkv) * hd), generator=g, device="cuda").to(ty[act])
    return g, table.cuda(), kp, vp, qkv.split([nq * hd, nkv * hd, nkv * hd], 1)


def fill(torch, g, kp, vp, table, lens):
    page = kp.shape[1]
    for b, n in enumerate(lens):
        for i in range(0, max(n, 0), page):
            m = min(page, n - i)
            for p in (kp, vp):
                p[int(table[b, i // page]), :m] = torch.randn((m, p.shape[2]), generator=g, device="cuda").to(p.dtype)


def gather(p, table, b, n):
    return p[table[b, :-(-n // p.shape[1])].long()].reshape(-1, p.shape[2])[:n]


# activations, pages, heads, KV heads, head_dim, page, cached rows
CASES = [
    ("f32", "f32", 4, 4, 128, 16, [0]),
    ("f32", "f32", 16, 16, 128, 16, [128, 0, 31, 32, 33]),
    ("f32", "f32", 8, 2, 64, 32, [7, 700, 255, 256, 257]),
    ("f32", "f32", 6, 2, 40, 16, [100, 3]),
    ("f32", "f32", 4, 1, 256, 16, [300, 40]),
    ("f32", "f32", 2, 2, 136, 16, [77]),
    ("f32", "bf16", 8, 2, 128, 16, [0, 1, 15, 16, 17, 513]),
    ("f32", "bf16", 4, 4, 64, 64, [1000]),
    ("f32", "bf16", 8, 4, 256, 16, [130]),
    ("f32", "bf16", 2, 1, 200, 32, [130, 4]),
    ("f32", "bf16", 5, 1, 8, 16, [130, 4]),
    ("bf16", "bf16", 32, 8, 128, 16, [2500, 77, 0, 1024]),
    ("bf16", "bf16", 64, 2, 64, 128, [300, 5000]),  # 32 heads a KV head: two head tiles
    ("bf16", "bf16", 17, 1, 128, 16, [40]),
    ("bf16", "bf16", 3, 3, 80, 16, [90, 12]),
    ("bf16", "bf16", 2, 1, 248, 16, [400]),
]


@pytest.mark.parametrize("act,cache,nq,nkv,hd,page,lens", CASES)
@pytest.mark.parametrize("mode", ["append", "read", "no_rope"])
def test_paged_attention(torch, ctx, act, cache, nq, nkv, hd, page, lens, mode):
    import attn_ref as ref
    import raster_amd

    print(f"[gpu] paged {act}/{cache} {nq}/{nkv}x{hd} page={page} {lens} {mode}", flush=True)
    add = mode != "read"
    lens = lens + [-1]  # an idle slot
    n = len(lens)
    g, table, kp, vp, (q, k, v) = make(torch, hd + sum(lens), act, cache, nq, nkv, hd, [x + 1 for x in lens], page, n)
    fill(torch, g, kp, vp, table, lens)
    k0, v0 = kp.clone(), vp.clone()
    theta, scale = 0.0 if mode == "no_rope" else THETA, hd ** -0.5
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = raster_amd.paged_attention(ctx, q, k if add else None, v if add else None, kp, vp, table, lt, nq, nkv, hd,
                                     theta, scale, max_len=max(lens) + 1)
    pos = torch.tensor(lens, device="cuda")
    rq, rk = (ref.rope(x.double().view(n, -1, hd), pos, THETA) if theta else x.double().view(n, -1, hd)
              for x in (q, k))
    half, hq = ref.HALF[q.dtype], 2.0 ** -8 if act == "bf16" else 2.0 ** -22
    for b, m in enumerate(lens):
        if m < 0:
            assert bool((out[b] == 0).all())
            continue
        if add:  # the new row: rotated in f32 (two products and their sum), rounded once
            page_id, r = int(table[b, m // page]), m % page
            got = kp[page_id, r].double().view(nkv, hd)
            tol = (ref.HALF[kp.dtype] + 2.0 ** -21) * (rk[b].abs() + 1)
            assert bool(((got - rk[b]).abs() <= tol).all())
            assert torch.equal(vp[page_id, r], v[b].to(vp.dtype))
            k0[page_id, r], v0[page_id, r] = kp[page_id, r], vp[page_id, r]
        if m + add == 0:
            assert bool((out[b] == 0).all())
            continue
        keys, values = (gather(p, table, b, m + add).double().view(-1, nkv, hd) for p in (kp, vp))
        see = torch.ones((1, m + add), dtype=torch.bool, device="cuda")
        for h in range(nq):
            j = h // (nq // nkv)
            want, _, bound = ref.attend(rq[b, h:h + 1], keys[:, j], values[:, j], scale, see, half, hq)
            got = out[b, h * hd:(h + 1) * hd].double()
            assert bool(((got - want[0]).abs() <= bound[0]).all()), (b, h, float(((got - want[0]).abs() / bound).max()))
    # nothing else was written
    assert torch.equal(kp.nan_to_num(7.0), k0.nan_to_num(7.0)) and torch.equal(vp.nan_to_num(7.0), v0.nan_to_num(7.0))


def test_any_split_gives_the_same_within_rounding(torch, ctx):
    """max_len only sizes the split: a larger one changes sums' order, nothing else."""
    import raster_amd

    nq, nkv, hd, lens = 8, 2, 128, [700, 3000, 9]
    print("[gpu] paged max_len", flush=True)
    g, table, kp, vp, (q, _, _) = make(torch, 3, "f32", "f32", nq, nkv, hd, lens, 16, 3)
    fill(torch, g, kp, vp, table, lens)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    outs = [raster_amd.paged_attention(ctx, q, None, None, kp, vp, table, lt, nq, nkv, hd, THETA, hd ** -0.5, max_len=m)
            for m in (3000, 50000, 10 ** 6)]
    for o in outs[1:]:
        assert float((o - outs[0]).abs().max()) <= 1e-5 * float(outs[0].abs().max())
    again = raster_amd.paged_attention(ctx, q, None, None, kp, vp, table, lt, nq, nkv, hd, THETA, hd ** -0.5,
                                       max_len=3000)
    assert torch.equal(again, outs[0])


def test_bad_pages_and_lengths(torch, ctx):
    """Page numbers outside the cache and sequences past max_len or their table: NaN, the
    other sequences as ever, nothing written."""
    import raster_amd

    nq, nkv, hd, lens = 4, 2, 64, [40, 50, 60, 70]
    print("[gpu] paged bad pages", flush=True)
    g, table, kp, vp, (q, k, v) = make(torch, 5, "f32", "f32", nq, nkv, hd, [n + 1 for n in lens], 16, 4)
    fill(torch, g, kp, vp, table, lens)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    args = (nq, nkv, hd, THETA, hd ** -0.5)
    good = raster_amd.paged_attention(ctx, q, k, v, kp.clone(), vp.clone(), table, lt, *args)
    bad = table.clone()
    bad[0, 1] = kp.shape[0]      # read
    bad[1, 3] = -1               # appended (row 50 is in page 3)
    far = lt.clone()
    far[3] = 10 ** 6             # past the table
    k1, v1 = kp.clone(), vp.clone()
    out = raster_amd.paged_attention(ctx, q, k, v, k1, v1, bad, far, *args)
    for b in (0, 1, 3):
        assert bool(torch.isnan(out[b]).all())
    assert torch.equal(out[2], good[2])
    wrote = [(int(table[b, lens[b] // 16]), lens[b] % 16) for b in (0, 2)]
    for p, was in ((k1, kp), (v1, vp)):
        same = (p.nan_to_num(7.0) == was.nan_to_num(7.0)).all(-1)
        for at in wrote:
            same[at] = True
        assert bool(same.all())
    out = raster_amd.paged_attention(ctx, q, k, v, kp.clone(), vp.clone(), table, lt, *args, max_len=61)
    assert torch.equal(out[:3], good[:3]) and bool(torch.isnan(out[3]).all())


@pytest.mark.parametrize("act,cache,nq,nkv,hd,page,lens,past", [
    ("f32", "f32", 4, 2, 128, 16, [37, 0, 1, 16], [0, 5, 15, 1000]),
    ("f32", "bf16", 3, 1, 40, 32, [33, 2], [31, 100000]),
    ("bf16", "bf16", 32, 8, 128, 16, [300, 1, 77], [0, 128, 5]),
    ("bf16", "bf16", 2, 2, 8, 16, [5], [3]),
    ("bf16", "bf16", 2, 1, 256, 64, [70], [0]),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_append(torch, ctx, act, cache, nq, nkv, hd, page, lens, past, in_place):
    import attn_ref as ref
    import raster_amd

    print(f"[gpu] append {act}/{cache} {nq}/{nkv}x{hd} {lens} {past}", flush=True)
    n, tail = sum(lens), 3
    lens2, past2 = lens + [2], past + [-1]  # a sequence left out, and rows of none behind it
    _, table, kp, vp, (q, k, v) = make(torch, n, act, cache, nq, nkv, hd,
                                       [a + b for a, b in zip(lens, past)] + [1], page, n + 2 + tail)
    cu = torch.tensor([sum(lens2[:i]) for i in range(len(lens2) + 1)], dtype=torch.int32, device="cuda")
    pt = torch.tensor(past2, dtype=torch.int32, device="cuda")
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    qo, ko = (q, k) if in_place else (torch.full_like(q, 7.0), torch.full_like(k, 7.0))
    raster_amd.pages_append(ctx, q, k, v, kp, vp, table, cu, pt, nq, nkv, hd, THETA, q_out=qo, k_out=ko)
    seen = torch.zeros(kp.shape[:2], dtype=torch.bool, device="cuda")
    at = 0
    for b, (m, p0) in enumerate(zip(lens, past)):
        if m == 0:
            continue
        pos = torch.arange(p0, p0 + m, device="cuda")
        wq, wk = (ref.rope(x[at:at + m].double().view(m, -1, hd), pos, THETA).view(m, -1) for x in (q0, k0))
        for got, want in ((qo[at:at + m], wq), (ko[at:at + m], wk)):
            tol = (ref.HALF[got.dtype] + 2.0 ** -21) * (want.abs() + 1)
            assert bool(((got.double() - want).abs() <= tol).all())
        pages, r = table[b].long()[pos // page], pos % page
        stored = kp[pages, r].double()
        assert bool(((stored - wk).abs() <= (ref.HALF[kp.dtype] + 2.0 ** -21) * (wk.abs() + 1)).all())
        assert torch.equal(vp[pages, r], v0[at:at + m].to(vp.dtype))
        seen[pages, r] = True
        at += m
    assert torch.equal(qo[n:], q0[n:] if in_place else torch.full_like(qo[n:], 7.0))
    assert torch.equal(ko[n:], k0[n:] if in_place else torch.full_like(ko[n:], 7.0))
    assert torch.equal(v, v0) and bool(torch.isnan(kp[~seen]).all()) and bool(torch.isnan(vp[~seen]).all())


def test_append_without_a_page(torch, ctx):
    import raster_amd

    print("[gpu] append without a page", flush=True)
    _, table, kp, vp, (q, k, v) = make(torch, 1, "f32", "f32", 2, 2, 64, [40], 16, 70)
    table[0, 1] = 10 ** 6
    cu = torch.tensor([0, 70], dtype=torch.int32, device="cuda")
    past = torch.zeros(1, dtype=torch.int32, device="cuda")
    qo, ko = raster_amd.pages_append(ctx, q, k, v, kp, vp, table, cu, past, 2, 2, 64, THETA)
    lost = torch.zeros(70, dtype=torch.bool, device="cuda")
    lost[16:32] = lost[48:] = True  # the bad page, and what the table (4 pages) does not reach or has none for
    ok = ~lost
    assert bool(torch.isnan(qo[lost]).all()) and bool(torch.isnan(ko[lost]).all())
    assert bool(torch.isfinite(qo[ok]).all()) and int(torch.isfinite(kp).all(-1).sum()) == int(ok.sum())


@pytest.mark.parametrize("planes,pages,page,width,n", [(1, 2, 16, 8, 1), (6, 40, 16, 72, 17), (4, 700, 16, 64, 300),
                                                       (3, 10, 16, 1032, 5)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_copy(torch, ctx, planes, pages, page, width, n, t):
    import raster_amd

    print(f"[gpu] copy {planes}x{pages}x{page}x{width} {n} {t}", flush=True)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[t]
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn((planes, pages, page, width), generator=g, device="cuda").to(dt)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = order[:n], order[n:2 * n]
    if n > 2:
        src[1] = src[0]  # one page to two places
    want = x.clone()
    want[:, dst] = x[:, src]
    raster_amd.pages_copy(ctx, x, src, dst)
    assert torch.equal(x, want)


def test_graphs(torch, ctx):
    """Attention with its append captured, replayed on another stream between eager work."""
    import raster_amd

    nq, nkv, hd, lens = 8, 2, 128, [300, 2000]
    print("[gpu] paged graphs", flush=True)
    g, table, kp, vp, (q, k, v) = make(torch, 8, "bf16", "bf16", nq, nkv, hd, [n + 1 for n in lens], 16, 2)
    fill(torch, g, kp, vp, table, lens)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def call():
        return raster_amd.paged_attention(ctx, q, k, v, kp, vp, table, lt, nq, nkv, hd, THETA, hd ** -0.5, max_len=2001)

    want = call().clone()
    torch.cuda.synchronize()
    gr, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(gr, stream=s):
        out = call()
    other = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(other):
            gr.replay()
        again = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(again, want)


@pytest.mark.parametrize("batch", [65, 300, 5000])
def test_append_of_many_sequences(torch, ctx, batch):
    import raster_amd

    print(f"[gpu] append {batch} sequences", flush=True)
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 3, (batch,), generator=gen)
    lens[batch // 3] = 40
    n = int(lens.sum())
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
    past = torch.randint(0, 17, (batch,), generator=gen)
    table = torch.randperm(4 * batch, generator=gen).int().view(batch, 4)
    kp, vp = (torch.zeros((4 * batch, 16, 64), device="cuda") for _ in range(2))
    q, k, v = (torch.randn((n, 64), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
               for i in range(3))
    qo, ko = raster_amd.pages_append(ctx, q, k, v, kp, vp, table.cuda(), cu.int().cuda(), past.int().cuda(), 1, 1, 64,
                                     0.0)
    owner = torch.repeat_interleave(torch.arange(batch), lens)
    pos = past[owner] + torch.arange(n) - cu[owner]
    at = (table[owner, pos // 16].long() * 16 + pos % 16).cuda()
    assert torch.equal(qo, q) and torch.equal(ko, k)
    for p, x in ((kp, k), (vp, v)):
        want = torch.zeros_like(p).view(-1, 64)
        want[at] = x
        assert torch.equal(p.view(-1, 64), want)


def test_offsets_past_32_bits(torch, ctx):
    """A cache of 2 x 2 planes of 4.3 GiB, its last pages used."""
    import raster_amd

    print("[gpu] paged offsets past 2^32", flush=True)
    nq, nkv, hd, total, used = 8, 8, 128, 140000, 64
    data = torch.empty((2, total, 16, nkv * hd), dtype=torch.bfloat16, device="cuda")
    small = torch.randn((2, used, 16, nkv * hd), generator=torch.Generator(device="cuda").manual_seed(2),
                        device="cuda").to(torch.bfloat16)
    data[:, total - used:] = small
    table = torch.randperm(used, generator=torch.Generator().manual_seed(3)).int().view(2, -1).cuda()
    lens = torch.tensor([300, 511], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn((2, nq * hd), generator=torch.Generator(device="cuda").manual_seed(4 + i),
                           device="cuda").to(torch.bfloat16) for i in range(3))
    outs = []
    for pages, first in ((small, 0), (data, total - used)):
        outs.append(raster_amd.paged_attention(ctx, q, k, v, pages[0], pages[1], table + first, lens, nq, nkv, hd, THETA,
                                               hd ** -0.5))
        cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
        raster_amd.pages_append(ctx, q, k, v, pages[0], pages[1], table + first, cu, lens - 100, nq, nkv, hd, THETA)
        raster_amd.pages_copy(ctx, pages, [first + 3, first + 40], [first + 5, first + 63])
    assert torch.equal(outs[0], outs[1]) and torch.equal(data[:, total - used:], small)


def test_append_and_copy_captured(torch, ctx):
    """The copy's page numbers belong to the graph; its host lists may change after the call."""
    import raster_amd

    print("[gpu] append and copy captured", flush=True)
    pages = torch.zeros((4, 12, 16, 128), device="cuda")
    q, k, v = (torch.zeros((20, 128), device="cuda") for _ in range(3))
    table = torch.tensor([[3, 1]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    past = torch.zeros(1, dtype=torch.int32, device="cuda")
    src, dst = [3, 1], [7, 11]
    gr, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(gr, stream=s):
        qo, ko = raster_amd.pages_append(ctx, q, k, v, pages[0], pages[1], table, cu, past, 1, 1, 128, THETA)
        raster_amd.pages_copy(ctx, pages, src, dst)
    src[:], dst[:] = [0, 0], [2, 4]
    for i in range(3):
        for j, t in enumerate((q, k, v)):
            t.copy_(torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(10 * i + j), device="cuda"))
        pages.zero_()
        past.fill_(i)
        gr.replay()
        torch.cuda.synchronize()
        want = torch.zeros_like(pages)
        wq, wk = raster_amd.pages_append(ctx, q, k, v, want[0], want[1], table, cu, past, 1, 1, 128, THETA)
        want[:, [7, 11]] = want[:, [3, 1]]
        assert torch.equal(pages, want) and torch.equal(qo, wq) and torch.equal(ko, wk)


def test_threads(torch, ctx):
    """Four host threads, each on a stream of its own, on one context."""
    import threading

    import raster_amd

    nq, nkv, hd = 8, 2, 128
    print("[gpu] paged and prompt calls of four threads", flush=True)
    work = []
    for i, lens in enumerate(([300, 2000], [17], [900, 1, 64], [4000])):
        g, table, kp, vp, (q, k, v) = make(torch, i, "bf16", "bf16", nq, nkv, hd, [n + 1 for n in lens], 16, len(lens))
        fill(torch, g, kp, vp, table, lens)
        lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
        rows = torch.randn((200 + i, (nq + 2 * nkv) * hd), generator=g, device="cuda").to(torch.bfloat16)
        pq, pk, pv = rows.split([nq * hd, nkv * hd, nkv * hd], 1)
        cu = torch.tensor([0, 100, 200 + i], dtype=torch.int32, device="cuda")
        lse = torch.empty((nq, 200 + i), device="cuda")

        def call(a=(q, k, v, kp, vp, table, lt), n=max(lens) + 1, b=(pq, pk, pv), cu=cu, lse=lse):
            x = raster_amd.paged_attention(ctx, *a, nq, nkv, hd, THETA, hd ** -0.5, max_len=n)
            y = raster_amd.prompt_attention(ctx, *b, cu, nq, nkv, hd, hd ** -0.5, lse=lse)
            return [x, y, *raster_amd.prompt_attention_bwd(ctx, y, *b, y, lse, cu, nq, nkv, hd, hd ** -0.5)]

        work.append((call, [t.clone() for t in call()]))
    torch.cuda.synchronize()
    wrong = []

    def run(call, want):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = call()
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(1)
            s.synchronize()

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong


@pytest.mark.parametrize("nq,nkv,lens", [(64, 64, [2048, 2047, 5, 0]), (64, 64, [2049, 300, 2048, 1]), (8, 8, [600, 513, 512, 40]),
                                         (8, 8, [9000, 1025, 1024, 2000])])
def test_range_sizes(torch, ctx, nq, nkv, lens):
    """Lengths at the ends of ranges of 512, 1024 and 2048 rows, by what plan_paged_attention chooses for the shape."""
    import attn_ref as ref
    import raster_amd

    print(f"[gpu] paged ranges {nq}/{nkv} {lens}", flush=True)
    hd = 64
    g, table, kp, vp, (q, k, v) = make(torch, 3, "f32", "f32", nq, nkv, hd, [n + 1 for n in lens], 16, len(lens))
    fill(torch, g, kp, vp, table, lens)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = raster_amd.paged_attention(ctx, q, k, v, kp, vp, table, lt, nq, nkv, hd, 0.0, hd ** -0.5, max_len=max(lens) + 1)
    for b, n in enumerate(lens):
        kk, vv = gather(kp, table, b, n + 1).double(), gather(vp, table, b, n + 1).double()
        see = torch.ones((1, n + 1), dtype=torch.bool, device="cuda")
        for h in range(0, nq, 7):
            at = slice(h * hd, (h + 1) * hd)
            want, _, bound = ref.attend(q[b:b + 1, at].double(), kk[:, at], vv[:, at], hd ** -0.5, see, ref.U)
            assert bool(((out[b:b + 1, at].double() - want).abs() <= bound).all()), (b, h)


@pytest.mark.parametrize("act,cache,nq,nkv,hd,page,lens", [
    ("f32", "f32", 40, 2, 128, 16, [40, 900, 0]),   # 20 heads a KV head: two head tiles
    ("f32", "f32", 33, 1, 64, 32, [300, 17]),       # three
    ("f32", "bf16", 34, 2, 256, 16, [130, 600]),
    ("f32", "bf16", 17, 1, 80, 64, [1, 2000]),
])
@pytest.mark.parametrize("mode", ["append", "read", "no_rope"])
def test_many_heads_a_kv_head_in_f32(torch, ctx, act, cache, nq, nkv, hd, page, lens, mode):
    test_paged_attention(torch, ctx, act, cache, nq, nkv, hd, page, lens, mode)


@pytest.mark.parametrize("nq,nkv,hd,lens", [(32, 8, 128, [4000, 333, 64]), (16, 2, 64, [900, 5000]), (4, 1, 256, [700]),
                                            (6, 2, 80, [1500])])
def test_bf16_over_bf16_pages_rounds_its_result_only(torch, ctx, nq, nkv, hd, lens):
    """Queries and weights enter in two bf16 terms, off by 2^-16 at most: but for that and f32 sums, a result
    is off by its own rounding, half a step. (With weights rounded to bf16 the first case is past it.)"""
    import attn_ref as ref
    import raster_amd

    print(f"[gpu] paged bf16 precision {nq}/{nkv}x{hd} {lens}", flush=True)
    n = len(lens)
    g, table, kp, vp, (q, _, _) = make(torch, hd, "bf16", "bf16", nq, nkv, hd, lens, 16, n)
    fill(torch, g, kp, vp, table, lens)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = raster_amd.paged_attention(ctx, q, None, None, kp, vp, table, lt, nq, nkv, hd, 0.0, hd ** -0.5,
                                     max_len=max(lens))
    for b, m in enumerate(lens):
        keys, values = (gather(p, table, b, m).double().view(-1, nkv, hd) for p in (kp, vp))
        see = torch.ones((1, m), dtype=torch.bool, device="cuda")
        for h in range(nq):
            j = h // (nq // nkv)
            want, _, bound = ref.attend(q[b:b + 1, h * hd:(h + 1) * hd].double(), keys[:, j], values[:, j], hd ** -0.5,
                                        see, 2.0 ** -16, 2.0 ** -16)
            err = (out[b:b + 1, h * hd:(h + 1) * hd].double() - want).abs()
            assert bool((err <= bound + ref.HALF[torch.bfloat16] * want.abs()).all()), (b, h, float((err / want.abs()).max()))
