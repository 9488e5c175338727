"""PagedCache.rows over caches of any length, type and head size."""
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


def by_index(torch, cache, seqs, lens):
    """The rows' places in the pages, from the page numbers."""
    at = [torch.tensor(cache._pages[s], dtype=torch.long)[:, None] * cache.page_size + torch.arange(cache.page_size)
          for s in seqs]
    return torch.cat([x.flatten()[:n] for x, n in zip(at, lens)]).cuda()


def of(torch, ctx, dtype, nkv, hd, page, lens, more=0):
    """A cache with sequences of `lens` rows, their pages taken in turns, filled with numbers."""
    import raster_amd

    cache = raster_amd.PagedCache(ctx, 2, sum(-(-n // page) for n in lens) + 1, nkv, hd, page, len(lens), dtype=dtype)
    seqs = [cache.add() for _ in lens]
    for i in range(2):
        for s, n in zip(seqs, lens):
            cache.reserve([s], n // 2 if i == 0 else n - n // 2)
            cache.advance([s], n // 2 if i == 0 else n - n // 2)
    g = torch.Generator(device="cuda").manual_seed(hd)
    for plane in (2, 3):  # (a part at a time: a plane's numbers are wanted in 32 bits first)
        for x in cache.data[plane].split(64):
            if dtype == torch.int8:
                x.copy_(torch.randint(-127, 128, x.shape, generator=g, device="cuda", dtype=torch.int32))
            else:
                x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
    if cache.scales is not None:
        cache.scales.uniform_(0.5, 2, generator=g)
    return cache, seqs


@pytest.mark.parametrize("dtype,nkv,hd,page", [("float16", 2, 64, 16), ("float32", 3, 12, 32), ("bfloat16", 1, 512, 16),
                                               ("float64", 2, 8, 16), ("float32", 1, 8, 1 << 17)])
def test_caches_that_no_operator_takes(torch, ctx, dtype, nkv, hd, page):
    print(f"[gpu] rows of {dtype} {nkv}x{hd} {page}", flush=True)
    cache, seqs = of(torch, ctx, getattr(torch, dtype), nkv, hd, page, [100, 7, 0, 300])
    lens = [100, 300, 0, 100]
    pick = [seqs[0], seqs[3], seqs[2], seqs[0]]
    at = by_index(torch, cache, pick, lens)
    for got, pages in zip(cache.rows(1, pick), (cache.kpages(1), cache.vpages(1))):
        assert got.dtype == pages.dtype and torch.equal(got, pages.view(-1, nkv * hd)[at])
    for got, pages in zip(cache.rows(1, pick, dtype=torch.float32), (cache.kpages(1), cache.vpages(1))):
        assert torch.equal(got, pages.view(-1, nkv * hd)[at].float())
    assert cache.rows(1, [])[0].shape == (0, nkv * hd)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("page,lens", [(16, [9000000, 5, 0, 8000001]), (65536, [17000000, 300])])
def test_rows_past_one_launch(torch, ctx, dtype, page, lens):
    print(f"[gpu] rows of {dtype} {page} {lens}", flush=True)
    cache, seqs = of(torch, ctx, getattr(torch, dtype), 1, 8, page, lens)
    at = by_index(torch, cache, seqs, lens)
    got = cache.rows(1, seqs)
    names = list(cache.layer_scales(1).values()) or [None, None]
    for x, pages, scales in zip(got, (cache.kpages(1), cache.vpages(1)), names):
        want = pages.view(-1, 8)[at]
        if scales is not None:
            want = want.float() * scales.reshape(-1, 1)[at // 16]
        assert torch.equal(x, want)


def test_rows_leaves_the_views_alone(torch, ctx):
    """A captured graph's view follows the cache from the next view() or sync() on, not from a look at its rows."""
    print("[gpu] rows and views", flush=True)
    cache, seqs = of(torch, ctx, torch.float32, 2, 64, 16, [100, 7])
    view = cache.view()
    table, lens = view.table.clone(), view.lens.clone()
    cache.free(seqs[1])
    s = cache.add()
    cache.reserve([s], 30)
    cache.advance([s], 30)
    lens2 = [30, 100]
    at = by_index(torch, cache, [s, seqs[0]], lens2)
    for got, pages in zip(cache.rows(1, [s, seqs[0]]), (cache.kpages(1), cache.vpages(1))):
        assert torch.equal(got, pages.view(-1, 128)[at])
    assert torch.equal(view.table, table) and torch.equal(view.lens, lens)
    cache.sync()
    assert not torch.equal(view.table, table) and int(view.lens[s]) == 30
