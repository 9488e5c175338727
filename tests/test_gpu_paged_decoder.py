"""The operators of prompts and pages together, as a serving loop uses them: packed
prompts through decoder layers, forks, batched decode steps, pages freed and
compacted, prompts that go on, and a captured step. Every token's output is
compared with the C oracle's decoder layer over that token's own history.

Bar: max|y - ref| < 2e-2 max|ref|, the decode step's 1e-3 (test_gpu_decoder.py) times 20.
A weight exp(s) of the softmax errs by the absolute error of its score s = q.k, which
is |s| times the relative error of q and k; that is the decode step's at the same q, but its
cached keys are drawn with rms 1, where these keys are the layers' own, of rms 20 (20.1 and
20.5 in the two layers). The operators by themselves are held to their roundings in
test_gpu_paged.py and test_gpu_prompt.py."""
import numpy as np
import pytest

from raster_amd import workloads as wl

pytestmark = pytest.mark.gpu
TOL = 2e-2
CFG = dict(wl.DECODER, d=512, n_q=8, n_kv=2, head_dim=64, ffn=1024, cached=0)


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


@pytest.fixture(scope="module")
def weights():
    return wl.decoder_weights(CFG, seed=5)[0]


class History:
    """A sequence on the oracle: every layer's rows, token by token."""

    def __init__(self, orc, weights, other=None):
        self.orc, self.weights = orc, weights
        width = CFG["n_kv"] * CFG["head_dim"]
        empty = [np.zeros((0, width), np.float32)] * len(weights)
        self.k, self.v = (list(other.k), list(other.v)) if other else (list(empty), list(empty))

    def token(self, x):
        for i, L in enumerate(self.weights):
            n = len(self.k[i]) + 1
            kc, vc = (np.concatenate([c[i], np.zeros((1, c[i].shape[1]), np.float32)]) for c in (self.k, self.v))
            x, kc, vc = self.orc.decoder_layer(x, L["weights"], L["gain1"], L["gain2"], kc, vc, CFG["d"], CFG["n_q"],
                                               CFG["n_kv"], CFG["head_dim"], CFG["ffn"], n, CFG["eps"], CFG["theta"])
            self.k[i], self.v[i] = kc.reshape(n, -1), vc.reshape(n, -1)
        return x


def close(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape and np.all(np.isfinite(got))
    assert np.max(np.abs(got - want)) < TOL * np.max(np.abs(want))


class Run:
    def __init__(self, torch, ctx, orc, weights, fused, max_seqs):
        import raster_amd
        from raster_amd.decoder import DecoderLayer

        self.torch, self.orc, self.weights = torch, orc, weights
        self.layers = [DecoderLayer(ctx, L["weights"], L["gain1"], L["gain2"], CFG["d"], CFG["n_q"], CFG["n_kv"],
                                    CFG["head_dim"], CFG["ffn"], CFG["eps"], CFG["theta"], fused=fused) for L in weights]
        self.cache = raster_amd.PagedCache(ctx, len(weights), 40, CFG["n_kv"], CFG["head_dim"], max_seqs=max_seqs,
                                           seq_pages=8)
        self.rng, self.hist = np.random.default_rng(11), {}

    def x(self, rows):
        return self.rng.standard_normal((rows, CFG["d"])).astype(np.float32)

    def add(self):
        s = self.cache.add()
        self.hist[s] = History(self.orc, self.weights)
        return s

    def fork(self, s):
        n = self.cache.fork(s)
        self.hist[n] = History(self.orc, self.weights, self.hist[s])
        return n

    def free(self, s):
        self.cache.free(s)
        del self.hist[s]

    def prefill(self, seqs, lens):
        print(f"[gpu] prefill {seqs} {lens}", flush=True)
        x = self.x(sum(lens))
        self.cache.reserve(seqs, lens)
        cu = self.torch.from_numpy(np.cumsum([0] + lens).astype(np.int32)).cuda()
        h = self.torch.from_numpy(x).cuda()
        for i, layer in enumerate(self.layers):
            h = layer.prefill(h, cu, self.cache, i, seqs, lens)
        self.cache.advance(seqs, lens)
        owner = [s for s, n in zip(seqs, lens) for _ in range(n)]
        close(h.cpu(), np.stack([self.hist[s].token(r) for s, r in zip(owner, x)]))

    def step(self, h, view):
        for i, layer in enumerate(self.layers):
            h = layer.step_paged(h, self.cache, i, view)
        return h

    def decode(self, seqs):
        print(f"[gpu] decode {seqs}", flush=True)
        x = self.x(len(seqs))
        self.cache.reserve(seqs, 1)
        h = self.step(self.torch.from_numpy(x).cuda(), self.cache.view(seqs))
        self.cache.advance(seqs, 1)
        close(h.cpu(), np.stack([self.hist[s].token(r) for s, r in zip(seqs, x)]))

    def check_rows(self):
        for i in range(len(self.layers)):
            for s, want in self.hist.items():
                k, v = self.cache.rows(i, [s])
                close(k.cpu(), want.k[i])
                close(v.cpu(), want.v[i])

    def close(self):
        for layer in self.layers:
            layer.destroy()


@pytest.mark.parametrize("fused", [True, False], ids=["fused", "unfused"])
def test_serving_loop(torch, ctx, orc, weights, fused):
    r = Run(torch, ctx, orc, weights, fused, 6)
    a, b, c = r.add(), r.add(), r.add()
    r.prefill([a, b, c], [37, 1, 18])
    for _ in range(2):
        r.decode([a, c, b])
    d = r.fork(a)  # shares three pages, the last part-filled
    e = r.fork(a)
    for _ in range(10):  # a, d and e go apart, over the page's end
        r.decode([e, a, d])
    r.free(b)
    r.free(a)
    used = r.cache.compact()
    assert used == 40 - r.cache.free_pages() and max(max(p) for p in r.cache._pages.values()) == used - 1
    r.prefill([d, c], [5, 20])  # prompts that go on
    f = r.add()
    r.prefill([f], [16])  # ends with its page
    r.decode([c, d, e, f])
    r.check_rows()
    r.close()


def test_more_sequences_than_the_fused_linears_take(torch, ctx, orc, weights):
    r = Run(torch, ctx, orc, weights, True, 18)
    first = r.add()
    r.prefill([first], [17])
    seqs = [first] + [r.fork(first) for _ in range(16)]
    r.decode(seqs)
    r.decode(seqs[::-1])
    r.close()


@pytest.mark.parametrize("fused", [True, False], ids=["fused", "unfused"])
def test_captured_step_follows_the_cache(torch, ctx, orc, weights, fused):
    """One captured step over all slots: replays with sequences added, forked, freed and
    moved between them."""
    r = Run(torch, ctx, orc, weights, fused, 5)
    a, b = r.add(), r.add()
    r.prefill([a, b], [15, 30])
    xin = torch.zeros((5, CFG["d"]), device="cuda")
    view = r.cache.view()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r.cache.reserve([a, b], 1)
        r.cache.sync()
        r.step(xin, view)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y = r.step(xin, view)
    for i in range(6):
        seqs = sorted(r.hist)
        print(f"[gpu] replay {i} {seqs}", flush=True)
        x = r.x(len(seqs))
        r.cache.reserve(seqs, 1)
        r.cache.sync()
        xin.zero_()
        xin[torch.tensor(seqs, device="cuda")] = torch.from_numpy(x).cuda()
        g.replay()
        torch.cuda.synchronize()
        r.cache.advance(seqs, 1)
        close(y.cpu()[seqs], np.stack([r.hist[q].token(t) for q, t in zip(seqs, x)]))
        if i == 1:
            r.fork(b)
        elif i == 3:
            r.free(a)
            r.cache.compact()
            r.prefill([r.add()], [21])
        _ = torch.ones(16, device="cuda").sum().item()
    r.check_rows()
    r.close()


def test_prefill_refuses_another_batch_and_rows_without_pages(torch, ctx, orc, weights):
    r = Run(torch, ctx, orc, weights, False, 3)
    a, b = r.add(), r.add()
    x, cu = torch.zeros((9, CFG["d"]), device="cuda"), torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    for seqs, lens in (([a], [4, 5]), ([a, b], [9]), ([a, b], [4, 4]), ([a, b, a], [4, 4, 1])):
        with pytest.raises(ValueError):
            r.layers[0].prefill(x, cu, r.cache, 0, seqs, lens)
    with pytest.raises(ValueError):
        r.layers[0].prefill(x, cu, r.cache, 0, [a, 7], [4, 5])
    # nothing reserved: NaN, and nothing is written
    out = r.layers[0].prefill(x, cu, r.cache, 0, [a, b], [4, 5])
    assert bool(torch.isnan(out).all()) and not bool(r.cache.data.any())
    out = r.layers[0].step_paged(x[:2].contiguous(), r.cache, 0, r.cache.view([a, b]))
    assert bool(torch.isnan(out).all()) and not bool(r.cache.data.any())
    with pytest.raises(ValueError):
        r.cache.advance([a, b], [4, 5])
    r.close()


def test_fork_after_rows_reserved_ahead(torch, ctx, orc, weights):
    """Room reserved, then a fork, then steps of both without another reservation: each writes to pages of
    its own. Without the room, a step after a fork is refused."""
    r = Run(torch, ctx, orc, weights, True, 3)
    a = r.add()
    r.prefill([a], [18])
    r.cache.reserve([a], 5)
    b = r.fork(a)
    for _ in range(3):
        x = r.x(2)
        h = r.step(torch.from_numpy(x).cuda(), r.cache.view([a, b]))
        r.cache.advance([a, b], 1)
        close(h.cpu(), np.stack([r.hist[s].token(t) for s, t in zip([a, b], x)]))
    r.check_rows()
    c = r.fork(b)
    x = torch.zeros((2, CFG["d"]), device="cuda")
    for seqs in ([a, b], [a, c]):
        with pytest.raises(ValueError):
            r.step(x, r.cache.view(seqs))
    with pytest.raises(ValueError):
        r.layers[0].prefill(x, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), r.cache, 0, [c], [2])
    r.check_rows()  # nothing was written
    r.decode([a, b, c])
    r.close()


@pytest.mark.parametrize("cache_type", ["bf16", "f32"])
def test_prefill_does_not_depend_on_the_rest_of_the_batch(torch, ctx, weights, cache_type):
    """A fresh prompt beside another fresh one and beside one that goes on: the same rows in the same products,
    so the same bits, in the outputs and in the pages; over bf16 pages too, where keys are attended as stored."""
    import ctypes as C

    import raster_amd
    from raster_amd import _lib
    from raster_amd.decoder import DecoderLayer

    layers = [DecoderLayer(ctx, L["weights"], L["gain1"], L["gain2"], CFG["d"], CFG["n_q"], CFG["n_kv"],
                           CFG["head_dim"], CFG["ffn"], CFG["eps"], CFG["theta"], fused=False) for L in weights]
    g = torch.Generator(device="cuda").manual_seed(2)
    n, past = 70, 16
    x, first = (torch.randn((rows, CFG["d"]), generator=g, device="cuda") for rows in (2 * n, past))
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    tiles = []
    for rows_k in (2 * n, 2 * n + past):  # (one kernel for both: another would add in another order)
        p, t = _lib.Prompt(_lib.RQ_F32, 2, 2 * n, rows_k, CFG["n_q"], CFG["n_kv"], CFG["head_dim"], 16, 16, 1, 0.125), C.c_int()
        _lib.call("rq_prompt_attention_tile", ctx.handle, C.byref(p), C.byref(t))
        tiles.append(t.value)
    assert tiles[0] == tiles[1]
    got = []
    for goes_on in (False, True):
        print(f"[gpu] prefill over {cache_type} pages, goes on: {goes_on}", flush=True)
        cache = raster_amd.PagedCache(ctx, len(layers), 40, CFG["n_kv"], CFG["head_dim"], max_seqs=3, seq_pages=8,
                                      dtype={"bf16": torch.bfloat16, "f32": torch.float32}[cache_type])
        a, b = cache.add(), cache.add()
        if goes_on:
            cache.reserve([b], past)
            h = first
            for i, layer in enumerate(layers):
                h = layer.prefill(h, torch.tensor([0, past], dtype=torch.int32, device="cuda"), cache, i, [b], [past])
            cache.advance([b], past)
        cache.reserve([a, b], n)
        h = x
        for i, layer in enumerate(layers):
            h = layer.prefill(h, cu, cache, i, [a, b], [n, n])
            got.append(h[:n].clone())
        cache.advance([a, b], n)
        got += [t for i in range(len(layers)) for t in cache.rows(i, [a])]
    half = len(got) // 2
    assert all(torch.equal(s, t) for s, t in zip(got[:half], got[half:]))
    for layer in layers:
        layer.destroy()
