"""Decoder layers over a PagedCache in 8 bits and with a sliding window: packed prompts, prompts that go on, forks, batched
steps, pages moved, a captured step. Each layer's output is compared with the layer's own linears around attention in
64 bits over the rows as the cache holds them; the operators by themselves are held to their roundings
in test_gpu_paged_q8.py, test_gpu_paged_window.py and test_gpu_window.py.

Bar: max|y - ref| < 2e-3 max|ref|, the decode step's 1e-3 (test_gpu_decoder.py) for the linears' other order of sums,
and as much again for the weights: scores of up to a few hundred (keys of rms 20) carry errors of 2^-20 of that."""
import math

import numpy as np
import pytest

from raster_amd import workloads as wl

pytestmark = pytest.mark.gpu
TOL = 2e-3
CFG = dict(wl.DECODER, d=512, n_q=8, n_kv=2, head_dim=64, ffn=1024, cached=0)
HD, NQ, NKV = CFG["head_dim"], CFG["n_q"], CFG["n_kv"]


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


class Run:
    def __init__(self, torch, ctx, weights, dtype, window, sinks, max_seqs, fused=True):
        import raster_amd
        from raster_amd.decoder import DecoderLayer

        self.torch, self.window, self.sinks = torch, window, sinks
        self.layers = [DecoderLayer(ctx, L["weights"], L["gain1"], L["gain2"], CFG["d"], NQ, NKV, HD, CFG["ffn"],
                                    CFG["eps"], CFG["theta"], fused=fused, window=window, sinks=sinks) for L in weights]
        self.cache = raster_amd.PagedCache(ctx, len(weights), 40, NKV, HD, max_seqs=max_seqs, seq_pages=10, dtype=dtype)
        self.rng = np.random.default_rng(11)

    def x(self, rows):
        return self.torch.from_numpy(self.rng.standard_normal((rows, CFG["d"])).astype(np.float32)).cuda()

    def expect(self, li, x, seqs, lens, fused=False):
        """The layer's output for rows x, lens[b] new ones of each sequence, which are appended but not advanced over.
        Queries by the linear that the layer takes (their error would be that of scores, times keys of rms 20)."""
        import attn_ref as ref
        from raster_amd.decoder import residual_add, rms_norm

        torch, layer = self.torch, self.layers[li]
        q = (layer.w_qkv.matmul_fused(x, norm_gain=layer.g1, norm_eps=layer.eps) if fused else
             layer.w_qkv.matmul(rms_norm(torch, x, layer.g1, layer.eps)))
        q = q[:, :NQ * HD].double().view(-1, NQ, HD)
        out, at = torch.zeros((x.shape[0], NQ * HD), dtype=torch.float64, device="cuda"), 0
        for s, n in zip(seqs, lens):
            past = self.cache.length(s)
            k, v = (t.double().view(-1, NKV, HD) for t in self.cache.rows(li, [s], n))
            pos = torch.arange(past, past + n, device="cuda")
            qr = ref.rope(q[at:at + n], pos, CFG["theta"])
            j = torch.arange(past + n, device="cuda")
            see = j <= pos[:, None]
            if self.window:
                see &= (pos[:, None] - j < self.window) | (j < self.sinks)
            for h in range(NQ):
                g = h // (NQ // NKV)
                p = torch.softmax((qr[:, h] @ k[:, g].T / math.sqrt(HD)).masked_fill(~see, -torch.inf), 1)
                out[at:at + n, h * HD:(h + 1) * HD] = p @ v[:, g]
            at += n
        return layer._mlp(residual_add(x, layer.w_o.matmul(out.float())))

    def check(self, got, want, what):
        assert bool(self.torch.isfinite(got).all())
        off = float((got - want).abs().max() / want.abs().max())
        assert off < TOL, (what, off)

    def prefill(self, seqs, lens):
        print(f"[gpu] prefill {seqs} {lens}", flush=True)
        self.cache.reserve(seqs, lens)
        cu = self.torch.from_numpy(np.cumsum([0] + lens).astype(np.int32)).cuda()
        h = self.x(sum(lens))
        for i, layer in enumerate(self.layers):
            x, h = h, layer.prefill(h, cu, self.cache, i, seqs, lens)
            self.check(h, self.expect(i, x, seqs, lens), ("prefill", i))
        self.cache.advance(seqs, lens)

    def decode(self, seqs):
        print(f"[gpu] decode {seqs}", flush=True)
        self.cache.reserve(seqs, 1)
        h, view = self.x(len(seqs)), self.cache.view(seqs)
        for i, layer in enumerate(self.layers):
            x, h = h, layer.step_paged(h, self.cache, i, view)
            self.check(h, self.expect(i, x, seqs, [1] * len(seqs), layer.fused), ("step", i))
        self.cache.advance(seqs, 1)

    def rows(self, seqs):
        return [t for i in range(len(self.layers)) for t in self.cache.rows(i, seqs)]

    def close(self):
        for layer in self.layers:
            layer.destroy()


@pytest.mark.parametrize("cache,window,sinks", [("int8", None, 0), ("int8", 20, 3), ("float32", 33, 4), ("bfloat16", 16, 0)])
@pytest.mark.parametrize("fused", [True, False], ids=["fused", "unfused"])
def test_serving_loop(torch, ctx, weights, cache, window, sinks, fused):
    r = Run(torch, ctx, weights, getattr(torch, cache), window, sinks, 6, fused)
    a, b, c = (r.cache.add() for _ in range(3))
    r.prefill([a, b, c], [37, 1, 18])
    for _ in range(2):
        r.decode([a, c, b])
    before = r.rows([a])
    d = r.cache.fork(a)  # shares three pages, the last part-filled
    assert all(torch.equal(x, y) for x, y in zip(before, r.rows([d])))
    for _ in range(10):  # a and d go apart, over the page's end
        r.decode([a, d])
    # whole blocks are as they were; the one that was part-filled may have been rounded anew
    assert all(torch.equal(x[:32], y[:32]) for x, y in zip(before, r.rows([d])))
    r.cache.free(b)
    r.cache.free(a)
    before = r.rows([c, d])
    used = r.cache.compact()
    assert used == 40 - r.cache.free_pages()
    assert all(torch.equal(x, y) for x, y in zip(before, r.rows([c, d])))
    r.prefill([d, c], [5, 20])  # prompts that go on
    f = r.cache.add()
    r.prefill([f], [16])  # ends with its page, on pages used before
    r.decode([c, d, f])
    r.close()


def test_a_fork_on_int8_pages_writes_its_own(torch, ctx, weights):
    """A part-filled page is copied with its scales before either goes on: the other's rows keep their bits."""
    r = Run(torch, ctx, weights, torch.int8, None, 0, 4)
    a = r.cache.add()
    r.prefill([a], [21])
    b = r.cache.fork(a)
    before = r.rows([a])
    for _ in range(3):
        r.decode([b])
    assert all(torch.equal(x, y) for x, y in zip(before, r.rows([a])))
    r.decode([a])
    r.close()


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
def test_captured_step_follows_the_cache(torch, ctx, weights, window, sinks):
    """One captured step over all slots of an int8 cache: replays give what the same steps give uncaptured on a
    second cache, bit for bit, with sequences added, forked and freed between them."""
    runs = [Run(torch, ctx, weights, torch.int8, window, sinks, 5) for _ in range(2)]
    for r in runs:
        r.rng = np.random.default_rng(3)
        r.prefill([r.cache.add(), r.cache.add()], [15, 30])
    r, plain = runs
    xin, view = torch.zeros((5, CFG["d"]), device="cuda"), r.cache.view()

    def step(run, h, v):
        for i, layer in enumerate(run.layers):
            h = layer.step_paged(h, run.cache, i, v)
        return h

    keep = r.cache.data.clone(), r.cache.scales.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(r, xin, view)
    s.synchronize()
    r.cache.data.copy_(keep[0])
    r.cache.scales.copy_(keep[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y = step(r, xin, view)
    seqs = [0, 1]
    for i in range(6):
        x = r.x(5)
        for run in runs:
            run.cache.reserve(seqs, 1)
            run.cache.sync()
        xin.copy_(x)
        g.replay()
        want = step(plain, x, plain.cache.view())
        torch.cuda.synchronize()
        for run in runs:
            run.cache.advance(seqs, 1)
        assert torch.equal(y[seqs], want[seqs])
        assert all(torch.equal(p, q) for p, q in zip(r.rows(seqs), plain.rows(seqs)))
        if i == 1:
            seqs = [0, 1, {run.cache.fork(1) for run in runs}.pop()]
        elif i == 3:
            for run in runs:
                run.cache.free(0)
                run.cache.compact()
            seqs = seqs[1:]
        _ = torch.ones(16, device="cuda").sum().item()
    for run in runs:
        run.close()


def test_refusals(torch, ctx, weights):
    from raster_amd.decoder import DecoderLayer

    L = weights[0]
    args = (ctx, L["weights"], L["gain1"], L["gain2"], CFG["d"], NQ, NKV, HD, CFG["ffn"])
    for kw in (dict(window=-1), dict(window=4, sinks=-2)):
        with pytest.raises(ValueError):
            DecoderLayer(*args, **kw)
    r = Run(torch, ctx, weights, torch.int8, 8, 0, 2)
    with pytest.raises(ValueError):  # the step over contiguous caches has no window
        r.layers[0].step(r.x(1)[0], torch.zeros((4, NKV * HD), device="cuda"), torch.zeros((4, NKV * HD), device="cuda"), 0)
    a = r.cache.add()
    with pytest.raises(ValueError):  # nothing reserved
        r.layers[0].prefill(r.x(3), torch.tensor([0, 3], dtype=torch.int32, device="cuda"), r.cache, 0, [a], [3])
    assert not bool(r.cache.data.any()) and not bool(r.cache.scales.any())
    with pytest.raises(ValueError):
        r.cache.rows(0, [a], 1)
    k, v = r.cache.rows(0, [a])
    assert k.shape == (0, NKV * HD) and k.dtype == torch.float32 and v.shape == k.shape
    assert r.cache.rows(0, [])[0].shape == (0, NKV * HD)
    r.close()
