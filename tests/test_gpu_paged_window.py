"""rq_paged_attention_window over f32 and bf16 pages against 64 bits (attn_ref.py states the tolerances)."""
import pytest

from test_gpu_paged import THETA, ctx, fill, gather, make, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu

# activations, pages, heads, KV heads, head_dim, page, cached rows
CASES = [
    ("f32", "f32", 16, 16, 128, 16, [128, 0, 31, 32, 33]),
    ("f32", "f32", 8, 2, 64, 32, [7, 700, 255, 256, 257]),
    ("f32", "f32", 6, 2, 40, 16, [100, 3]),
    ("f32", "f32", 4, 1, 256, 16, [300, 40]),
    ("f32", "bf16", 8, 2, 128, 16, [0, 1, 15, 16, 17, 513]),
    ("f32", "bf16", 8, 4, 256, 16, [130]),
    ("f32", "bf16", 5, 1, 8, 16, [130, 4]),
    ("bf16", "bf16", 32, 8, 128, 16, [2500, 77, 0, 1024, 9000]),
    ("bf16", "bf16", 64, 2, 64, 128, [300, 5000]),
    ("bf16", "bf16", 3, 3, 80, 16, [90, 12]),
    ("bf16", "bf16", 2, 1, 248, 16, [400]),
]


@pytest.mark.parametrize("act,cache,nq,nkv,hd,page,lens", CASES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 17), (64, 0), (1000, 4)])
@pytest.mark.parametrize("mode", ["append", "read"])
def test_window(torch, ctx, act, cache, nq, nkv, hd, page, lens, window, sinks, mode):  # noqa: F811
    import attn_ref as ref
    import raster_amd

    print(f"[gpu] paged window {act}/{cache} {nq}/{nkv}x{hd} page={page} {lens} {window}+{sinks} {mode}", flush=True)
    add = mode == "append"
    lens = lens + [-1]
    n = len(lens)
    g, table, kp, vp, (q, k, v) = make(torch, hd + sum(lens), act, cache, nq, nkv, hd, [x + 1 for x in lens], page, n)
    fill(torch, g, kp, vp, table, lens)
    # what no query sees is gone: NaN, and no page where all rows of it are
    for b, m in enumerate(lens):
        gone = [r for r in range(max(m, 0)) if m + add - 1 - r >= window and r >= sinks]
        for r in gone:
            at = (int(table[b, r // page]), r % page)
            kp[at], vp[at] = float("nan"), float("inf")
        for i in range(-(-max(m, 0) // page)):
            if (i + 1) * page <= m and all(r in set(gone) for r in range(i * page, (i + 1) * page)):
                table[b, i] = -1
    lost = table.clone()
    k0, v0, t0 = kp.clone(), vp.clone(), table.clone()
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scale = hd ** -0.5
    out = raster_amd.paged_attention(ctx, q, k if add else None, v if add else None, kp, vp, lost, lt, nq, nkv, hd,
                                     THETA, scale, max_len=max(lens) + 1, window=window, sinks=sinks)
    pos = torch.tensor(lens, device="cuda")
    rq = ref.rope(q.double().view(n, nq, hd), pos, THETA)
    half, hq = ref.HALF[q.dtype], 2.0 ** -8 if act == "bf16" else 2.0 ** -22
    for b, m in enumerate(lens):
        if m < 0 or m + add == 0:
            assert bool((out[b] == 0).all())
            continue
        if add:
            at = (int(t0[b, m // page]), m % page)
            k0[at], v0[at] = kp[at], vp[at]
            assert bool(torch.isfinite(kp[at]).all()) and torch.equal(vp[at], v[b].to(vp.dtype))
        j = torch.arange(m + add, device="cuda")
        j = j[(m + add - 1 - j < window) | (j < sinks)]
        pages = t0[b].long()[j // page]
        keys, values = (p[pages, j % page].double().view(-1, nkv, hd) for p in (kp, vp))
        see = torch.ones((1, len(j)), dtype=torch.bool, device="cuda")
        for h in range(nq):
            i = h // (nq // nkv)
            want, _, bound = ref.attend(rq[b, h:h + 1], keys[:, i], values[:, i], scale, see, half, hq)
            got = out[b, h * hd:(h + 1) * hd].double()
            assert bool(((got - want[0]).abs() <= bound[0]).all()), (b, h, float(((got - want[0]).abs() / bound).max()))
    assert torch.equal(kp.nan_to_num(7.0), k0.nan_to_num(7.0)) and torch.equal(vp.nan_to_num(7.0), v0.nan_to_num(7.0))


def test_a_window_of_everything_is_none(torch, ctx):  # noqa: F811
    import raster_amd

    nq, nkv, hd, lens = 8, 2, 128, [700, 3000, 9]
    print("[gpu] paged window of everything", flush=True)
    g, table, kp, vp, (q, _, _) = make(torch, 3, "f32", "f32", nq, nkv, hd, lens, 16, 3)
    fill(torch, g, kp, vp, table, lens)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    outs = [raster_amd.paged_attention(ctx, q, None, None, kp, vp, table, lt, nq, nkv, hd, THETA, hd ** -0.5,
                                       max_len=3000, **see)
            for see in ({}, dict(window=3000), dict(window=2990, sinks=10), dict(window=0, sinks=5), dict(window=None))]
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_graphs_follow_the_lengths(torch, ctx):  # noqa: F811
    """A captured windowed step, replayed as the lengths grow past the window."""
    import raster_amd

    nq, nkv, hd, n = 8, 2, 64, 2
    print("[gpu] paged window graphs", flush=True)
    g, table, kp, vp, (q, k, v) = make(torch, 8, "f32", "f32", nq, nkv, hd, [400, 400], 16, n)
    fill(torch, g, kp, vp, table, [300, 300])
    lt = torch.tensor([40, 290], dtype=torch.int32, device="cuda")

    def call():
        return raster_amd.paged_attention(ctx, q, k, v, kp, vp, table, lt, nq, nkv, hd, THETA, hd ** -0.5, max_len=400,
                                          window=50, sinks=4)

    call()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = call()
    for step in range(20):
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(call(), out)
        lt += 1
