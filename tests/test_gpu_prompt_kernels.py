"""Which kernel a prompt runs on, and the kernel of long sequences against every head in 64 bits.

rq_prompt_attention_tile names the kernel, so that each shape below is known to reach the one that it is
for; tolerances are attn_ref.py's, as in test_gpu_prompt.py."""
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


def tile(ctx, t, nq, nkv, hd, lq, lk):
    """Queries of a workgroup of the kernel for this batch."""
    p = _lib.Prompt({"f32": _lib.RQ_F32, "bf16": _lib.RQ_BF16}[t], len(lq), sum(lq), sum(lk), nq, nkv, hd, 0x10000,
                    0x10000, 1, 0.125)
    n = C.c_int(-1)
    _lib.call("rq_prompt_attention_tile", ctx.handle, C.byref(p), C.byref(n))
    return n.value


MORE = [
    ("f32", 64, 8, 64, [300, 129, 90], [300, 129, 90]),
    ("f32", 64, 8, 56, [300, 0, 90], [310, 129, 77]),
    ("f32", 48, 4, 128, [64, 7, 33], [900, 300, 64]),  # few queries after many keys
    ("f32", 32, 8, 128, [16, 1, 31], [700, 90, 131]),
    ("f32", 32, 8, 128, [290, 300], [1900, 1300]),
    ("f32", 64, 8, 64, [64] * 8, [300] * 8),
    ("f32", 64, 8, 56, [20] * 8, [90] * 8),
]


def test_every_kernel_has_a_case(ctx):
    """The tiles that the cases here and in test_gpu_prompt.py reach, by type and padded head size."""
    from test_gpu_prompt import CASES

    seen = {(t, 64 if hd <= 64 else 128 if hd <= 128 else 256, tile(ctx, t, nq, nkv, hd, lq, lk))
            for t, nq, nkv, hd, lq, lk in CASES + MORE + [("bf16", *c) for c in LONG]}
    want = {(t, w, n) for t in ("f32", "bf16") for w in (64, 128) for n in (32, 64, 128)}
    want |= {("bf16", 256, 64), ("bf16", 256, 128), ("f32", 256, 128), ("bf16", 128, 256)}
    assert want <= seen, want - seen


@pytest.mark.parametrize("nq,nkv,hd,batch,new,keys,want", [
    (32, 8, 128, 4, 64, 4096, 32), (64, 8, 128, 4, 64, 4096, 64), (32, 8, 128, 8, 64, 2048, 64), (32, 8, 128, 8, 16, 1000, 32),
    (16, 16, 128, 8, 128, 1024, 64), (32, 8, 128, 2, 300, 3000, 128), (64, 8, 64, 4, 64, 4096, 32), (64, 8, 64, 8, 64, 2048, 64),
    (64, 8, 64, 16, 64, 1024, 64), (64, 8, 64, 16, 20, 1024, 32)])
def test_f32_tile_of_few_queries(ctx, nq, nkv, hd, batch, new, keys, want):
    """The fastest of the three by the times beside the rule, for queries that go on after many keys."""
    if _cus() != 256:
        pytest.skip("the times are of 256 CUs")
    assert tile(ctx, "f32", nq, nkv, hd, [new] * batch, [keys] * batch) == want


def _cus():
    import torch

    return torch.cuda.get_device_properties(0).multi_processor_count


def test_tile_of_an_empty_batch(ctx):
    assert tile(ctx, "bf16", 4, 2, 128, [], []) == 0 and tile(ctx, "bf16", 4, 2, 128, [0], [9]) == 0


LONG = [
    (16, 4, 128, [4600], [4600]),
    (12, 3, 72, [5000, 4000], [5000, 4700]),      # the end of a longer sequence
    (16, 16, 128, [8300, 1, 4100], [8300, 1, 4100]),  # a single token beside long ones
    (16, 2, 104, [9000, 0], [8200, 77]),          # more queries than keys: the first see none; no queries
    (16, 4, 128, [4200], [17000]),
    (12, 12, 128, [4999], [0]),                   # no keys
]


@pytest.mark.parametrize("t,nq,nkv,hd,lq,lk", MORE)
@pytest.mark.parametrize("is_causal", [True, False], ids=["causal", "full"])
def test_forward(torch, ctx, t, nq, nkv, hd, lq, lk, is_causal):
    import test_gpu_prompt

    test_gpu_prompt.test_forward(torch, ctx, t, nq, nkv, hd, lq, lk, is_causal)


@pytest.mark.parametrize("nq,nkv,hd,lq,lk", LONG)
@pytest.mark.parametrize("is_causal", [True, False], ids=["causal", "full"])
def test_pair_kernel(torch, ctx, nq, nkv, hd, lq, lk, is_causal):
    import raster_amd
    from test_gpu_prompt import check_forward, cu_of, rows

    print(f"[gpu] pair kernel {nq}/{nkv}x{hd} {lq} {lk} causal={is_causal}", flush=True)
    assert tile(ctx, "bf16", nq, nkv, hd, lq, lk) == 256
    g = torch.Generator(device="cuda").manual_seed(sum(lq) + sum(lk))
    q, k, v = (rows(torch, g, sum(n), w * hd, torch.bfloat16, pad=8) for n, w in ((lq, nq), (lk, nkv), (lk, nkv)))
    scale, lse = hd ** -0.5, torch.empty((nq, sum(lq)), device="cuda")
    out = raster_amd.prompt_attention(ctx, q, k, v, cu_of(torch, lq), nq, nkv, hd, scale, causal=is_causal,
                                      cu_k=None if lq == lk else cu_of(torch, lk), lse=lse)
    check_forward(torch, q, k, v, out, lse, lq, lk, nq, nkv, hd, scale, is_causal)


# queries, keys; a query sees the keys up to its own number + keys - queries
MASKED = [("bf16", 16, 4, 128, 4600, 4600, 256), ("bf16", 16, 4, 128, 4600, 4613, 256), ("bf16", 12, 3, 72, 4999, 4000, 256),
          ("bf16", 64, 8, 128, 700, 709, 64), ("bf16", 4, 2, 128, 300, 333, 32), ("bf16", 128, 8, 128, 700, 700, 128),
          ("f32", 64, 8, 104, 700, 719, 128), ("f32", 4, 1, 256, 300, 307, 128)]


@pytest.mark.parametrize("t,nq,nkv,hd,lq,lk,kernel", MASKED)
def test_reach_of_a_masked_nan(torch, ctx, t, nq, nkv, hd, lq, lk, kernel):
    """A NaN or inf in k reaches no query that does not see its key; one in v only queries that see a key
    less than 95 before it, on each kernel and with queries anywhere in their tiles of keys."""
    import raster_amd
    from test_gpu_prompt import cu_of, rows

    print(f"[gpu] masked NaN {t} {nq}/{nkv}x{hd} {lq} {lk}", flush=True)
    assert tile(ctx, t, nq, nkv, hd, [lq], [lk]) == kernel
    g = torch.Generator(device="cuda").manual_seed(lq + lk)
    ty = {"bf16": torch.bfloat16, "f32": torch.float32}[t]
    q, k, v = (rows(torch, g, n, w * hd, ty) for n, w in ((lq, nq), (lk, nkv), (lk, nkv)))
    cu, cu_k, scale = cu_of(torch, [lq]), cu_of(torch, [lk]), hd ** -0.5
    want = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, cu_k=cu_k)
    for at in (lk // 3, lk // 3 + 41, lk - 1):
        sees = max(at - (lk - lq), 0)  # the first query that sees key `at`
        for x, first in ((k, sees), (v, max(sees - 94, 0))):
            keep = x[at].clone()
            for bad in (float("nan"), float("inf")):
                x[at] = bad
                out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, cu_k=cu_k)
                assert torch.equal(out[:first], want[:first]), (at, bad)
                assert not bool(torch.isfinite(out[sees:]).all(1).any())
            x[at] = keep


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_gradient_leaves_rows_of_no_sequence_alone(torch, ctx, t):
    """dout . out, which the workspace keeps first ([n_q][rows_q]), is formed for the rows of sequences only:
    the others, before, behind or of a padded batch, are not read."""
    from test_gpu_prompt import cu_of, rows

    nq, nkv, hd, lens, first, n = 4, 2, 64, [70, 0, 45], 5, 160
    print(f"[gpu] gradient, rows of no sequence {t}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    ty = {"bf16": torch.bfloat16, "f32": torch.float32}[t]
    q, k, v, out, do = (rows(torch, g, n, w * hd, ty) for w in (nq, nkv, nkv, nq, nq))
    lse, cu = torch.zeros((nq, n), device="cuda"), cu_of(torch, lens, first)
    p = _lib.Prompt({"f32": _lib.RQ_F32, "bf16": _lib.RQ_BF16}[t], len(lens), n, n, nq, nkv, hd, cu.data_ptr(), None, 1,
                    0.125)
    need = C.c_size_t()
    _lib.call("rq_prompt_attention_bwd_work", C.byref(p), C.byref(need))
    work = torch.full((need.value // 4,), 7.0, device="cuda")
    grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
    args = [a for x in (do, q, k, v, out) for a in (x.data_ptr(), x.stride(0))]
    _lib.call("rq_prompt_attention_bwd", ctx.handle, C.byref(p), *args, lse.data_ptr(),
              *[a for x in grads for a in (x.data_ptr(), x.stride(0))], work.data_ptr(), need.value,
              torch.cuda.current_stream().cuda_stream)
    none = torch.ones(n, dtype=torch.bool, device="cuda")
    none[first:first + sum(lens)] = False
    delta = work[:nq * n].view(nq, n)
    assert bool((delta[:, none] == 7).all()) and not bool((delta[:, ~none] == 7).any())
    assert all(bool((x[none] == 7).all()) for x in grads)


# longer than test_gpu_prompt.py's gradients; both forms of dQ (workgroups of 128 and 64 queries) in bf16, split and whole
# steps of dK and dV
GRADIENTS = [
    ("bf16", 8, 2, 128, [2049, 700], [2049, 700]),
    ("bf16", 32, 8, 128, [2200, 1], [2200, 1]),
    ("bf16", 16, 2, 64, [4097], [4097]),
    ("bf16", 6, 2, 80, [1300], [2311]),           # the end of a longer sequence
    ("bf16", 4, 4, 256, [1025, 513], [1025, 600]),
    ("bf16", 4, 1, 128, [1500], [401]),           # more queries than keys
    ("f32", 16, 2, 64, [2049, 700], [2049, 700]),
    ("f32", 8, 8, 128, [1500], [1500]),
    ("f32", 2, 1, 256, [1025], [1100]),
]


@pytest.mark.parametrize("t,nq,nkv,hd,lq,lk", GRADIENTS)
@pytest.mark.parametrize("is_causal", [True, False], ids=["causal", "full"])
def test_long_gradient(torch, ctx, t, nq, nkv, hd, lq, lk, is_causal):
    import test_gpu_prompt

    test_gpu_prompt.test_gradient(torch, ctx, t, nq, nkv, hd, lq, lk, is_causal)


@pytest.mark.parametrize("t,nq,nkv,hd,lq,lk", [("bf16", 4, 2, 128, 500, 513), ("bf16", 32, 8, 64, 4500, 4500),
                                               ("f32", 4, 2, 64, 500, 461), ("f32", 2, 1, 256, 300, 307)])
def test_reach_of_a_masked_nan_in_the_gradient(torch, ctx, t, nq, nkv, hd, lq, lk):
    """A NaN in k or v reaches dq of no query whose last key is 95 or more before it; one in q or dout no dk or dv
    of a key 95 or more past the last that its query sees."""
    import raster_amd
    from test_gpu_prompt import cu_of, rows

    print(f"[gpu] masked NaN, gradient {t} {nq}/{nkv}x{hd} {lq} {lk}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(lq + lk)
    ty = {"bf16": torch.bfloat16, "f32": torch.float32}[t]
    q, k, v, do = (rows(torch, g, n, w * hd, ty) for n, w in ((lq, nq), (lk, nkv), (lk, nkv), (lq, nq)))
    cu, cu_k, scale, off = cu_of(torch, [lq]), cu_of(torch, [lk]), hd ** -0.5, lk - lq
    lse = torch.empty((nq, lq), device="cuda")
    out = raster_amd.prompt_attention(ctx, q, k, v, cu, nq, nkv, hd, scale, cu_k=cu_k, lse=lse)

    def grads():
        return raster_amd.prompt_attention_bwd(ctx, do, q, k, v, out, lse, cu, nq, nkv, hd, scale, cu_k=cu_k)

    want = grads()
    for at in (200, lq - 1):
        for x in (k, v):
            keep = x[at + off].clone()
            x[at + off] = float("nan")
            dq = grads()[0]
            assert torch.equal(dq[:max(at - 94, 0)], want[0][:max(at - 94, 0)])
            assert bool(torch.isnan(dq[at:]).any(1).all())
            x[at + off] = keep
        for x in (q, do):
            keep = x[at].clone()
            x[at] = float("nan")
            for got, clean in zip(grads()[1:], want[1:]):
                assert torch.equal(got[at + off + 95:], clean[at + off + 95:])
                assert bool(torch.isnan(got[:at + off + 1]).any(1).all())
            x[at] = keep


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch", [64, 300, 5000])
def test_many_sequences_of_a_seeded_packing(torch, ctx, dtype, batch):
    """More sequences than a wave has lanes, empty ones and single tokens among them, the packing from the seed
    too: every row against one dense product with a mask of equal sequences."""
    import attn_ref as ref
    import raster_amd
    from test_gpu_prompt import heads, rows

    print(f"[gpu] prompt {dtype} {batch} sequences", flush=True)
    nq, nkv, hd, scale = 2, 1, 64, 0.125
    ty = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g, gc = torch.Generator(device="cuda").manual_seed(batch), torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 4, (batch,), generator=gc)
    lens[torch.randperm(batch, generator=gc)[batch // 4:]] = 0
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
