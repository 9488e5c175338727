"""Cases of attention with a sliding window and of the paged cache in 8 bits.

A case is a dict of plain values; `op` names the call:

  prompt   attention over packed prompts, causal, of the last `window` keys and the first `sinks`
  train    the same in a training step: forward with its log-sum-exp, then the gradient
  decode   one new token of every sequence over a paged cache (f32, bf16 or int8): RoPE, append, attention,
           with a window or without (window 0)
  append   RoPE of packed prompts' q and k, and their k and v into an int8 cache's pages
  rows     the stored rows of sequences as values, packed

An int8 cache has a scale for each 16 rows and KV head. Rows x go into such a block with its scale raised to
max |x| / 127 (the codes before them are rounded anew when it rises), codes round(x / scale), in f32.
Codes and scales are outputs as the cache holds them: with this arithmetic they are the same numbers everywhere.

With `own` the calls of raster_amd are made, without it the same results come
from elementary torch operations in 32 bits. The heads are those of this
repository's decoder (16 x 128) and attention tests (32/8, 64/8, 16/2, 8/4).
"""
import math

import torch

own = False

THETA = 1e4
BLOCK = 16  # rows of a scale
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}
SIZES = {"f32": 4, "bf16": 2, "i8": 1}


def listed():
    return [
        # the decoder's own f32 activations: several prompts of odd lengths packed, one of them a single
        # token, one of them the rest of a prompt whose first 389 keys came before
        {"name": "prompt_ragged_f32", "op": "prompt", "t": "f32", "lens": "613,1,1024,250,89", "lens_k":
         "613,1,1024,639,89", "nq": 16, "nkv": 16, "hd": 128, "window": 256, "sinks": 4},
        # a long document into a grouped-query model with a window: the largest call
        {"name": "prompt_long", "op": "prompt", "t": "bf16", "lens": "16384", "lens_k": "", "nq": 32, "nkv": 8,
         "hd": 128, "window": 4096, "sinks": 4},
        # a packed fine-tuning batch, odd lengths
        {"name": "train_packed", "op": "train", "t": "bf16", "lens": "4096,777,1500,331,1999,64", "lens_k": "",
         "nq": 32, "nkv": 8, "hd": 128, "window": 1024, "sinks": 4},
        # a small model trained in f32 on short examples, a short window without sinks
        {"name": "train_small_f32", "op": "train", "t": "f32", "lens": "129,300,64,511", "lens_k": "", "nq": 16,
         "nkv": 2, "hd": 64, "window": 100, "sinks": 0},
        # one user, one token, the decoder's 128 positions in 8 bits
        {"name": "decode_one_i8", "op": "decode", "t": "f32", "cache": "i8", "lens": "128", "page": 16, "nq": 16,
         "nkv": 16, "hd": 128, "window": 0, "sinks": 0},
        # a serving batch of mixed lengths, new and old sequences, f32 activations
        {"name": "decode_batch_i8", "op": "decode", "t": "f32", "cache": "i8", "lens":
         "0,17,4095,900,2300,64,8191,333,1024,5001,48,700,3100,1,260,1999,6400,120,77,2048,512,31,1500,7000,15,"
         "4200,96,840,1280,16,3700,601", "page": 16, "nq": 32, "nkv": 8, "hd": 128, "window": 0, "sinks": 0},
        # long contexts in 8 bits
        {"name": "decode_long_i8", "op": "decode", "t": "bf16", "cache": "i8", "lens":
         "65535,32768,50001,60000,40960,65000,57344,61111", "page": 64, "nq": 64, "nkv": 8, "hd": 128, "window": 0,
         "sinks": 0},
        # streams of very different ages, each seeing its last 4096 tokens and the first 4
        {"name": "decode_window", "op": "decode", "t": "bf16", "cache": "bf16", "lens":
         "65535,3,20000,4096,4100,50001,900,12345,33000,8191,64,5000,40960,1,2047,60000", "page": 16, "nq": 32,
         "nkv": 8, "hd": 128, "window": 4096, "sinks": 4},
        # a few short prompts into the cache, f32
        {"name": "append_small", "op": "append", "t": "f32", "cache": "i8", "lens": "37,5,1", "past": "0,128,40",
         "page": 16, "nq": 16, "nkv": 16, "hd": 128},
        # a prefill batch into the cache
        {"name": "append_batch", "op": "append", "t": "bf16", "cache": "i8", "lens": "4096,613,1999,1,1483", "past":
         "0,0,2048,77,0", "page": 16, "nq": 32, "nkv": 8, "hd": 128},
        # what the keys of prompts that go on after the small append are
        {"name": "rows_small", "op": "rows", "t": "f32", "cache": "i8", "lens": "37,133,41", "page": 16, "nq": 16,
         "nkv": 16, "hd": 128},
        # the same after the prefill batch
        {"name": "rows_batch", "op": "rows", "t": "bf16", "cache": "i8", "lens": "4096,613,4047,78,1483", "page": 16,
         "nq": 32, "nkv": 8, "hd": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(v):
    return ",".join(str(x) for x in v)


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "decode", "decode", "decode", "append", "rows"])
    nq, nkv = rng.choice([(16, 16), (32, 8), (64, 8), (16, 2), (8, 4), (12, 12), (24, 12)])
    hd = rng.choice([64, 128, 128, 128, 80, 256])
    t = rng.choice(["f32", "bf16", "bf16"])
    sinks = rng.choice([0, 1, 4, 4, _log(rng, 1, 200)])
    if op in ("prompt", "train"):
        top = 1500 if t == "f32" else 3000
        lens = [_log(rng, 1, top) for _ in range(_log(rng, 1, 8))]
        while len(lens) * max(lens) ** 2 * nq * hd * (3.5 if op == "train" else 1) > 32 * 128 * 8192 ** 2:
            lens = [-(-n // 2) for n in lens]
        if op == "train" or rng.random() < 0.6:
            lens_k = ""
        else:
            lens_k = _text([n + rng.choice([0, _log(rng, 1, 500)]) for n in lens])
        return {"op": op, "t": t, "lens": _text(lens), "lens_k": lens_k, "nq": nq, "nkv": nkv, "hd": hd,
                "window": _log(rng, 1, 2000), "sinks": sinks}
    page = rng.choice([16, 32, 64, 128])
    if op == "decode":
        cache = rng.choice(["i8", "i8", "bf16" if t == "bf16" else rng.choice(["f32", "bf16"])])
        window = 0 if cache == "i8" and rng.random() < 0.6 else _log(rng, 1, 5000)
        lens = [_log(rng, 1, 9000) - 1 for _ in range(_log(rng, 1, 48))]
        return {"op": op, "t": t, "cache": cache, "lens": _text(lens), "page": page, "nq": nq, "nkv": nkv, "hd": hd,
                "window": window, "sinks": sinks if window else 0}
    lens = [_log(rng, 1, 2000) for _ in range(_log(rng, 1, 8))]
    case = {"op": op, "t": t, "cache": "i8", "lens": _text(lens), "page": page, "nq": nq, "nkv": nkv, "hd": hd}
    if op == "append":
        case["past"] = _text([rng.choice([0, _log(rng, 1, 4000)]) for _ in lens])
    return case


def _ints(text):
    return [int(x) for x in text.split(",")]


def _lens(case):
    lq = _ints(case["lens"])
    return lq, _ints(case["lens_k"]) if case.get("lens_k") else lq


def _seen(i, window, sinks):
    """Keys that the query at position i sees."""
    if window == 0 or i < window:
        return i + 1
    return window + min(sinks, i + 1 - window)


def _seen_before(n, window, sinks):
    """The same, summed over the positions before n."""
    a = min(n, window + sinks)  # those that see all keys up to their own
    return a * (a + 1) // 2 + (n - a) * (window + sinks)


def work(case):
    op, nq, nkv, hd, e = case["op"], case["nq"], case["nkv"], case["hd"], SIZES[case["t"]]
    if op in ("prompt", "train"):
        lq, lk = _lens(case)
        w, z = case["window"], case["sinks"]
        rq, rk = sum(lq) * nq * hd, sum(lk) * nkv * hd
        pairs = sum(_seen_before(b, w, z) - _seen_before(b - a, w, z) for a, b in zip(lq, lk))
        if op == "prompt":
            return {"bytes": e * (2 * rq + 2 * rk), "flops": 4 * hd * nq * pairs}
        # forward and backward: q, k, v, dout in; out, dq, dk, dv and the log-sum-exp out
        return {"bytes": e * (4 * rq + 4 * rk) + 4 * sum(lq) * nq, "flops": 14 * hd * nq * pairs}
    lens = _ints(case["lens"])
    per_row = 2 * nkv * hd * SIZES[case["cache"]] + (8 * nkv / BLOCK if case["cache"] == "i8" else 0)
    if op == "decode":
        b, seen = len(lens), sum(_seen(n, case["window"], case["sinks"]) for n in lens)
        return {"bytes": int((seen - b) * per_row + b * (2 * nq + 2 * nkv) * hd * e + b * per_row),
                "flops": 4 * hd * nq * seen}
    rows = sum(lens)
    if op == "append":
        return {"bytes": int(rows * (hd * e * (2 * nq + 3 * nkv) + per_row)), "flops": 3 * rows * hd * (nq + 3 * nkv)}
    return {"bytes": int(rows * (per_row + 2 * nkv * hd * e)), "flops": 2 * rows * nkv * hd}


def _cu(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _randn(g, t, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[t])


def _stored(g, case, pages):
    """Pages with something in them: (pages, scales)."""
    page, nkv, hd = case["page"], case["nkv"], case["hd"]
    if case["cache"] != "i8":
        return _randn(g, case["cache"], pages, page, nkv * hd), None
    x = torch.randn((pages, page // BLOCK, BLOCK, nkv, hd), generator=g, device="cuda")
    s = x.abs().amax((2, 4)) * torch.tensor(1 / 127, device="cuda")
    return (x / s[:, :, None, :, None]).round_().to(torch.int8).view(pages, page, nkv * hd), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    if op in ("prompt", "train"):
        lq, lk = _lens(case)
        rows, rows_k = sum(lq), sum(lk)
        if lk == lq:  # one product's output holds q, k and v side by side
            qkv = _randn(g, case["t"], rows, (nq + 2 * nkv) * hd)
            s["q"], s["k"], s["v"] = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
        else:
            s["q"] = _randn(g, case["t"], rows, nq * hd)
            s["k"], s["v"] = (_randn(g, case["t"], rows_k, nkv * hd) for _ in range(2))
        s["cu"], s["cu_k"] = _cu(lq), None if lk == lq else _cu(lk)
        s["max_q"], s["max_k"] = max(lq), max(lk)
        if op == "train":
            s["dout"] = _randn(g, case["t"], rows, nq * hd)
        return s
    lens = _ints(case["lens"])
    past = lens if op == "decode" else _ints(case["past"]) if op == "append" else [0] * len(lens)
    new = [1] * len(lens) if op == "decode" else lens
    page, rows = case["page"], sum(new)
    if op != "rows":
        qkv = _randn(g, case["t"], rows, (nq + 2 * nkv) * hd)
        s["q"], s["k"], s["v"] = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
    need = [-(-(p + n) // page) for p, n in zip(past, new)]
    total = sum(need) + 3
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed))
    table, at = torch.zeros((len(need), max(need)), dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    s["table"] = table.cuda()
    s["kpages"], s["kscales"] = _stored(g, case, total)
    s["vpages"], s["vscales"] = _stored(g, case, total)
    s["past"] = torch.tensor(past, dtype=torch.int32, device="cuda")
    s["max_len"], s["rows"] = max(p + n for p, n in zip(past, new)), rows
    s["cu"] = _cu(new)
    return s


def _cache(s):
    """The cache's own buffers, as outputs."""
    names = ("kpages", "vpages") + (("kscales", "vscales") if s["cache"] == "i8" else ())
    return {n: s[n] for n in names}


# ---- the framework's calls ------------------------------------------------------


def _run_own(s):
    import raster_amd as rq

    ctx, op = rq.context(0), s["op"]
    nq, nkv, hd = s["nq"], s["nkv"], s["hd"]
    if op == "prompt":
        return rq.prompt_attention(ctx, s["q"], s["k"], s["v"], s["cu"], nq, nkv, hd, hd ** -0.5, cu_k=s["cu_k"],
                                   window=s["window"], sinks=s["sinks"])
    if op == "train":
        lse = torch.empty((nq, s["q"].shape[0]), device="cuda")
        see = {"window": s["window"], "sinks": s["sinks"]}
        out = rq.prompt_attention(ctx, s["q"], s["k"], s["v"], s["cu"], nq, nkv, hd, hd ** -0.5, lse=lse, **see)
        dq, dk, dv = rq.prompt_attention_bwd(ctx, s["dout"], s["q"], s["k"], s["v"], out, lse, s["cu"], nq, nkv, hd,
                                             hd ** -0.5, **see)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    scales = {"kscales": s["kscales"], "vscales": s["vscales"]}
    if op == "decode":
        out = rq.paged_attention(ctx, s["q"], s["k"], s["v"], s["kpages"], s["vpages"], s["table"], s["past"], nq,
                                 nkv, hd, THETA, hd ** -0.5, max_len=s["max_len"], window=s["window"],
                                 sinks=s["sinks"], **scales)
        return {"out": out} | _cache(s)
    if op == "append":
        q, k = rq.pages_append(ctx, s["q"], s["k"], s["v"], s["kpages"], s["vpages"], s["table"], s["cu"], s["past"],
                               nq, nkv, hd, THETA, **scales)
        return {"q": q, "k": k} | _cache(s)
    k, v = rq.pages_rows(ctx, s["kpages"], s["vpages"], s["table"], s["cu"], s["rows"], nkv, hd, TYPES[s["t"]],
                         **scales)
    return {"k": k, "v": v}


# ---- the plain form ----------------------------------------------------------------


def _pad(x, cu, longest, heads, hd):
    """Packed rows [rows, heads * hd] as f32 [sequences, heads, longest, hd] (rows past an end repeat another)."""
    at = cu[:-1].long()[:, None] + torch.arange(longest, device="cuda")
    return x[at.clamp(max=x.shape[0] - 1)].float().view(-1, longest, heads, hd).transpose(1, 2).contiguous()


def _unpad(y, cu, rows):
    """[sequences, heads, longest, hd] back to packed rows [rows, heads * hd]."""
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(cu.long(), r, right=True) - 1
    return y[b, :, r - cu.long()[b]].reshape(rows, -1)


def _grouped(q, k):
    """Scores [sequences, nkv, group * longest, keys] of q [sequences, nq, longest, hd] with k [sequences, nkv, keys, hd]."""
    n, nkv = k.shape[:2]
    return torch.matmul(q.reshape(n, nkv, -1, q.shape[-1]), k.transpose(2, 3).contiguous())


def _visible(s, cu_k):
    """[sequences, 1, 1, longest, longest_k]: whether query i sees key j."""
    lq, lk = s["cu"][1:] - s["cu"][:-1], cu_k[1:] - cu_k[:-1]
    i, j = torch.arange(s["max_q"], device="cuda")[:, None], torch.arange(s["max_k"], device="cuda")
    at = i + (lk - lq)[:, None, None]  # the query's position
    see = (j <= at) & ((j > at - s["window"]) | (j < s["sinks"]))
    return (see & (j < lk[:, None, None]) & (i < lq[:, None, None]))[:, None, None]


def _plain_prompt(s):
    nq, nkv, hd, lq, lk = s["nq"], s["nkv"], s["hd"], s["max_q"], s["max_k"]
    cu, cu_k = s["cu"], s["cu"] if s["cu_k"] is None else s["cu_k"]
    q, k, v = _pad(s["q"], cu, lq, nq, hd), _pad(s["k"], cu_k, lk, nkv, hd), _pad(s["v"], cu_k, lk, nkv, hd)
    n = q.shape[0]
    see = _visible(s, cu_k)
    x = _grouped(q, k).view(n, nkv, nq // nkv, lq, lk).mul_(hd ** -0.5).masked_fill_(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = x.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    p /= torch.where(z == 0, torch.ones_like(z), z)
    out = torch.matmul(p.view(n, nkv, -1, lk), v).view(n, nq, lq, hd)
    lse = (z.log() + m).view(n, nq, lq, 1)
    return q, k, v, p.view(n, nkv, -1, lk), out, lse


def _run_train(s):
    nq, nkv, hd, lq = s["nq"], s["nkv"], s["hd"], s["max_q"]
    t, rows = TYPES[s["t"]], s["q"].shape[0]
    q, k, v, p, out, lse = _plain_prompt(s)
    n = q.shape[0]
    inside = (torch.arange(lq, device="cuda") < (s["cu"][1:] - s["cu"][:-1])[:, None])[:, None, :, None]
    do = _pad(s["dout"], s["cu"], lq, nq, hd) * inside
    delta = (do * out).sum(-1, keepdim=True).view(n, nkv, -1, 1)
    dog, pt = do.view(n, nkv, -1, hd), p.transpose(2, 3).contiguous()
    dv = torch.matmul(pt, dog)
    ds = _grouped(do, v).sub_(delta).mul_(p).mul_(hd ** -0.5)
    dq = torch.matmul(ds, k).view(n, nq, lq, hd)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q.view(n, nkv, -1, hd))
    back = [_unpad(y, s["cu"], rows).to(t) for y in (out, dq, dk, dv)]
    return {"out": back[0], "lse": _unpad(lse, s["cu"], rows).t().contiguous(), "dq": back[1], "dk": back[2],
            "dv": back[3]}


def _rope(x, heads, hd, pos):
    """x [rows, heads * hd] rotated by its rows' positions, in f32 (angles in 64 bits)."""
    freq = torch.exp(torch.arange(hd // 2, device="cuda", dtype=torch.float64) * (-2.0 / hd * math.log(THETA)))
    ang = pos.double()[:, None] * freq
    c, sn = ang.cos().float()[:, None], ang.sin().float()[:, None]
    a, b = x.float().view(-1, heads, hd).split(hd // 2, 2)
    return torch.cat([a * c - b * sn, b * c + a * sn], 2).view(x.shape[0], -1)


def _store_i8(pages, scales, slot, x):
    """Rows x [rows, nkv, hd] at rows `slot` of all pages; the rows behind them in a block are left as they are."""
    n, nkv, hd = x.shape
    codes, sc, block, row = pages.view(-1, BLOCK, nkv, hd), scales.view(-1, nkv), slot // BLOCK, slot % BLOCK
    new = torch.zeros_like(sc).scatter_reduce_(0, block[:, None].expand(n, nkv), x.abs().amax(2), "amax")[block]
    first = torch.full_like(sc[:, 0], BLOCK).scatter_reduce_(0, block, row.float(), "amin")[block]
    old = torch.where(first[:, None] > 0, sc[block], torch.zeros_like(new))
    s = torch.maximum(old, new * torch.tensor(1 / 127, device="cuda"))
    f = torch.where(s > 0, old / s, torch.ones_like(s))
    held = codes[block]
    before = (torch.arange(BLOCK, device="cuda") < first[:, None])[:, :, None, None]
    codes[block] = torch.where(before, (held.float() * f[:, None, :, None]).round_().to(torch.int8), held)
    sc[block] = s
    c = torch.where(s[:, :, None] > 0, x / s[:, :, None], torch.zeros_like(x))
    codes.view(-1, nkv, hd)[slot] = c.round_().clamp_(-127, 127).to(torch.int8)


def _store(s, seq, pos, k, v):
    """Rows k, v (f32) into the pages of sequences `seq` at positions `pos`."""
    nkv, hd, page = s["nkv"], s["hd"], s["page"]
    slot = s["table"].long()[seq, pos // page] * page + pos % page
    if s["cache"] == "i8":
        _store_i8(s["kpages"], s["kscales"], slot, k.view(-1, nkv, hd))
        _store_i8(s["vpages"], s["vscales"], slot, v.float().view(-1, nkv, hd))
    else:
        s["kpages"].view(-1, nkv * hd)[slot] = k.to(TYPES[s["cache"]])
        s["vpages"].view(-1, nkv * hd)[slot] = v.to(TYPES[s["cache"]])


def _values(s, which, ids):
    """Pages `ids` as f32 values [..., page, nkv, hd]."""
    x = s[which + "pages"][ids].float().view(*ids.shape, s["page"], s["nkv"], s["hd"])
    if s["cache"] == "i8":
        x = x * s[which + "scales"][ids].repeat_interleave(BLOCK, -2)[..., None]
    return x


def _run_decode(s):
    nq, nkv, hd = s["nq"], s["nkv"], s["hd"]
    past = s["past"].long()
    n, rows = past.shape[0], s["table"].shape[1] * s["page"]
    q, k = _rope(s["q"], nq, hd, past), _rope(s["k"], nkv, hd, past)
    _store(s, torch.arange(n, device="cuda"), past, k, s["v"])
    keys, values = (_values(s, x, s["table"].long()).view(n, rows, nkv, hd).transpose(1, 2).contiguous() for x in "kv")
    j, at = torch.arange(rows, device="cuda"), past[:, None]
    see = (j <= at) & ((j > at - s["window"]) | (j < s["sinks"]) if s["window"] else j >= 0)
    see = see[:, None, None]
    x = _grouped(q.view(n, nq, 1, hd), keys).mul_(hd ** -0.5).masked_fill_(~see, -math.inf)
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    out = torch.matmul(p, values * see.transpose(2, 3)).view(n, -1).to(TYPES[s["t"]])
    return {"out": out} | _cache(s)


def _of_rows(s):
    """Every packed row's sequence, and its number there."""
    cu, r = s["cu"].long(), torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(cu, r, right=True) - 1
    return seq, r - cu[seq]


def _run_append(s):
    t = TYPES[s["t"]]
    seq, at = _of_rows(s)
    pos = at + s["past"].long()[seq]
    q, k = _rope(s["q"], s["nq"], s["hd"], pos), _rope(s["k"], s["nkv"], s["hd"], pos)
    _store(s, seq, pos, k, s["v"])
    return {"q": q.to(t), "k": k.to(t)} | _cache(s)


def _run_rows(s):
    seq, at = _of_rows(s)
    page = s["table"].long()[seq, at // s["page"]]
    slot = page * s["page"] + at % s["page"]
    nkv, hd, t = s["nkv"], s["hd"], TYPES[s["t"]]
    k, v = (s[x + "pages"].view(-1, nkv, hd)[slot].float() * s[x + "scales"].view(-1, nkv)[slot // BLOCK][..., None]
            for x in "kv")
    return {"k": k.to(t).view(-1, nkv * hd), "v": v.to(t).view(-1, nkv * hd)}


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "prompt":
        return _unpad(_plain_prompt(s)[4], s["cu"], s["q"].shape[0]).to(TYPES[s["t"]])
    return {"train": _run_train, "decode": _run_decode, "append": _run_append, "rows": _run_rows}[s["op"]](s)


# ---- the definition, in 64 bits ----------------------------------------------------


def _exact_rotated_rows(x, heads, hd, at):
    y = x.double().reshape(-1, heads, hd)
    i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    a = (at.double()[:, None] * THETA ** (-2 * i / hd))[:, None]
    lo, hi = y[..., :hd // 2], y[..., hd // 2:]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)


def _exact_hidden(a, b, window, sinks):
    """Of a queries and b keys: the pairs that do not see each other."""
    at, j = torch.arange(b - a, b, device="cuda")[:, None], torch.arange(b, device="cuda")[None]
    late = j > at
    gone = (at - j >= window) & (j >= sinks) if window else torch.zeros_like(late)
    return late | gone


def _exact_attend(case, s):
    """Every head of every sequence by itself."""
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    lq, lk = _lens(case)
    f64 = dict(dtype=torch.float64, device="cuda")
    r = {"out": torch.zeros((sum(lq), nq * hd), **f64), "lse": torch.zeros((nq, sum(lq)), **f64)}
    if case["op"] == "train":
        r |= {"dq": torch.zeros((sum(lq), nq * hd), **f64), "dk": torch.zeros((sum(lk), nkv * hd), **f64),
              "dv": torch.zeros((sum(lk), nkv * hd), **f64)}
    q0 = k0 = 0
    for a, b in zip(lq, lk):
        hidden = _exact_hidden(a, b, case["window"], case["sinks"])
        for h in range(nq):
            g = h // (nq // nkv)
            at, kt = (slice(q0, q0 + a), slice(h * hd, h * hd + hd)), (slice(k0, k0 + b), slice(g * hd, g * hd + hd))
            q, k, v = s["q"][at].double(), s["k"][kt].double(), s["v"][kt].double()
            x = (q @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
            r["lse"][h, q0:q0 + a] = torch.logsumexp(x, 1)
            p = torch.softmax(x, 1)
            r["out"][at] = p @ v
            if case["op"] == "train":
                do = s["dout"][at].double()
                dp = do @ v.T
                dx = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(hd)
                r["dq"][at] = dx @ k
                r["dk"][kt] += dx.T @ q
                r["dv"][kt] += p.T @ do
        q0, k0 = q0 + a, k0 + b
    return r if case["op"] == "train" else r["out"]


def _exact_put(codes, scales, row, x):
    """Rows x [n, nkv, hd] behind the first `row` ones of a sequence: codes [blocks, 16, nkv, hd] and scales
    [blocks, nkv] of it, in 64 bits."""
    i = 0
    while i < len(x):
        b, r = divmod(row + i, BLOCK)
        part = x[i:i + BLOCK - r]
        old = scales[b] if r else torch.zeros_like(scales[b])
        s = torch.maximum(old, part.abs().amax((0, 2)) / 127)
        safe = torch.where(s > 0, s, torch.ones_like(s))
        codes[b, :r] = torch.round(codes[b, :r] * (old / safe)[:, None])
        codes[b, r:r + len(part)] = torch.round(part / safe[:, None]).clamp(-127, 127)
        scales[b] = s
        i += len(part)


def _exact_stored(case, s, b, past, k, v):
    """Keys and values [rows, nkv, hd] of sequence b with the rows k, v behind its first `past` ones, and the
    outputs' pages brought up to date."""
    nkv, hd, page = case["nkv"], case["hd"], case["page"]
    n = past + len(k)
    mine = s["table"][b, :-(-n // page)].long()
    got = []
    for which, x in (("k", k), ("v", v)):
        held = s[which + "pages"][mine].double()
        if case["cache"] == "i8":
            codes, scales = held.view(-1, BLOCK, nkv, hd), s[which + "scales"][mine].double().view(-1, nkv)
            _exact_put(codes, scales, past, x)
            s[which + "pages"][mine] = codes.view(-1, page, nkv * hd).to(torch.int8)
            s["exact_" + which][mine] = scales.view(len(mine), -1, nkv)
            held = (codes * scales[:, None, :, None]).view(-1, nkv, hd)
        else:
            flat = held.view(-1, nkv, hd)
            flat[past:n] = x
            s["exact_" + which][mine] = held
            held = flat.clone()
            held[past:n] = x.to(TYPES[case["cache"]]).double()  # attended as it is stored
        got.append(held[:n])
    return got


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("prompt", "train"):
        return _exact_attend(case, s)
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    lens = _ints(case["lens"])
    if op == "rows":
        out = []
        for which in "kv":
            rows = []
            for b, n in enumerate(lens):
                mine = s["table"][b, :-(-n // page)].long()
                x = s[which + "pages"][mine].double().view(-1, BLOCK, nkv, hd)
                rows.append((x * s[which + "scales"][mine].double().view(-1, 1, nkv, 1)).view(-1, nkv * hd)[:n])
            out.append(torch.cat(rows))
        return {"k": out[0], "v": out[1]}
    i8 = case["cache"] == "i8"
    for which in "kv":
        s["exact_" + which] = (s[which + "scales"] if i8 else s[which + "pages"]).double()
    past = lens if op == "decode" else _ints(case["past"])
    new = [1] * len(lens) if op == "decode" else lens
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(past, new)])
    q, k = _exact_rotated_rows(s["q"], nq, hd, pos), _exact_rotated_rows(s["k"], nkv, hd, pos)
    v = s["v"].double().reshape(-1, nkv, hd)
    out, r = torch.empty((len(pos), nq * hd), dtype=torch.float64, device="cuda"), 0
    for b, (p, n) in enumerate(zip(past, new)):
        keys, values = _exact_stored(case, s, b, p, k[r:r + n], v[r:r + n])
        if op == "decode":
            hidden = _exact_hidden(1, p + 1, case["window"], case["sinks"])[0]
            for h in range(nq):
                g = h // (nq // nkv)
                x = keys[:, g] @ q[b, h] / math.sqrt(hd)
                out[b, h * hd:h * hd + hd] = torch.softmax(x.masked_fill(hidden, -math.inf), 0) @ values[:, g]
        r += n
    first = {"out": out} if op == "decode" else {"q": q.reshape(-1, nq * hd), "k": k.reshape(-1, nkv * hd)}
    if i8:
        return first | {"kpages": s["kpages"], "vpages": s["vpages"], "kscales": s["exact_k"], "vscales": s["exact_v"]}
    return first | {"kpages": s["exact_k"], "vpages": s["exact_v"]}
