"""Cases of the attention and paged-cache operators around the quantized linears.

A case is a dict of plain values; `op` names the call:

  prompt   attention over packed prompts, causal, grouped heads
  train    the same in a training step: forward with its log-sum-exp, then the gradient
  decode   one new token of every sequence over a paged cache: RoPE, append, attention
  append   RoPE of packed prompts' q and k, and their k and v into the cache's pages
  copy     pages copied within the cache of all layers: fork, copy-on-write, compaction

With `own` the calls of raster_amd are made, without it the same results come
from elementary torch operations in 32 bits. The heads are those of this
repository's decoder (16 x 128) and attention tests (32/8, 64/8, 16/2, 8/4).
"""
import math

import torch

own = False

THETA = 1e4
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one short prompt of a chat, as it comes in: launches and latency
        {"name": "prompt_short", "op": "prompt", "t": "bf16", "lens": "37", "lens_k": "", "nq": 16, "nkv": 16,
         "hd": 128},
        # the decoder's own f32 activations: several prompts of odd lengths packed, one of them a single
        # token, one of them the rest of a prompt whose first 389 keys came before
        {"name": "prompt_ragged_f32", "op": "prompt", "t": "f32", "lens": "613,1,1024,250,89", "lens_k":
         "613,1,1024,639,89", "nq": 16, "nkv": 16, "hd": 128},
        # a long document into a grouped-query model: the largest call
        {"name": "prompt_long", "op": "prompt", "t": "bf16", "lens": "8192", "lens_k": "", "nq": 32, "nkv": 8,
         "hd": 128},
        # a packed fine-tuning batch, odd lengths
        {"name": "train_packed", "op": "train", "t": "bf16", "lens": "2048,777,1500,331,1999,64", "lens_k": "",
         "nq": 32, "nkv": 8, "hd": 128},
        # a small model trained in f32 on short examples
        {"name": "train_small_f32", "op": "train", "t": "f32", "lens": "129,300,64,511", "lens_k": "", "nq": 16,
         "nkv": 2, "hd": 64},
        # one user, one token, the decoder's f32 cache of 128 positions
        {"name": "decode_one", "op": "decode", "t": "f32", "cache": "f32", "lens": "128", "page": 16, "nq": 16,
         "nkv": 16, "hd": 128},
        # a serving batch of mixed lengths, new and old sequences, f32 activations over a bf16 cache
        {"name": "decode_batch", "op": "decode", "t": "f32", "cache": "bf16", "lens":
         "0,17,4095,900,2300,64,8191,333,1024,5001,48,700,3100,1,260,1999,6400,120,77,2048,512,31,1500,7000,15,"
         "4200,96,840,1280,16,3700,601", "page": 16, "nq": 32, "nkv": 8, "hd": 128},
        # long contexts
        {"name": "decode_long", "op": "decode", "t": "bf16", "cache": "bf16", "lens":
         "65535,32768,50001,60000,40960,65000,57344,61111", "page": 64, "nq": 64, "nkv": 8, "hd": 128},
        # a few short prompts into the cache, f32
        {"name": "append_small", "op": "append", "t": "f32", "cache": "f32", "lens": "37,5,1", "past": "0,128,40",
         "page": 16, "nq": 16, "nkv": 16, "hd": 128},
        # a prefill batch into the cache
        {"name": "append_batch", "op": "append", "t": "bf16", "cache": "bf16", "lens": "4096,613,1999,1,1483", "past":
         "0,0,2048,77,0", "page": 16, "nq": 32, "nkv": 8, "hd": 128},
        # a beam forked: the last, part-filled page of each of 12 sequences, all layers
        {"name": "copy_fork", "op": "copy", "t": "bf16", "planes": 32, "pages": 256, "page": 16, "width": 1024,
         "n": 12},
        # a cache compacted after many sequences ended
        {"name": "copy_compact", "op": "copy", "t": "bf16", "planes": 32, "pages": 4096, "page": 16, "width": 1024,
         "n": 1300},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(v):
    return ",".join(str(x) for x in v)


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "decode", "decode", "append", "copy"])
    nq, nkv = rng.choice([(16, 16), (32, 8), (64, 8), (16, 2), (8, 4), (12, 12), (24, 12)])
    hd = rng.choice([64, 128, 128, 128, 80, 256])
    t = rng.choice(["f32", "bf16", "bf16"])
    if op in ("prompt", "train"):
        top = 1500 if t == "f32" else 3000
        lens = [_log(rng, 1, top) for _ in range(_log(rng, 1, 8))]
        # no more than the largest listed call (a training step does three and a half times a forward's products)
        while len(lens) * max(lens) ** 2 * nq * hd * (3.5 if op == "train" else 1) > 32 * 128 * 8192 ** 2:
            lens = [-(-n // 2) for n in lens]
        if op == "train" or rng.random() < 0.6:
            lens_k = ""
        else:
            lens_k = _text([n + rng.choice([0, _log(rng, 1, 500)]) for n in lens])
        return {"op": op, "t": t, "lens": _text(lens), "lens_k": lens_k, "nq": nq, "nkv": nkv, "hd": hd}
    page = rng.choice([16, 32, 64, 128])
    cache = "bf16" if t == "bf16" else rng.choice(["f32", "bf16"])
    if op == "decode":
        lens = [_log(rng, 1, 9000) - 1 for _ in range(_log(rng, 1, 48))]
        return {"op": op, "t": t, "cache": cache, "lens": _text(lens), "page": page, "nq": nq, "nkv": nkv, "hd": hd}
    if op == "append":
        lens = [_log(rng, 1, 2000) for _ in range(_log(rng, 1, 8))]
        past = [rng.choice([0, _log(rng, 1, 4000)]) for _ in lens]
        return {"op": op, "t": t, "cache": cache, "lens": _text(lens), "past": _text(past), "page": page, "nq": nq,
                "nkv": nkv, "hd": hd}
    pages = _log(rng, 8, 3000)
    return {"op": op, "t": t, "planes": 2 * _log(rng, 1, 16), "pages": pages, "page": rng.choice([16, 32]),
            "width": nkv * min(hd, 128), "n": _log(rng, 1, max(1, pages // 2))}


def _ints(text):
    return [int(x) for x in text.split(",")]


def _lens(case):
    lq = _ints(case["lens"])
    return lq, _ints(case["lens_k"]) if case.get("lens_k") else lq


def _pairs(lq, lk):
    """(query, key) pairs that a causal mask aligned at the ends leaves."""
    n = 0
    for a, b in zip(lq, lk):
        first = b - a + 1  # keys that the first query sees
        n += a * first + a * (a - 1) // 2
    return n


def _size(t):
    return 4 if t == "f32" else 2


def work(case):
    op = case["op"]
    if op == "copy":
        return {"bytes": 2 * case["n"] * case["planes"] * case["page"] * case["width"] * _size(case["t"]), "flops": 0}
    nq, nkv, hd, e = case["nq"], case["nkv"], case["hd"], _size(case["t"])
    if op in ("prompt", "train"):
        lq, lk = _lens(case)
        rq, rk, pairs = sum(lq) * nq * hd, sum(lk) * nkv * hd, _pairs(lq, lk)
        if op == "prompt":
            return {"bytes": e * (2 * rq + 2 * rk), "flops": 4 * hd * nq * pairs}
        # forward and backward: q, k, v, dout in; out, dq, dk, dv and the log-sum-exp out
        return {"bytes": e * (4 * rq + 4 * rk) + 4 * sum(lq) * nq, "flops": 14 * hd * nq * pairs}
    ce, lens = _size(case["cache"]), _ints(case["lens"])
    if op == "decode":
        b = len(lens)
        return {"bytes": sum(lens) * 2 * nkv * hd * ce + b * (2 * nq + 2 * nkv) * hd * e + b * 2 * nkv * hd * ce,
                "flops": 4 * hd * nq * (sum(lens) + b)}
    rows = sum(lens)
    return {"bytes": rows * hd * (e * (2 * nq + 3 * nkv) + ce * 2 * nkv), "flops": 3 * rows * hd * (nq + nkv)}


def _cu(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _randn(g, t, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[t])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    if op == "copy":
        s["pages_all"] = _randn(g, case["t"], case["planes"], case["pages"], case["page"], case["width"])
        order = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed)).tolist()
        s["src"], s["dst"] = order[:case["n"]], order[case["n"]:2 * case["n"]]
        return s
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
    past = lens if op == "decode" else _ints(case["past"])
    new = [1] * len(lens) if op == "decode" else lens
    page, rows = case["page"], sum(new)
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
    s["kpages"], s["vpages"] = (_randn(g, case["cache"], total, page, nkv * hd) for _ in range(2))
    s["past"] = torch.tensor(past, dtype=torch.int32, device="cuda")
    s["max_len"] = max(p + n for p, n in zip(past, new))
    if op == "append":
        s["cu"] = _cu(lens)
    return s


# ---- the framework's calls ------------------------------------------------------


def _run_own(s):
    import raster_amd as rq

    ctx, op = rq.context(0), s["op"]
    if op == "copy":
        return rq.pages_copy(ctx, s["pages_all"], s["src"], s["dst"])
    nq, nkv, hd = s["nq"], s["nkv"], s["hd"]
    if op == "prompt":
        return rq.prompt_attention(ctx, s["q"], s["k"], s["v"], s["cu"], nq, nkv, hd, hd ** -0.5, cu_k=s["cu_k"])
    if op == "train":
        lse = torch.empty((nq, s["q"].shape[0]), device="cuda")
        out = rq.prompt_attention(ctx, s["q"], s["k"], s["v"], s["cu"], nq, nkv, hd, hd ** -0.5, lse=lse)
        dq, dk, dv = rq.prompt_attention_bwd(ctx, s["dout"], s["q"], s["k"], s["v"], out, lse, s["cu"], nq, nkv, hd,
                                             hd ** -0.5)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if op == "decode":
        out = rq.paged_attention(ctx, s["q"], s["k"], s["v"], s["kpages"], s["vpages"], s["table"], s["past"], nq,
                                 nkv, hd, THETA, hd ** -0.5, max_len=s["max_len"])
        return {"out": out, "kpages": s["kpages"], "vpages": s["vpages"]}
    q, k = rq.pages_append(ctx, s["q"], s["k"], s["v"], s["kpages"], s["vpages"], s["table"], s["cu"], s["past"], nq,
                           nkv, hd, THETA)
    return {"q": q, "k": k, "kpages": s["kpages"], "vpages": s["vpages"]}


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


def _causal(cu, cu_k, longest, longest_k):
    """[sequences, 1, 1, longest, longest_k]: whether query i sees key j."""
    lq, lk = cu[1:] - cu[:-1], cu_k[1:] - cu_k[:-1]
    i, j = torch.arange(longest, device="cuda")[:, None], torch.arange(longest_k, device="cuda")
    see = (j <= i + (lk - lq)[:, None, None]) & (j < lk[:, None, None]) & (i < lq[:, None, None])
    return see[:, None, None]


def _plain_prompt(s):
    nq, nkv, hd, lq, lk = s["nq"], s["nkv"], s["hd"], s["max_q"], s["max_k"]
    cu, cu_k = s["cu"], s["cu"] if s["cu_k"] is None else s["cu_k"]
    q, k, v = _pad(s["q"], cu, lq, nq, hd), _pad(s["k"], cu_k, lk, nkv, hd), _pad(s["v"], cu_k, lk, nkv, hd)
    n = q.shape[0]
    see = _causal(cu, cu_k, lq, lk)
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


def _store(s, seq, pos, k, v):
    """Rows k, v into the pages of sequences `seq` at positions `pos`."""
    page = s["table"].long()[seq, pos // s["page"]]
    s["kpages"][page, pos % s["page"]] = k.to(TYPES[s["cache"]])
    s["vpages"][page, pos % s["page"]] = v.to(TYPES[s["cache"]])


def _run_decode(s):
    nq, nkv, hd = s["nq"], s["nkv"], s["hd"]
    past = s["past"].long()
    n, rows = past.shape[0], s["table"].shape[1] * s["page"]
    q, k = _rope(s["q"], nq, hd, past), _rope(s["k"], nkv, hd, past)
    _store(s, torch.arange(n, device="cuda"), past, k, s["v"])
    keys, values = (p[s["table"].long()].view(n, rows, nkv, hd).transpose(1, 2).float().contiguous()
                    for p in (s["kpages"], s["vpages"]))
    see = (torch.arange(rows, device="cuda") <= past[:, None])[:, None, None]
    x = _grouped(q.view(n, nq, 1, hd), keys).mul_(hd ** -0.5).masked_fill_(~see, -math.inf)
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    out = torch.matmul(p, values * see.transpose(2, 3)).view(n, -1).to(TYPES[s["t"]])
    return {"out": out, "kpages": s["kpages"], "vpages": s["vpages"]}


def _run_append(s):
    t, cu = TYPES[s["t"]], s["cu"].long()
    r = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu, r, right=True) - 1
    pos = r - cu[seq] + s["past"].long()[seq]
    q, k = _rope(s["q"], s["nq"], s["hd"], pos), _rope(s["k"], s["nkv"], s["hd"], pos)
    _store(s, seq, pos, k, s["v"])
    return {"q": q.to(t), "k": k.to(t), "kpages": s["kpages"], "vpages": s["vpages"]}


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "copy":
        src, dst = (torch.tensor(s[x], device="cuda") for x in ("src", "dst"))
        s["pages_all"][:, dst] = s["pages_all"][:, src]
        return s["pages_all"]
    if op == "prompt":
        return _unpad(_plain_prompt(s)[4], s["cu"], s["q"].shape[0]).to(TYPES[s["t"]])
    return {"train": _run_train, "decode": _run_decode, "append": _run_append}[op](s)


# ---- the definition, in 64 bits ----------------------------------------------------


def _exact_rotated(row, heads, hd, at):
    x = row.double().reshape(heads, hd)
    out = torch.empty_like(x)
    i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    a = at * THETA ** (-2 * i / hd)
    out[:, :hd // 2] = x[:, :hd // 2] * torch.cos(a) - x[:, hd // 2:] * torch.sin(a)
    out[:, hd // 2:] = x[:, hd // 2:] * torch.cos(a) + x[:, :hd // 2] * torch.sin(a)
    return out.reshape(-1)


def _exact_rotated_rows(x, heads, hd, at):
    y = x.double().reshape(-1, heads, hd)
    i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    a = (at.double()[:, None] * THETA ** (-2 * i / hd))[:, None]
    lo, hi = y[..., :hd // 2], y[..., hd // 2:]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1).reshape(x.shape[0], -1)


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
        hidden = torch.ones((a, b), dtype=torch.bool, device="cuda").triu(b - a + 1)
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


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "copy":
        pages = s["pages_all"]
        for a, b in zip(s["src"], s["dst"]):
            pages[:, b] = pages[:, a]
        return pages
    if op in ("prompt", "train"):
        return _exact_attend(case, s)
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    lens = _ints(case["lens"])
    kp, vp = s["kpages"].double(), s["vpages"].double()
    table = s["table"].tolist()
    if op == "append":
        past, pos, pages = _ints(case["past"]), [], []
        for b, n in enumerate(lens):
            pos += range(past[b], past[b] + n)
            pages += [table[b][x // page] for x in range(past[b], past[b] + n)]
        pos, pages = torch.tensor(pos, device="cuda"), torch.tensor(pages, device="cuda")
        q, k = _exact_rotated_rows(s["q"], nq, hd, pos), _exact_rotated_rows(s["k"], nkv, hd, pos)
        kp[pages, pos % page], vp[pages, pos % page] = k, s["v"].double()
        return {"q": q, "k": k, "kpages": kp, "vpages": vp}
    out = torch.empty((len(lens), nq * hd), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        last = (table[b][n // page], n % page)
        # the new row is stored in the cache's type and attended as it is stored
        kp[last], vp[last] = _exact_rotated(s["k"][b], nkv, hd, n), s["v"][b].double()
        mine = s["table"][b].long()
        keys, values = (p[mine].reshape(-1, nkv, hd)[:n + 1].clone() for p in (kp, vp))
        keys[n], values[n] = (x[last].to(TYPES[case["cache"]]).double().view(nkv, hd) for x in (kp, vp))
        q = _exact_rotated(s["q"][b], nq, hd, n).view(nq, hd)
        for h in range(nq):
            g = h // (nq // nkv)
            p = torch.softmax(keys[:, g] @ q[h] / math.sqrt(hd), 0)
            out[b, h * hd:h * hd + hd] = p @ values[:, g]
    return {"out": out, "kpages": kp, "vpages": vp}
