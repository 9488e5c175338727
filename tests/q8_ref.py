"""The 8-bit cache's append in plain torch, f32 operation by operation: what include/rq.h says, one block at a time."""
import torch

BLOCK = 16


def put(codes, scales, row, x):
    """Rows x [n, heads, hd] (f32) behind the first `row` ones of codes [blocks, 16, heads, hd] int8 and scales
    [blocks, heads] f32, in place."""
    i = 0
    while i < len(x):
        b, r = divmod(row + i, BLOCK)
        part = x[i:i + BLOCK - r]
        s0 = scales[b] if r else torch.zeros_like(scales[b])
        fin = torch.isfinite(part).all(2).all(0) & torch.isfinite(s0)
        s = torch.maximum(s0, part.abs().amax((0, 2)) * torch.tensor(1 / 127, device=x.device))
        s = torch.where(fin, s, torch.full_like(s, float("nan")))
        rises = s > s0
        ratio = torch.where(rises, s0 / s, torch.ones_like(s))
        codes[b, :r] = torch.round(codes[b, :r].float() * ratio[:, None]).to(torch.int8)
        y = torch.where((s > 0)[:, None], part / s[:, None], torch.zeros_like(part))
        codes[b, r:r + len(part)] = torch.round(y).clamp(-127, 127).to(torch.int8)
        scales[b] = s
        i += len(part)


class Cache:
    """int8 pages and their scales, shuffled, with sequences of `need` rows; `free` further pages."""

    def __init__(self, seed, nkv, hd, need, page, fill, pad=0, spare=2):
        """fill[b]: rows of sequence b that are there, from N(0, 1). pad: floats between the pages' scales."""
        g = torch.Generator(device="cuda").manual_seed(seed)
        pages = [-(-n // page) for n in need]
        total = sum(pages) + spare
        ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(need), max(max(pages), 0) + 1), 2 ** 30, dtype=torch.int32)
        for b, n in enumerate(pages):
            table[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
        self.nkv, self.hd, self.page, self.table = nkv, hd, page, table.cuda()
        self.k, self.v = (torch.randint(-128, 128, (total, page, nkv * hd), generator=g, device="cuda",
                                        dtype=torch.int32).to(torch.int8) for _ in range(2))
        per = page // BLOCK * nkv
        self._s = torch.full((2, total, per + pad), float("nan"), device="cuda")
        self.ks, self.vs = (s[:, :per].view(total, page // BLOCK, nkv) if pad == 0 else
                            s.as_strided((total, page // BLOCK, nkv), (per + pad, nkv, 1), s.storage_offset())
                            for s in self._s)
        for b, n in enumerate(fill):
            if n > 0:
                for which in "kv":
                    self.append(which, b, 0, torch.randn((n, nkv, hd), generator=g, device="cuda"))

    def clone(self):
        c = object.__new__(Cache)
        c.__dict__.update(self.__dict__)
        c.k, c.v, c._s = self.k.clone(), self.v.clone(), self._s.clone()
        c.ks, c.vs = (s.as_strided(self.ks.shape, self.ks.stride(), s.storage_offset()) for s in c._s)
        return c

    def scales(self):
        return dict(kscales=self.ks, vscales=self.vs)

    def _mine(self, b, n):
        return self.table[b, :-(-n // self.page)].long()

    def _of(self, which):
        return (self.k, self.ks) if which == "k" else (self.v, self.vs)

    def append(self, which, b, row, x):
        mine = self._mine(b, row + len(x))
        pages, scales = self._of(which)
        codes, sc = pages[mine].view(-1, BLOCK, self.nkv, self.hd), scales[mine].reshape(-1, self.nkv)
        put(codes, sc, row, x)
        pages[mine], scales[mine] = codes.view(-1, self.page, self.nkv * self.hd), sc.view(len(mine), -1, self.nkv)

    def values(self, which, b, n):
        """Rows 0 .. n - 1 of sequence b, f64 [n, nkv, hd]."""
        mine = self._mine(b, n)
        pages, scales = self._of(which)
        codes, sc = pages[mine].view(-1, BLOCK, self.nkv, self.hd), scales[mine].reshape(-1, self.nkv)
        return (codes.double() * sc.double()[:, None, :, None]).reshape(-1, self.nkv, self.hd)[:n]

    def same(self, other):
        """Whether all bits are other's, NaN scales alike."""
        return (torch.equal(self.k, other.k) and torch.equal(self.v, other.v)
                and torch.equal(self._s.nan_to_num(-7.0), other._s.nan_to_num(-7.0)))


def rope32(x, pos, theta):
    """x [rows, heads, hd] f32 rotated in f32 operation by operation, from angles in 64 bits."""
    if not theta:
        return x
    hd = x.shape[-1]
    f = theta ** (-2 * torch.arange(hd // 2, dtype=torch.float64, device=x.device) / hd)
    a = (pos.double()[:, None] * f)[:, None]
    c, s = a.cos().float(), a.sin().float()
    lo, hi = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
