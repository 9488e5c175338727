"""A key-value cache in pages for a batch of sequences: what the decoder layers'
prefill and step_paged run on.

The pages of all layers lie in one tensor [2 * layers, pages, page_size,
n_kv * head_dim] (a layer's keys, then its values), so one pages_copy moves a
page in every layer. A page number means the same place in every plane. Which
sequence holds which pages is kept on the host: pages have reference counts, so
a fork shares those with rows in them, and the last, part-filled page is copied when one of
its holders reserves room to go on writing (copy-on-write), or at the fork when the sequence
has reserved room in it already. So rows are reserved, then appended, and a reservation
holds until its rows are used up, forks or not. The sequences' page table and lengths are uploaded
when they have changed, on the current stream; a graph captured over the device
arrays goes on reading them, so its replays follow later changes. One cache is used
by one thread and on one stream at a time.

With dtype int8 the rows are codes, and `scales` holds one f32 scale for each 16 rows and KV head, in
every plane beside the pages; they are copied and moved together. Rows of 128 elements a head take
0.501 of bf16 ones' bytes (0.504 at most, with the scales of a page filled up to 16 bytes).
"""
from __future__ import annotations

import heapq
from typing import NamedTuple

import numpy as np

from .attention import pages_copy, pages_rows
from .quant import Context, _need, _t

__all__ = ["PagedCache", "PagedView"]


class PagedView(NamedTuple):
    """Some sequences of a cache, in the order of a batch: device arrays for the operators."""

    table: object   # int32 [batch, pages of a sequence]
    lens: object    # int32 [batch], rows stored
    max_len: int    # no sequence has more rows (paged_attention's max_len)


class _SeqsView(PagedView):
    """A view of chosen sequences, which step_paged looks up again."""

    seqs: tuple = ()


class _Pages(list):
    """A sequence's pages."""

    room = 0  # rows that it has reserved, those stored included


class PagedCache:
    scales = None  # int8: f32 [2 * layers, pages, 1, scales of a page]

    def __init__(self, ctx: Context, layers: int, pages: int, n_kv: int, head_dim: int, page_size: int = 16,
                 max_seqs: int = 16, seq_pages: int | None = None, dtype=None):
        """max_seqs sequences of at most seq_pages pages each (default: all of them). dtype:
        f32 (default), bf16 or int8."""
        torch = _t()
        _need(layers > 0 and pages > 0 and max_seqs > 0, "layers, pages and max_seqs must be positive")
        _need(page_size >= 16 and page_size & (page_size - 1) == 0, "page_size must be a power of two from 16 on")
        self.ctx, self.layers, self.n_kv, self.head_dim, self.page_size = ctx, layers, n_kv, head_dim, page_size
        dev = torch.device("cuda", ctx.device)
        self.data = torch.zeros((2 * layers, pages, page_size, n_kv * head_dim), dtype=dtype or torch.float32,
                                device=dev)
        if self.data.dtype == torch.int8:  # (a page's scales end at a multiple of 16 bytes, for the copies)
            self.scales = torch.zeros((2 * layers, pages, 1, (page_size // 16 * n_kv + 3) // 4 * 4), device=dev)
        self._refs = [0] * pages
        self._free = list(range(pages))  # a heap: the lowest page first
        self._pages: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._slots = list(range(max_seqs))
        self._host_table = np.full((max_seqs, seq_pages or pages), -1, np.int32)  # (-1: no page, refused by the operators)
        self._host_lens = np.full(max_seqs, -1, np.int32)
        self._table = torch.full(self._host_table.shape, -1, dtype=torch.int32, device=dev)
        self._lens = torch.full((max_seqs,), -1, dtype=torch.int32, device=dev)
        self._dirty = False

    # ---- the operators' arrays -------------------------------------------------
    def kpages(self, layer: int):
        return self.data[2 * layer]

    def vpages(self, layer: int):
        return self.data[2 * layer + 1]

    def layer_scales(self, layer: int) -> dict:
        """The operators' kscales and vscales for a layer's pages; {} but for int8."""
        if self.scales is None:
            return {}
        shape = (self.data.shape[1], self.page_size // 16, self.n_kv)
        return {name: plane[:, 0, :shape[1] * shape[2]].unflatten(1, shape[1:])
                for name, plane in (("kscales", self.scales[2 * layer]), ("vscales", self.scales[2 * layer + 1]))}

    def _copy(self, src, dst) -> None:
        pages_copy(self.ctx, self.data, src, dst)
        if self.scales is not None:
            pages_copy(self.ctx, self.scales, src, dst)

    def view(self, seqs=None, max_len: int | None = None) -> PagedView:
        """The device arrays of `seqs`, as of now; None: of all slots, those without a
        sequence idle, and following the cache's later changes from the next view() or sync()
        on (a captured graph's view). max_len defaults to the rows that the sequences
        have pages for; of all slots, to the rows that the table can hold: a step is planned
        for it, so give the largest length that is served, or seq_pages, when that is far less
        (32 sequences of 1000 rows: 32 us planned for 1001 rows, 40 for 65536, 287 for 1 Mi)."""
        seqs = None if seqs is None else self._different(seqs)
        self.sync()
        if seqs is None:
            rows = self._host_table.shape[1] * self.page_size
            table, lens = self._table, self._lens
        else:
            rows = max((len(self._pages[self._known(s)]) for s in seqs), default=0) * self.page_size
            at = _t().tensor(seqs, dtype=_t().long, device=self._table.device)
            table, lens = self._table[at], self._lens[at]
        view = (PagedView if seqs is None else _SeqsView)(table, lens, rows if max_len is None else max_len)
        if seqs is not None:
            view.seqs = tuple(seqs)
        return view

    def sync(self) -> None:
        """Uploads the page table and the lengths if they have changed."""
        if self._dirty:
            torch = _t()
            self._table.copy_(torch.from_numpy(self._host_table))
            self._lens.copy_(torch.from_numpy(self._host_lens))
            self._dirty = False

    # ---- sequences -----------------------------------------------------------------
    def _known(self, seq: int) -> int:
        if seq not in self._pages:
            raise ValueError(f"sequence {seq} is not in the cache")
        return seq

    def _different(self, seqs) -> list:
        seqs = list(seqs)
        _need(len(set(seqs)) == len(seqs), "a sequence may stand in a batch once")
        return seqs

    def length(self, seq: int) -> int:
        return self._len[self._known(seq)]

    def free_pages(self) -> int:
        return len(self._free)

    def add(self) -> int:
        """A new, empty sequence -> its number (a slot of the page table)."""
        if not self._slots:
            raise RuntimeError("the cache has no free slot for a sequence")
        seq = heapq.heappop(self._slots)
        self._pages[seq], self._len[seq] = _Pages(), 0
        self._host_lens[seq] = 0
        self._dirty = True
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence with the rows of `seq`, on the same pages. Room that `seq` has reserved
        stays its own: the new sequence reserves for itself, and gets a copy of a part-filled
        page in which `seq` has room (RuntimeError when no page is free for it)."""
        pages, n = self._pages[self._known(seq)], self._len[seq]
        own = n % self.page_size > 0 and pages.room > n
        if own and not self._free:
            raise RuntimeError("the cache is full: a page is wanted for the fork")
        new = self.add()
        held = _Pages(pages[:-(-n // self.page_size)])
        for p in held[:-1] if own else held:
            self._refs[p] += 1
        if own:
            held[-1] = self._take()
            self._copy([pages[len(held) - 1]], [held[-1]])
        held.room = n
        self._pages[new], self._len[new] = held, n
        self._host_table[new, :len(held)] = held
        self._host_lens[new] = n
        return new

    def reserve(self, seqs, rows) -> None:
        """Room for `rows` more rows (a number, or one a sequence) of each sequence: pages
        of its own from the row it goes on at. All or nothing: RuntimeError when there
        are not enough pages, ValueError when a sequence would outgrow the table."""
        seqs = self._different(seqs)
        rows = [rows] * len(seqs) if isinstance(rows, int) else list(rows)
        _need(len(rows) == len(seqs), "one number of rows for each sequence")
        want, refs = 0, {}
        plan = []
        for s, n in zip(seqs, rows):
            have, used = self._pages[self._known(s)], self._len[s]
            _need(n >= 0, "rows must not be negative")
            total = -(-(used + n) // self.page_size)
            _need(total <= self._host_table.shape[1], f"sequence {s} would outgrow its {self._host_table.shape[1]} pages")
            # pages that rows will be written to and somebody else holds: the last holder keeps it
            shared = []
            for i in range(used // self.page_size, len(have)) if n > 0 else ():
                left = refs.get(have[i], self._refs[have[i]])
                if left > 1:
                    refs[have[i]] = left - 1
                    shared.append(i)
            plan.append((s, shared, max(0, total - len(have))))
            want += len(shared) + plan[-1][2]
        if want > len(self._free):
            raise RuntimeError(f"the cache is full: {want} pages are wanted, {len(self._free)} are free")
        src, dst = [], []
        for s, shared, more in plan:
            for i in shared:
                old, new = self._pages[s][i], self._take()
                src.append(old)
                dst.append(new)
                self._refs[old] -= 1
                self._pages[s][i] = new
            self._pages[s].extend(self._take() for _ in range(more))
            self._host_table[s, :len(self._pages[s])] = self._pages[s]
            self._dirty |= bool(shared or more)
        for s, n in zip(seqs, rows):
            self._pages[s].room = max(self._pages[s].room, self._len[s] + n)
        if src:
            self._copy(src, dst)

    def need_own(self, seqs, rows=1) -> None:
        """ValueError when the next rows (a number, or one a sequence) of one of `seqs` would go to a page
        that another sequence holds too: a fork after which neither has reserved. Rows without a page are not
        looked at (the operators give NaN for them)."""
        rows = [rows] * len(seqs) if isinstance(rows, int) else rows
        for s, n in zip(seqs, rows):
            pages, at = self._pages[self._known(s)], self._len[s]
            for p in pages[at // self.page_size:-(-(at + n) // self.page_size)] if n > 0 else ():
                _need(self._refs[p] == 1, f"sequence {s} shares the page of its next rows: reserve them first")

    def advance(self, seqs, rows) -> None:
        """The rows that the operators have appended now count."""
        seqs = self._different(seqs)
        rows = [rows] * len(seqs) if isinstance(rows, int) else list(rows)
        _need(len(rows) == len(seqs), "one number of rows for each sequence")
        for s, n in zip(seqs, rows):
            _need(0 <= n <= len(self._pages[self._known(s)]) * self.page_size - self._len[s],
                  f"sequence {s} has no pages for {n} more rows")
        self.need_own(seqs, rows)
        for s, n in zip(seqs, rows):
            self._len[s] += n
            self._host_lens[s] = self._len[s]
        self._dirty = True

    def free(self, seq: int) -> None:
        """Ends a sequence; pages that no other holds are free again."""
        for p in self._pages.pop(self._known(seq)):
            self._drop(p)
        del self._len[seq]
        self._host_lens[seq], self._host_table[seq] = -1, -1
        heapq.heappush(self._slots, seq)
        self._dirty = True

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers -> how many are in use."""
        used = [p for p, n in enumerate(self._refs) if n]
        src = [p for p in used if p >= len(used)]
        dst = [p for p in range(len(used)) if not self._refs[p]]
        if src:
            self._copy(src, dst)
            to = dict(zip(src, dst))
            for old, new in to.items():
                self._refs[new], self._refs[old] = self._refs[old], 0
            for s, pages in self._pages.items():
                pages[:] = [to.get(p, p) for p in pages]
                self._host_table[s, :len(pages)] = pages
            self._free = list(range(len(used), len(self._refs)))
            self._dirty = True
        return len(used)

    def rows(self, layer: int, seqs, more=0, dtype=None):
        """The stored rows of `seqs`, one after another, and `more` (a number, or one a
        sequence) behind each that are appended but not advanced over yet: (keys, values)
        [rows, n_kv * head_dim], copies, of `dtype` (f32 or bf16; default the cache's, f32 for int8)."""
        torch = _t()
        seqs = list(seqs)
        more = [more] * len(seqs) if isinstance(more, int) else list(more)
        _need(len(more) == len(seqs), "one number of rows for each sequence")
        lens = [self._len[self._known(s)] + n for s, n in zip(seqs, more)]
        for s, n in zip(seqs, lens):
            _need(0 <= n <= len(self._pages[s]) * self.page_size, f"sequence {s} has no {n} rows")
        if dtype is None:
            dtype = torch.float32 if self.scales is not None else self.data.dtype
        if not self._for_operators():
            at = [np.arange(n) % self.page_size + np.repeat(np.array(self._pages[s], np.int64), self.page_size)[:n] * self.page_size
                  for s, n in zip(seqs, lens)]
            at = torch.from_numpy(np.concatenate([np.zeros(0, np.int64), *at])).to(self.data.device)
            return tuple(x.view(-1, x.shape[-1])[at].to(dtype) for x in (self.kpages(layer), self.vpages(layer)))
        calls = self._cut(seqs, lens)
        if len(calls) == 1:
            return self._rows(layer, *calls[0], dtype)
        k, v = (torch.empty((sum(lens), self.n_kv * self.head_dim), dtype=dtype, device=self.data.device) for _ in range(2))
        done = 0
        for call in calls:
            part = slice(done, done + sum(call[2]))
            self._rows(layer, *call, dtype, k_out=k[part], v_out=v[part])
            done = part.stop
        return k, v

    def _rows(self, layer: int, seqs, page: int, lens, dtype, **out):
        """lens[i] rows of seqs[i] from page number `page` of it on (not 0: of one sequence). Page numbers and row numbers
        go to the device in one copy (as two, with the table looked up there: one sequence of 40 rows 55 us, so 33)."""
        wide = -(-max(lens, default=0) // self.page_size)
        table = self._host_table[seqs, page:page + wide] if seqs else np.zeros((0, 0), np.int32)
        ids = np.concatenate([table.ravel(), np.cumsum([0] + lens, dtype=np.int32)])
        ids = _t().from_numpy(ids).to(self.data.device)
        table, cu = ids[:table.size].view(table.shape), ids[table.size:]
        return pages_rows(self.ctx, self.kpages(layer), self.vpages(layer), table, cu, sum(lens), self.n_kv,
                          self.head_dim, dtype, **out, **self.layer_scales(layer))

    def _cut(self, seqs, lens) -> list:
        """The rows of seqs in turn as (sequences, first page, rows of each), a pages_rows each, which takes fewer than
        2^24 rows: many sequences from their first page on, or pages of a longer one."""
        most = (1 << 24) - 1
        whole = most // self.page_size * self.page_size
        calls, room = [], -1
        for s, n in zip(seqs, lens):
            if n > whole:
                calls += [([s], r // self.page_size, [min(whole, n - r)]) for r in range(0, n, whole)]
                room = -1
            elif n <= room:
                calls[-1][0].append(s)
                calls[-1][2].append(n)
                room -= n
            else:
                calls.append(([s], 0, [n]))
                room = most - n
        return calls or [([], 0, [])]

    def _for_operators(self) -> bool:
        """Whether the operators take the cache's pages: others are a place for rows only."""
        torch = _t()
        return (self.data.dtype in (torch.float32, torch.bfloat16, torch.int8) and self.head_dim % 8 == 0
                and self.head_dim <= 256 and self.page_size <= 65536 and self.n_kv <= 65535
                and self.n_kv * self.head_dim <= 1 << 22)

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._refs[p] = 1
        return p

    def _drop(self, p: int) -> None:
        self._refs[p] -= 1
        if self._refs[p] == 0:
            heapq.heappush(self._free, p)
