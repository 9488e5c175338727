"""PagedCache's bookkeeping on the CPU: the pages' counts, copies and moves, with the
copies themselves recorded in place of pages_copy (which needs a GPU)."""
import random

import numpy as np
import pytest

import raster_amd.paged as paged


class Ctx:
    device = 0


class Cache(paged.PagedCache):
    """The host side alone, with every row's content modelled as (sequence's history)."""

    def __init__(self, pages, page_size=16, max_seqs=8, seq_pages=6):
        self.ctx, self.page_size = Ctx(), page_size
        self.data = np.zeros((pages, page_size), np.int64)
        self._refs, self._free = [0] * pages, list(range(pages))
        self._pages, self._len, self._slots = {}, {}, list(range(max_seqs))
        self._host_table = np.full((max_seqs, seq_pages), -1, np.int32)
        self._host_lens = np.full(max_seqs, -1, np.int32)
        self._dirty = False


@pytest.fixture
def copies(monkeypatch):
    done = []

    def fake(ctx, data, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        data[dst] = data[src]
        done.append((list(src), list(dst)))

    monkeypatch.setattr(paged, "pages_copy", fake)
    return done


def check(c):
    held = [p for pages in c._pages.values() for p in pages]
    assert [held.count(p) for p in range(len(c._refs))] == c._refs
    assert sorted(c._free) == [p for p, n in enumerate(c._refs) if n == 0]
    for s, pages in c._pages.items():
        assert len(set(pages)) == len(pages) and len(pages) * c.page_size >= c._len[s]
        assert list(c._host_table[s, :len(pages)]) == pages and np.all(c._host_table[s, len(pages):] == -1)
        assert c._host_lens[s] == c._len[s]
    assert all(c._host_lens[s] == -1 and np.all(c._host_table[s] == -1) for s in c._slots)


def write(c, s, values):
    for v in values:
        n = c._len[s]
        p = c._pages[s][n // c.page_size]
        assert c._refs[p] == 1, "a shared page is written"
        c.data[p, n % c.page_size] = v
        c.advance([s], 1)


def read(c, s):
    return [int(c.data[c._pages[s][i // c.page_size], i % c.page_size]) for i in range(c._len[s])]


def test_fork_copies_the_part_filled_page_once(copies):
    c = Cache(10)
    a = c.add()
    c.reserve([a], 20)
    write(c, a, range(20))
    b = c.fork(a)
    assert c._pages[a] == c._pages[b] and not copies
    c.reserve([a, b], 1)  # one of the two keeps the page, the other gets a copy
    assert len(copies) == 1 and len(copies[0][0]) == 1
    write(c, a, [100])
    write(c, b, [200])
    assert read(c, a) == [*range(20), 100] and read(c, b) == [*range(20), 200]
    check(c)
    c.reserve([a, b], 1)
    assert len(copies) == 1
    c.free(a)
    check(c)
    assert read(c, b) == [*range(20), 200]


def test_full_pages_stay_shared(copies):
    c = Cache(10)
    a = c.add()
    c.reserve([a], 32)
    write(c, a, range(32))
    b = c.fork(a)
    c.reserve([b], 5)
    assert not copies and c._pages[b][:2] == c._pages[a]
    check(c)


def test_refusals_change_nothing(copies):
    c = Cache(3, max_seqs=2, seq_pages=2)
    a = c.add()
    with pytest.raises(ValueError):
        c.reserve([a], 33)  # outgrows the table
    b = c.add()
    with pytest.raises(RuntimeError):
        c.add()
    with pytest.raises(RuntimeError):
        c.reserve([a, b], 32)  # four pages of three
    assert c.free_pages() == 3 and not c._pages[a]
    with pytest.raises(ValueError):
        c.reserve([a, a], 1)
    with pytest.raises(ValueError):
        c.reserve([a], -1)
    with pytest.raises(ValueError):
        c.advance([a], 1)  # nothing reserved
    with pytest.raises(ValueError):
        c.advance([a, a], 0)
    with pytest.raises(ValueError):
        c.view([a, a])
    with pytest.raises(ValueError):
        c.free(7)
    with pytest.raises(ValueError):
        c.fork(7)
    check(c)


def test_compact(copies):
    c = Cache(12)
    seqs = [c.add() for _ in range(5)]
    for i, s in enumerate(seqs):
        c.reserve([s], 17 + i)
        write(c, s, range(100 * i, 100 * i + 17 + i))
    for s in seqs[::2]:
        c.free(s)
    f = c.fork(seqs[3])
    want = {s: read(c, s) for s in (seqs[1], seqs[3], f)}
    assert c.compact() == 4
    assert all(p < 4 for pages in c._pages.values() for p in pages)
    assert {s: read(c, s) for s in want} == want
    check(c)
    assert c.compact() == 4  # nothing left to move
    assert len(copies) == 1


def test_random_histories(copies):
    rng = random.Random(3)
    for _ in range(60):
        c = Cache(rng.randint(4, 30), max_seqs=rng.randint(2, 6), seq_pages=rng.randint(2, 5))
        want, k = {}, 0
        for _ in range(120):
            op = rng.choice(["add", "write", "write", "write", "fork", "free", "compact"])
            live = list(want)
            try:
                if op == "add":
                    want[c.add()] = []
                elif op == "write" and live:
                    some = rng.sample(live, rng.randint(1, len(live)))
                    rows = [rng.randint(0, 20) for _ in some]
                    c.reserve(some, rows)
                    for s, n in zip(some, rows):
                        write(c, s, range(k, k + n))
                        want[s] = want[s] + list(range(k, k + n))
                        k += n
                elif op == "fork" and live:
                    s = rng.choice(live)
                    n = c.fork(s)
                    want[n] = list(want[s])
                elif op == "free" and live:
                    s = rng.choice(live)
                    c.free(s)
                    del want[s]
                elif op == "compact":
                    c.compact()
            except (RuntimeError, ValueError):
                pass  # full: nothing may have changed
            check(c)
            assert {s: read(c, s) for s in want} == want


def test_a_fork_leaves_rows_reserved_ahead_to_their_sequence(copies):
    """Rows reserved before a fork stay the sequence's own; the fork shares only pages with rows, and none
    that somebody may go on writing to."""
    c = Cache(10)
    a = c.add()
    c.reserve([a], 40)
    write(c, a, range(20))
    b = c.fork(a)
    assert c._pages[b][:1] == c._pages[a][:1] and len(c._pages[b]) == 2 and len(copies) == 1
    write(c, a, range(100, 120))  # as reserved, over the page's end
    write(c, b, range(200, 212))  # its own copy of the part-filled page
    assert read(c, a) == [*range(20), *range(100, 120)] and read(c, b) == [*range(20), *range(200, 212)]
    check(c)
    with pytest.raises(ValueError):
        c.advance([b], 1)  # the next page was a's reservation, not b's
    c.free(a)
    c.free(b)
    assert c.free_pages() == 10


def test_rows_do_not_count_on_a_page_that_another_holds(copies):
    c = Cache(10)
    a = c.add()
    c.reserve([a], 20)
    write(c, a, range(20))
    b = c.fork(a)
    for seqs in ([a], [b], [a, b]):
        with pytest.raises(ValueError):
            c.advance(seqs, 1)
        with pytest.raises(ValueError):
            c.need_own(seqs, 1)
    assert c.length(a) == c.length(b) == 20
    c.need_own([a, b], 0)
    c.reserve([b], 1)  # b's copy: the page is a's alone again
    c.need_own([a, b], 1)
    write(c, a, [100])
    write(c, b, [200])
    check(c)


def test_a_fork_that_wants_a_page_of_a_full_cache_changes_nothing(copies):
    c = Cache(2)
    a = c.add()
    c.reserve([a], 32)
    write(c, a, range(5))
    with pytest.raises(RuntimeError):
        c.fork(a)
    check(c)
    assert len(c._pages) == 1 and not copies
    write(c, a, range(5, 16))
    b = c.fork(a)  # no part-filled page
    assert read(c, b) == list(range(16)) and not copies
    check(c)


def test_random_histories_with_rows_reserved_ahead(copies):
    """Rows written later than they are reserved, with forks, ends and compaction between: no page with two
    holders is ever written (write() looks), whoever reserved."""
    rng = random.Random(4)
    for _ in range(60):
        c = Cache(rng.randint(6, 30), max_seqs=rng.randint(2, 6), seq_pages=rng.randint(2, 5))
        want, room, k = {}, {}, 0
        for _ in range(150):
            op = rng.choice(["add", "reserve", "reserve", "write", "write", "write", "fork", "free", "compact"])
            live = list(want)
            try:
                if op == "add":
                    s = c.add()
                    want[s], room[s] = [], 0
                elif op == "reserve" and live:
                    some = rng.sample(live, rng.randint(1, len(live)))
                    rows = [rng.randint(0, 30) for _ in some]
                    c.reserve(some, rows)
                    for s, n in zip(some, rows):
                        room[s] = max(room[s], len(want[s]) + n)
                elif op == "write" and live:
                    s = rng.choice(live)
                    n = rng.randint(0, room[s] - len(want[s]))
                    write(c, s, range(k, k + n))
                    want[s] = want[s] + list(range(k, k + n))
                    k += n
                elif op == "fork" and live:
                    s = rng.choice(live)
                    n = c.fork(s)
                    want[n], room[n] = list(want[s]), len(want[s])
                elif op == "free" and live:
                    s = rng.choice(live)
                    c.free(s)
                    del want[s], room[s]
                elif op == "compact":
                    c.compact()
            except RuntimeError:
                pass  # full
            except ValueError:
                assert op == "reserve"  # would outgrow the table
            check(c)
            assert {s: read(c, s) for s in want} == want


def test_a_view_unpacks_into_three():
    table, lens, max_len = paged.PagedView(1, 2, 3)
    assert (table, lens, max_len) == (1, 2, 3)
    view = paged._SeqsView(1, 2, 3)
    view.seqs = (4, 5)
    table, lens, max_len = view
    assert view == paged.PagedView(1, 2, 3) and view.seqs == (4, 5) and isinstance(view, paged.PagedView)
