"""How PagedCache.rows divides its rows over calls, on the CPU."""
import random

import pytest

import raster_amd.paged as paged

MOST = (1 << 24) - 1


@pytest.mark.parametrize("page", [16, 512, 65536])
def test_cut(page):
    c = object.__new__(paged.PagedCache)
    c.page_size = page
    rng = random.Random(page)
    cases = [[], [0], [5, 0, 7], [MOST], [MOST + 1], [MOST, 0, 1], [1, MOST], [3 * MOST, 5], [page] * 40, [0, 2 ** 31]]
    cases += [[rng.choice([0, 3, 10 ** 6, 9 * 10 ** 6, 2 ** 24, 4 * 10 ** 7]) for _ in range(rng.randint(1, 9))]
              for _ in range(200)]
    for lens in cases:
        seqs = [rng.randint(0, 3) for _ in lens]  # (a sequence may come again)
        calls = c._cut(seqs, lens)
        assert len(calls) >= 1
        got = []
        for ss, first, ns in calls:
            assert len(ss) == len(ns) and sum(ns) <= MOST and (first == 0 or len(ss) == 1)
            got += [(s, first * page, n) for s, n in zip(ss, ns)]
        it = iter(got)
        for s, n in zip(seqs, lens):  # in turn, each from its first row to its last
            at = 0
            while True:
                s1, first, m = next(it)
                assert s1 == s and first == at
                at += m
                if at == n:
                    break
        assert next(it, None) is None
        if sum(lens) <= MOST and all(n <= MOST // page * page for n in lens):
            assert len(calls) == 1
