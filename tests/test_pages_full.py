"""Rewinding sequences of a full cache: the pages that the call frees serve its own copies."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def sat():
    from satori_b200 import build
    build.build()
    import satori_b200
    return satori_b200


def _full(sat, pages):
    return sat.PagedCache(1, pages, 16, 1, 64, ctx=False)


def test_a_child_makes_room_in_a_full_cache(sat):
    c = _full(sat, 8)
    a = c.create(1)[0]
    c.extend([a], [48])
    child = c.fork([a])[0]
    c.extend([child], [80])                                   # 8 pages, 3 of them shared
    assert c.info()["free"] == 0 and c.length(child) == 128
    c.rewind([child], [40])
    assert c.length(child) == 40 and c.table(child).tolist() == [0, 1, 3] and c.copies().tolist() == [[2, 3]]
    assert c.info()["free"] == 4


def test_sharers_that_go_back_together(sat):
    """Copies are needed for all sharers but the last; the pages that all of them leave are free first."""
    c = _full(sat, 6)
    a = c.create(1)[0]
    c.extend([a], [96])
    b, d = c.fork([a, a])
    assert c.info()["free"] == 0
    c.rewind([a, b, d], [20, 30, 25])
    assert [c.table(x).tolist() for x in (a, b, d)] == [[0, 2], [0, 3], [0, 1]]
    assert c.copies().tolist() == [[1, 2], [1, 3]] and c.info()["free"] == 2


def test_what_frees_no_page_is_refused(sat):
    c = _full(sat, 4)
    a = c.create(1)[0]
    c.extend([a], [64])
    b, d = c.fork([a, a])
    for call in (([b], [20]), ([b, d], [20, 63]), ([a, b, d], [63, 62, 61])):
        with pytest.raises(sat.ContextFullError):
            c.rewind(*call)
        assert [c.length(x) for x in (a, b, d)] == [64] * 3 and c.info()["used"] == 4
    c.rewind([b, d], [48, 0])                                 # no copy at all
    assert c.length(b) == 48 and c.length(d) == 0


def test_random_rewinds_near_the_limit(sat):
    """Against the same tables with room to spare: what is taken gives the same lengths and contents, what is refused
    would not have freed a page."""
    rng = np.random.default_rng(11)
    taken = refused = 0
    for _ in range(300):
        c = _full(sat, 12)
        roots = c.create(2)
        c.extend(roots, [int(rng.integers(1, 70)), int(rng.integers(1, 40))])
        seqs = list(roots)
        try:
            for _ in range(5):
                p = int(rng.choice(seqs))
                seqs += c.fork([p], [int(rng.integers(c.length(p) + 1))])
                c.extend(seqs[-1:], [int(rng.integers(0, 30))])
        except sat.ContextFullError:
            pass
        some = [int(s) for s in rng.permutation(seqs)[:3]]
        at = [int(rng.integers(c.length(s) + 1)) for s in some]
        before = {s: (c.length(s), c.table(s).tolist()) for s in seqs}
        free = c.info()["free"]
        try:
            c.rewind(some, at)
        except sat.ContextFullError:
            refused += 1
            assert {s: (c.length(s), c.table(s).tolist()) for s in seqs} == before
            continue
        taken += 1
        pairs = dict(c.copies()[:, ::-1].tolist())
        assert len(pairs) <= free or c.info()["free"] > free
        for s in seqs:
            n = at[some.index(s)] if s in some else before[s][0]
            table = c.table(s).tolist()
            assert c.length(s) == n and len(table) == -(-n // 16)
            assert [pairs.get(p, p) if p not in before[s][1] or p in pairs else p for p in table] == before[s][1][:len(table)]
        held = {p for s in seqs for p in c.table(s).tolist()}
        assert c.info()["used"] == len(held)
    assert taken > 100
