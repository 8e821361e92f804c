"""The paged cache's tables and a batch's plan on the CPU (a cache without a context keeps its tables only):
page numbers, sharing, copies to make, all-or-nothing errors and refusals."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def sat():
    from satori_b200 import build
    build.build()
    import satori_b200
    return satori_b200


def _cache(sat, pages=32, page_tokens=16, **kw):
    return sat.PagedCache(2, pages, page_tokens, 2, 64, ctx=False, **kw)


def test_lowest_free_page_first(sat):
    c = _cache(sat)
    a, b = c.create(2)
    c.extend([a, b], [17, 16])
    assert c.table(a).tolist() == [0, 1] and c.table(b).tolist() == [2]
    c.free([a])
    c.extend([b], [40])                                       # 56 tokens: three more pages
    assert c.table(b).tolist() == [2, 0, 1, 3]
    assert c.length(b) == 56 and c.info()["used"] == 4 and c.info()["top"] == 4


@pytest.mark.parametrize("at", [0, 1, 15, 16, 17, 32, 40])
def test_fork_shares_full_pages_and_copies_the_tail(sat, at):
    c = _cache(sat)
    root = c.create(1)
    c.extend(root, [40])
    child = c.fork(root, [at])[0]
    whole = at // 16
    assert c.length(child) == at
    table = c.table(child).tolist()
    assert table[:whole] == [0, 1, 2][:whole]
    assert c.copies().tolist() == ([[whole, 3]] if at % 16 else [])
    assert table[whole:] == ([3] if at % 16 else [])
    c.free(root)                                              # shared pages outlive the parent
    assert c.info()["used"] == len(table)
    c.extend([child], [1])
    assert c.length(child) == at + 1


def test_copy_shares_nothing(sat):
    c = _cache(sat)
    root = c.create(1)
    c.extend(root, [33])
    two = c.copy(root * 2, [33, 20])
    assert c.table(two[0]).tolist() == [3, 4, 5] and c.table(two[1]).tolist() == [6, 7]
    assert c.copies().tolist() == [[0, 3], [1, 4], [2, 5], [0, 6], [1, 7]]


def test_rewind_splits_a_shared_page(sat):
    c = _cache(sat)
    a = c.create(1)[0]
    c.extend([a], [48])
    b, d = c.fork([a, a])
    c.rewind([b, d], [20, 16])                                # inside shared page 1; on a border
    assert c.table(b).tolist() == [0, 3] and c.copies().tolist() == [[1, 3]]
    assert c.table(d).tolist() == [0]
    c.rewind([a], [20])                                       # page 1 is a's alone now: nothing to copy
    assert c.table(a).tolist() == [0, 1] and c.copies().tolist() == []
    c.rewind([a, b, d], [0, 0, 0])
    assert c.info()["used"] == 0 and c.length(a) == 0


def test_rewind_of_all_sharers_leaves_one_on_the_page(sat):
    c = _cache(sat)
    a = c.create(1)[0]
    c.extend([a], [32])
    b, d = c.fork([a, a])
    c.rewind([a, b, d], [25, 26, 27])
    tables = [c.table(x).tolist() for x in (a, b, d)]
    assert tables == [[0, 2], [0, 3], [0, 1]]
    assert c.copies().tolist() == [[1, 2], [1, 3]]


def test_compact_moves_the_highest_pages_down(sat):
    c = _cache(sat)
    a, b, d = c.create(3)
    c.extend([a, b, d], [32, 48, 30])                         # pages 0-1, 2-4, 5-6
    e = c.fork([d], [16])[0]                                  # shares page 5
    c.free([b])
    assert c.compact() == 2
    assert c.copies().tolist() == [[5, 2], [6, 3]]
    assert c.table(d).tolist() == [2, 3] and c.table(e).tolist() == [2] and c.table(a).tolist() == [0, 1]
    assert c.info()["top"] == c.info()["used"] == 4
    assert c.compact() == 0


def test_full_cache_changes_nothing(sat):
    c = _cache(sat, pages=4)
    a, b = c.create(2)
    c.extend([a], [40])
    with pytest.raises(sat.ContextFullError):
        c.extend([a, b], [8, 17])                             # the second needs two of one free page
    assert c.length(a) == 40 and c.length(b) == 0 and c.info()["free"] == 1
    with pytest.raises(sat.ContextFullError):
        c.fork([a, a])
    child = c.fork([a])[0]
    with pytest.raises(sat.ContextFullError):
        c.rewind([child], [20])                               # would have to copy shared page 1
    assert c.length(child) == 40
    with pytest.raises(sat.ContextFullError):
        c.copy([a])
    batch = sat.DecodeBatch(c, 4)
    with pytest.raises(sat.ContextFullError):
        batch.step([a, child], [20, 1])
    assert c.length(a) == 40 and c.length(child) == 40


def test_refusals(sat):
    for bad in (dict(page_tokens=24), dict(page_tokens=8), dict(page_tokens=512), dict(pages=0)):
        with pytest.raises(sat.ArgumentError):
            _cache(sat, **bad)
    for dim in (0, -8):
        with pytest.raises(sat.ArgumentError):
            sat.PagedCache(1, 4, 16, 1, dim, ctx=False)
    for dim in (12, 264):
        with pytest.raises(sat.NotSupportedError):
            sat.PagedCache(1, 4, 16, 1, dim, ctx=False)
    with pytest.raises(sat.NotSupportedError):
        sat.PagedCache(1 << 12, 1 << 20, 16, 1, 64, ctx=False)
    with pytest.raises(sat.ArgumentError):
        sat.PagedCache(1, 4, 16, 1, 64, dtype="f64", ctx=False)
    c = _cache(sat)
    a, b = c.create(2)
    c.extend([a], [20])
    for call in (lambda: c.extend([a, a], [1, 1]), lambda: c.extend([a], [-1]), lambda: c.extend([a], [0x7FFFFFFF]),
                 lambda: c.extend([a], [1, 2]), lambda: c.extend([77], [1]), lambda: c.extend([-1], [1]),
                 lambda: c.extend([a], [1.5]), lambda: c.fork([a], [21]), lambda: c.fork([a], [-1]),
                 lambda: c.rewind([a], [21]), lambda: c.rewind([a, a], [1, 1]), lambda: c.free([a, a]),
                 lambda: c.free([a + 5]), lambda: c.table(99), lambda: c.create(-1)):
        with pytest.raises(sat.ArgumentError):
            call()
    assert c.length(a) == 20 and c.info()["used"] == 2
    c.free([a])
    with pytest.raises(sat.ArgumentError):
        c.length(a)
    again = c.create(1)[0]                                    # the slot is used again under another id
    assert again != a
    with pytest.raises(sat.ArgumentError):
        c.free([a])


def test_batch_refusals_and_disposal(sat):
    c = _cache(sat)
    for heads in (0, 3, -2):
        with pytest.raises(sat.ArgumentError):
            sat.DecodeBatch(c, heads)
    for rope in (dict(rope_base=-1.0), dict(rope_base=float("inf")), dict(rope_base=float("nan")),
                 dict(rope_base=1e4, rotary=12), dict(rope_base=1e4, rotary=72), dict(rope_base=1e4, rotary=-8)):
        with pytest.raises(sat.ArgumentError):
            sat.DecodeBatch(c, 4, **rope)
    batch = sat.DecodeBatch(c, 4)
    a, b = c.create(2)
    for seqs, counts in (([a, a], [1, 1]), ([a], [-1]), ([a], []), ([9], [1])):
        with pytest.raises(sat.ArgumentError):
            batch.step(seqs, counts)
    batch.step([a, b], [5, 0])
    assert batch.info()["rows"] == 5
    c.dispose()
    c.dispose()
    with pytest.raises(sat.DisposedError):
        batch.info()
    with pytest.raises(sat.DisposedError):
        c.create(1)
    batch.dispose()
    with pytest.raises(sat.DisposedError):
        batch.step([a], [1])


def test_plan_groups_what_sequences_share(sat):
    """A common prompt is one segment for all, a second fork level another, each tail its own; short common
    runs are left with their sequences."""
    c = _cache(sat, pages=400)
    root = c.create(1)
    c.extend(root, [1600])
    batch = sat.DecodeBatch(c, 4)
    four = c.fork(root * 4)
    batch.step(four, [1] * 4)
    assert batch.info()["segments"] == 1 + 4
    c.extend([four[0]], [799])
    pair = c.fork([four[0]] * 2)
    batch.step(four[1:] + pair, [1] * 5)
    assert batch.info()["segments"] == 2 + 5
    lone = c.create(1)
    batch.step(lone + four[1:3], [7, 1, 1])
    assert batch.info()["segments"] == 1 + 1 + 2 and batch.info()["rows"] == 9
    short = c.create(1)
    c.extend(short, [16])
    batch.step(c.fork(short * 3), [1] * 3)
    assert batch.info()["segments"] == 3


def test_tables_against_a_model(sat):
    """Random forks, extensions, rewinds, frees and compactions on page contents kept in numpy: every
    sequence reads back its own tokens, and no page is lost."""
    rng = np.random.default_rng(5)
    c = _cache(sat, pages=300)
    store = np.full((300, 16), -1)
    model: dict = {}
    fresh = 0

    def apply_copies():
        pairs = c.copies()
        assert len(set(pairs[:, 1].tolist()) | set(pairs[:, 0].tolist())) == \
            len(set(pairs[:, 0].tolist())) + len(pairs)       # destinations are distinct and no sources
        store[pairs[:, 1]] = store[pairs[:, 0]]

    for _ in range(400):
        op = rng.integers(6)
        ids = list(model)
        if op == 0 or not ids:
            model[c.create(1)[0]] = []
        elif op == 1:
            some = list(rng.choice(ids, min(len(ids), 3), replace=False))
            counts = rng.integers(0, 60, len(some))
            try:
                c.extend(some, counts)
            except sat.ContextFullError:
                continue
            for s, n in zip(some, counts):
                for t in range(len(model[s]), len(model[s]) + n):
                    store[c.table(s)[t // 16], t % 16] = fresh
                    model[s].append(fresh)
                    fresh += 1
        elif op == 2:
            parents = [int(v) for v in rng.choice(ids, 2)]
            at = [int(rng.integers(len(model[p]) + 1)) for p in parents]
            try:
                children = (c.fork if rng.integers(2) else c.copy)(parents, at)
            except sat.ContextFullError:
                continue
            apply_copies()
            for child, p, n in zip(children, parents, at):
                model[child] = model[p][:n]
        elif op == 3:
            some = list(rng.choice(ids, min(len(ids), 3), replace=False))
            at = [int(rng.integers(len(model[s]) + 1)) for s in some]
            try:
                c.rewind(some, at)
            except sat.ContextFullError:
                continue
            apply_copies()
            for s, n in zip(some, at):
                model[s] = model[s][:n]
        elif op == 4 and len(ids) > 6:
            gone = list(rng.choice(ids, 2, replace=False))
            c.free(gone)
            for s in gone:
                del model[s]
        elif op == 5:
            c.compact()
            apply_copies()
            assert c.info()["top"] == c.info()["used"]
        held = set()
        for s, tokens in model.items():
            table = c.table(s)
            held |= set(table.tolist())
            assert c.length(s) == len(tokens)
            got = store[table].reshape(-1)[:len(tokens)]
            assert got.tolist() == tokens
        assert c.info()["used"] == len(held)
