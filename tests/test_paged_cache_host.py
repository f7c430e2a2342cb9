"""The bookkeeping of a paged cache: pages, references, forks, copies before a write, compaction.  The tensors are on the host and the copies are
done by numpy: no GPU is needed."""
import numpy as np
import pytest

import tannic_amd as ta
from tannic_amd import ops
from tannic_amd.paged_cache import PagedCache


@pytest.fixture
def cache(monkeypatch):
    copies = []

    def copy_pages(pool, sources, targets):
        data = pool.buffer.array.view(np.int32).reshape(pool.shape)
        copies.extend(zip(list(sources), list(targets)))
        for a, b in zip(sources, targets):
            data[:, :, b] = data[:, :, a]
        return pool

    monkeypatch.setattr(ops, "copy_pages", copy_pages)
    monkeypatch.setattr(ta.Tensor, "write_raw", lambda self, raw: self.buffer.array.__setitem__(slice(self.offset, self.offset + raw.nbytes), np.ascontiguousarray(raw).view(np.uint8)))
    c = PagedCache(2, 8, 4, 1, 1, ta.int32, ta.Host())
    c.copies = copies
    return c


def write(cache, step, mark):
    """What append_pages does: token t of a sequence is written where the tables say."""
    data = cache.storage.buffer.array.view(np.int32).reshape(cache.storage.shape)
    table, starts, context = step.table.numpy(), step.starts.numpy(), step.context.numpy()
    for i in range(len(step.ids)):
        for t in range(starts[i + 1] - starts[i]):
            p = context[i] + t
            data[:, :, table[i, p // cache.page], :, p % cache.page] = mark * 1000 + p


def read(cache, sequence):
    data = cache.storage.buffer.array.view(np.int32).reshape(cache.storage.shape)
    pages = cache.pages_of(sequence)
    return [int(data[1, 1, pages[p // cache.page], 0, p % cache.page, 0]) for p in range(cache.length(sequence))]


def consistent(cache):
    """Every page has as many users as sequences name it, and is free if it has none."""
    users = np.zeros(cache.pages, int)
    for pages, length in cache._sequences.values():
        assert len(pages) >= -(-length // cache.page) and len(set(pages)) == len(pages)
        for p in pages:
            users[p] += 1
    assert list(users) == cache._users
    assert sorted(cache._free) == [p for p in range(cache.pages) if users[p] == 0] and len(set(cache._free)) == len(cache._free)


def go(cache, ids, new, mark=1, **more):
    step = cache.plan(ids, new, **more)
    write(cache, step, mark)
    cache.advance(step)
    consistent(cache)
    return step


def test_tables_of_a_step(cache):
    a, b = cache.add(), cache.add()
    step = cache.plan([a, b], [6, 0], columns=3)
    assert step.table.numpy().tolist() == [[0, 1, -1], [-1, -1, -1]] and step.starts.numpy().tolist() == [0, 6, 6] and step.context.numpy().tolist() == [0, 0]
    assert cache.length(a) == 0 and cache.free_pages == 6 and step.tokens == 6      # (planned, not yet written)
    assert cache.plan([a, b], [6, 0]).table.numpy().tolist() == [[0, 1], [-1, -1]]    # (again: the same pages)
    go(cache, [a, b], [6, 1])
    step = cache.plan([b, a], [4, 3])
    assert step.context.numpy().tolist() == [1, 6] and step.starts.numpy().tolist() == [0, 4, 7] and step.table.numpy().tolist() == [[2, 3, -1], [0, 1, 4]]
    assert step.table.shape == (2, 3) and step.table.dtype is ta.int32


def test_a_fork_copies_the_page_it_writes(cache):
    a = cache.add()
    go(cache, [a], [6], 1)
    b = cache.fork(a)
    assert cache.pages_of(a) == cache.pages_of(b) and cache.free_pages == 6 and not cache.copies
    go(cache, [b], [1], 2)
    assert cache.copies == [(1, 2)] and cache.pages_of(b) == (0, 2) and cache.pages_of(a) == (0, 1)
    go(cache, [a], [2], 3)
    assert len(cache.copies) == 1 and read(cache, a) == [1000, 1001, 1002, 1003, 1004, 1005, 3006, 3007] and read(cache, b) == [1000, 1001, 1002, 1003, 1004, 1005, 2006]
    c = cache.fork(a)       # at the end of a page: nothing is shared that anybody writes
    go(cache, [a, c], [1, 1], 4)
    assert len(cache.copies) == 1 and cache.pages_of(c)[:2] == cache.pages_of(a)[:2] and cache.pages_of(c)[2] != cache.pages_of(a)[2]


def test_several_users_of_a_page_in_one_step(cache):
    a = cache.add()
    go(cache, [a], [3], 1)
    b, c = cache.fork(a), cache.fork(a)
    step = cache.plan([a, b, c], [1, 1, 1])
    assert len(cache.copies) == 2 and len({cache.pages_of(i) for i in (a, b, c)}) == 3 and step.table.numpy()[2, 0] == 0      # (the last keeps it)
    consistent(cache)
    cache.free(a), cache.free(b), cache.free(c)
    consistent(cache)
    assert cache.free_pages == 8


def test_a_fork_of_a_planned_step_shares_none_of_its_pages_for_long(cache):
    a = cache.add()
    cache.plan([a], [9])
    b = cache.fork(a)       # (shares the pages that a's step was promised)
    go(cache, [a, b], [9, 6], 1)
    assert not set(cache.pages_of(a)) & set(cache.pages_of(b)[:2]) and read(cache, b) == [1000 + i for i in range(6)]


def test_too_few_pages_change_nothing(cache):
    a, b = cache.add(), cache.add()
    go(cache, [a], [18], 1)
    before = (cache.pages_of(a), cache.free_pages)
    with pytest.raises(ta.TannicError, match="6 pages are needed and 3 are free"):
        cache.plan([a, b], [7, 13])
    c = cache.fork(a)
    go(cache, [b], [12], 2)
    with pytest.raises(ta.TannicError, match="1 pages are needed and 0 are free"):
        cache.plan([c], [1])          # (a copy of the shared page)
    assert (cache.pages_of(a), cache.free_pages) == (before[0], 0) and not cache.copies
    consistent(cache)
    cache.free(a)
    go(cache, [c], [1], 3)             # the page is c's alone now
    assert not cache.copies


def test_refusals(cache):
    a = cache.add()
    for ids, new in (([a, a], [1, 1]), ([a], [1, 2]), ([a], [-1]), ([99], [1])):
        with pytest.raises(ta.TannicError):
            cache.plan(ids, new)
    with pytest.raises(ta.TannicError):
        cache.plan([a], [9], columns=2)
    step = cache.plan([a], [1], columns=1)
    with pytest.raises(ta.TannicError):
        cache.plan([a, cache.add()], [1, 1], into=step)
    with pytest.raises(ta.TannicError):
        cache.plan([a], [9], into=step)
    for call in (cache.fork, cache.free, cache.length, cache.pages_of):
        with pytest.raises(ta.TannicError):
            call(77)
    with pytest.raises(ta.TannicError):
        cache.truncate(a, 1)
    with pytest.raises(ValueError):
        PagedCache(1, 0, 4, 1, 1, ta.int32, ta.Host())


def test_truncate_gives_pages_back(cache):
    a = cache.add()
    go(cache, [a], [10], 1)
    b = cache.fork(a)
    cache.truncate(a, 4)
    consistent(cache)
    assert cache.pages_of(a) == (0,) and cache.length(a) == 4 and read(cache, b) == [1000 + i for i in range(10)]
    go(cache, [a], [2], 2)
    assert read(cache, a) == [1000, 1001, 1002, 1003, 2004, 2005]
    cache.truncate(b, 0)
    consistent(cache)
    assert cache.pages_of(b) == () and cache.free_pages == 6


def test_into_writes_the_same_tensors(cache):
    a, b = cache.add(), cache.add()
    step = go(cache, [a, b], [1, 3], columns=3)
    address = step.table.address
    again = cache.plan([b, a], [1, 1], into=step)
    assert again is step and step.table.address == address and step.context.numpy().tolist() == [3, 1] and step.starts.numpy().tolist() == [0, 1, 2] and step.ids == [b, a]


def test_compaction(cache):
    a, b, c = cache.add(), cache.add(), cache.add()
    go(cache, [a, b, c], [5, 9, 2], 1)
    d = cache.fork(c)
    want = [read(cache, i) for i in (b, c, d)]
    cache.free(a)
    assert cache.compact() == 2
    consistent(cache)
    assert [read(cache, i) for i in (b, c, d)] == want and max(cache.pages_of(b) + cache.pages_of(c)) == 3 and cache.pages_of(c) == cache.pages_of(d)
    assert cache.compact() == 0
    go(cache, [d], [1], 2)
    assert read(cache, c) == want[1] and read(cache, d) == want[2] + [2002]


def test_random_lives(cache):
    """Some hundred steps of sequences that come, go, fork, shrink and are moved together: everybody reads what they wrote."""
    rng = np.random.default_rng(31)
    told = {}
    for turn in range(400):
        act = rng.integers(0, 10)
        ids = list(told)
        if act == 0 or not ids:
            told[cache.add()] = []
        elif act == 1:
            i = ids[rng.integers(len(ids))]
            told[cache.fork(i)] = list(told[i])
        elif act == 2 and len(ids) > 2:
            i = ids[rng.integers(len(ids))]
            cache.free(i)
            del told[i]
        elif act == 3:
            i = ids[rng.integers(len(ids))]
            n = int(rng.integers(0, len(told[i]) + 1))
            cache.truncate(i, n)
            told[i] = told[i][:n]
        elif act == 4:
            cache.compact()
        else:
            some = [i for i in ids if rng.random() < 0.5]
            new = [int(rng.integers(0, 4)) for _ in some]
            try:
                step = cache.plan(some, new)
            except ta.TannicError:
                i = ids[rng.integers(len(ids))]
                cache.free(i)
                del told[i]
                continue
            write(cache, step, turn)
            cache.advance(step)
            for i, n in zip(some, new):
                told[i] += [turn * 1000 + len(told[i]) + x for x in range(n)]
        consistent(cache)
        for i, want in told.items():
            assert read(cache, i) == want, (turn, i)
