"""Steps of a paged cache that are not what they were planned as any more.  The tensors are on the host: no GPU is needed."""
import numpy as np
import pytest

import tannic_amd as ta
from tannic_amd.paged_cache import PagedCache


@pytest.fixture
def cache():
    return PagedCache(1, 8, 4, 1, 1, ta.int32, ta.Host())


def state(cache):
    return {i: (tuple(pages), length) for i, (pages, length) in cache._sequences.items()}, list(cache._users), list(cache._free)


def test_a_step_counts_once(cache):
    a, b = cache.add(), cache.add()
    step = cache.plan([a, b], [3, 5])
    cache.advance(step)
    before = state(cache)
    with pytest.raises(ta.TannicError, match="sequence 1 has 3 tokens"):
        cache.advance(step)
    assert state(cache) == before
    cache.plan([a, b], [1, 0], into=step)
    cache.advance(step)
    assert (cache.length(a), cache.length(b)) == (4, 5)


def test_a_step_of_a_sequence_that_is_gone_changes_none_of_the_others(cache):
    a, b = cache.add(), cache.add()
    step = cache.plan([a, b], [3, 5])
    cache.free(b)
    with pytest.raises(ta.TannicError, match="no sequence"):
        cache.advance(step)
    assert cache.length(a) == 0
    cache.advance(cache.plan([a], [3]))
    assert cache.length(a) == 3


@pytest.mark.parametrize("length", [0, 2])
def test_a_step_of_a_sequence_that_was_cut(length, cache):
    """Its tokens went behind others, or the pages that they went into were given back."""
    a = cache.add()
    cache.advance(cache.plan([a], [2]))
    step = cache.plan([a], [7])
    cache.truncate(a, length)
    before = state(cache)
    with pytest.raises(ta.TannicError, match="planned"):
        cache.advance(step)
    assert state(cache) == before


def test_steps_that_still_hold(cache):
    """A fork, another plan of the same tokens and a compaction between plan and advance."""
    a, b = cache.add(), cache.add()
    cache.advance(cache.plan([a, b], [5, 2]))
    cache.free(a)
    step = cache.plan([b], [3])
    c = cache.fork(b)
    cache.advance(step)
    assert cache.length(b) == 5 and cache.length(c) == 2
    cache.free(c)
    step = cache.plan([b], [1])
    again = cache.plan([b], [1])
    cache.advance(again)
    with pytest.raises(ta.TannicError):
        cache.advance(step)
    assert np.array_equal(step.context.numpy(), [5])
