"""Keys and values of many sequences in the pages of one cache: which page holds what, on the host.

The memory is one tensor ``[layers, 2, pages, kv heads, page, head size]``; ``keys(layer)`` and ``values(layer)`` are views of it as
``ops.append_pages`` and ``ops.attend_pages`` take them.  A sequence is a list of pages and a length.  ``fork`` shares a sequence's pages
with a new one; a shared page is copied when one of its sequences is about to write into it, and goes back to the free ones with its last
sequence.  Nothing here waits for the device but ``plan``, which uploads the tables of a step::

    cache = PagedCache(layers, pages, 16, kv_heads, head_dim, types.bfloat16, device)
    a = cache.add()
    step = cache.plan([a], [prompt_length])            # pages for the new tokens, tables on the device
    for layer in range(layers):
        x = decoder_layer.forward_paged(shape, weights[layer], x, cos, sin, cache, layer, step)
    cache.advance(step)                                # the new tokens are part of the sequences now
    b = cache.fork(a)                                  # goes on from here on its own
"""
import numpy as np

from . import ops, types
from .graph import Graph
from .ops import TannicError
from .tensor import Tensor


class Step:
    """What a step's calls take: ``table``, ``starts`` and ``context`` on the device; ``ids`` and ``new`` say whose tokens its rows are, ``lengths``
    how many tokens those had when it was planned."""

    def __init__(self, ids, new, lengths, whole, table, starts, context):
        self.ids, self.new, self.lengths, self._whole = ids, new, lengths, whole
        self.table, self.starts, self.context = table, starts, context

    @property
    def tokens(self):
        return sum(self.new)


class PagedCache:
    def __init__(self, layers, pages, page, kv_heads, head_dim, dtype, environment):
        if min(layers, pages, page, kv_heads, head_dim) < 1:
            raise ValueError("PagedCache: layers, pages, page, kv heads and head size are at least 1")
        self.page, self.pages = page, pages
        self.storage = Tensor(dtype, (layers, 2, pages, kv_heads, page, head_dim)).initialize(environment)
        self._free = list(range(pages - 1, -1, -1))      # the lowest on top
        self._users = [0] * pages
        self._sequences = {}                             # id -> [pages, length]
        self._last = 0

    # ---- what the operators take -----------------------------------------------------
    def keys(self, layer):
        return self.storage[layer, 0]

    def values(self, layer):
        return self.storage[layer, 1]

    # ---- sequences ----------------------------------------------------------------------
    @property
    def free_pages(self):
        return len(self._free)

    def length(self, sequence):
        return self._of(sequence)[1]

    def pages_of(self, sequence):
        return tuple(self._of(sequence)[0])

    def _of(self, sequence):
        try:
            return self._sequences[sequence]
        except KeyError:
            raise TannicError(f"PagedCache: there is no sequence {sequence}") from None

    def add(self):
        """A new, empty sequence."""
        self._last += 1
        self._sequences[self._last] = [[], 0]
        return self._last

    def fork(self, sequence):
        """A new sequence that shares all of ``sequence``'s pages."""
        pages, length = self._of(sequence)
        for p in pages:
            self._users[p] += 1
        self._last += 1
        self._sequences[self._last] = [list(pages), length]
        return self._last

    def free(self, sequence):
        """Forgets a sequence; pages that nobody else uses are free again."""
        pages, _ = self._of(sequence)
        del self._sequences[sequence]
        for p in reversed(pages):
            self._release(p)

    def truncate(self, sequence, length):
        """Drops a sequence's tokens behind ``length`` (drafts that were not accepted)."""
        mine = self._of(sequence)
        if not 0 <= length <= mine[1]:
            raise TannicError(f"PagedCache: sequence {sequence} has {mine[1]} tokens, not {length}")
        keep = -(-length // self.page)
        for p in reversed(mine[0][keep:]):
            self._release(p)
        del mine[0][keep:]
        mine[1] = length

    def _release(self, page):
        self._users[page] -= 1
        if self._users[page] == 0:
            self._free.append(page)

    # ---- a step -----------------------------------------------------------------------------
    def plan(self, ids, new, columns=None, into=None):
        """Gives the sequences ``ids`` pages for ``new[i]`` more tokens each and puts the step's tables on the device: sequence ``i``'s
        tokens are the ``new[i]`` rows behind those of the sequences before.  Shared pages that they will write into are copied first.
        ``columns``: pages a row of the table has room for (else as many as needed); ``into``: an earlier step of as many sequences
        whose tensors are written again, for a recording that reads them.  Raises, and changes nothing, if there are not enough pages, and
        inside a recording."""
        self._outside_a_recording()
        ids, new = list(ids), [int(n) for n in new]
        if len(ids) != len(new) or len(set(ids)) != len(ids) or any(n < 0 for n in new):
            raise TannicError("PagedCache: every sequence of a step once, with the number of its new tokens")
        sequences = [self._of(i) for i in ids]
        if into is not None:
            if len(into.ids) != len(ids):
                raise TannicError(f"PagedCache: a step of {len(ids)} sequences into the tensors of one of {len(into.ids)}")
            columns = into.table.shape[1]
        needed = [-(-(length + n) // self.page) for (_, length), n in zip(sequences, new)]
        width = max(needed, default=0) if columns is None else columns
        if any(n > width for n in needed):
            raise TannicError(f"PagedCache: a sequence needs {max(needed)} pages, the table has room for {width}")
        # pages that get new tokens and belong to somebody else too (with several of a page's users in this step the last one keeps it)
        users, shared, wanted = {}, [], 0
        for (pages, length), n, have in zip(sequences, new, needed):
            wanted += max(0, have - len(pages))
            for at in range(length // self.page, min(have, len(pages)) if n > 0 else 0):
                if users.setdefault(pages[at], self._users[pages[at]]) > 1:
                    users[pages[at]] -= 1
                    shared.append((pages, at))
        if wanted + len(shared) > len(self._free):
            raise TannicError(f"PagedCache: {wanted + len(shared)} pages are needed and {len(self._free)} are free")
        if shared:
            targets = self._free[:-len(shared) - 1:-1]
            ops.copy_pages(self.storage, [pages[at] for pages, at in shared], targets)
            for (pages, at), target in zip(shared, targets):
                self._users[pages[at]] -= 1
                pages[at] = self._take()
        for (pages, _), have in zip(sequences, needed):
            while len(pages) < have:
                pages.append(self._take())
        # one upload: the table, the starts, the lengths
        n = len(ids)
        whole = np.empty(n * width + 2 * n + 1, np.int32)
        table = whole[:n * width].reshape(n, width)
        table.fill(-1)
        for row, (pages, _) in zip(table, sequences):
            row[:min(len(pages), width)] = pages[:width]
        whole[n * width:n * width + n + 1] = np.concatenate([[0], np.cumsum(new)])
        lengths = [length for _, length in sequences]
        whole[n * width + n + 1:] = lengths
        if into is not None:
            into._whole.write_raw(whole)
            into.ids, into.new, into.lengths = ids, new, lengths
            return into
        t = Tensor(types.int32, whole.shape).initialize(self.storage.environment)
        t.write_raw(whole)
        return Step(ids, new, lengths, t, t[0:n * width].view(n, width), t[n * width:n * width + n + 1], t[n * width + n + 1:])

    def _outside_a_recording(self):
        # (the copies of pages would run with every replay, and not now)
        if Graph.records(self.storage.environment):
            raise TannicError("PagedCache: pages are planned and moved outside of a recording")

    def _take(self):
        page = self._free.pop()
        self._users[page] = 1
        return page

    def advance(self, step):
        """The step's tokens have been written, in every layer: they count from now on.  Raises, and changes nothing, if one of its sequences has
        changed its length or lost a page for them since the step was planned (freed, cut, or advanced already)."""
        sequences = [self._of(i) for i in step.ids]
        for i, (pages, length), n, planned in zip(step.ids, sequences, step.new, step.lengths):
            if length != planned or len(pages) * self.page < length + n:
                raise TannicError(f"PagedCache: sequence {i} has {length} tokens and {len(pages)} pages, the step was planned for {n} more behind {planned}")
        for entry, n in zip(sequences, step.new):
            entry[1] += n

    # ---- order --------------------------------------------------------------------------------
    def compact(self):
        """Moves the used pages to the front of the cache (steps planned before name the old places); how many moved.  Raises inside a recording."""
        self._outside_a_recording()
        used = sorted({p for pages, _ in self._sequences.values() for p in pages})
        count = len(used)
        holes = sorted(p for p in self._free if p < count)
        sources = [p for p in used if p >= count]
        if sources:
            ops.copy_pages(self.storage, sources, holes)
            where = dict(zip(sources, holes))
            for entry in self._sequences.values():
                entry[0] = [where.get(p, p) for p in entry[0]]
            for a, b in where.items():
                self._users[b], self._users[a] = self._users[a], 0
        self._free = list(range(self.pages - 1, count - 1, -1))
        return len(sources)
