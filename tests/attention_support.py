"""Attention by its definition in 64 bits, what an implementation may be off by, and paged caches to run it on."""
import numpy as np

import tannic_amd as ta

# half a step of a type, relative to the value
HALF = {ta.float16: 2.0 ** -11, ta.bfloat16: 2.0 ** -8, ta.float32: 2.0 ** -24, ta.float64: 2.0 ** -53}


def head_attention(q, k, v, scale, seen, live=None):
    """q [n, d] over k, v [length, d]; row i sees the first seen[i] keys, of those the live ones.  (result, bound of what it may be off
    by without the roundings of its type, sum of p |v|), all float64."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, length, d = q.shape[0], k.shape[0], q.shape[1]
    out, slack, size = np.zeros((n, d)), np.zeros((n, d)), np.zeros((n, d))
    for i in range(n):
        keys = np.arange(min(length, int(seen[i])))
        if live is not None:
            keys = keys[live[keys]]
        if keys.size == 0:
            continue
        s = k[keys] @ q[i] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i] = p @ v[keys]
        size[i] = p @ np.abs(v[keys])
        # scores are sums of d products in fp32, scaled and shifted: off by (d + 4) units of the largest sum of |q k|; the weights are
        # off by twice that, by what the exponential does to its argument (|s - max| units) and by the length of their sum
        off = 2 * (d + 4) * (np.abs(k[keys]) @ np.abs(q[i])).max() * abs(scale) + 2 * (s.max() - s).clip(max=90).max() + keys.size + 64
        slack[i] = off * size[i]
    return out, slack, size


def bound(out, slack, size, dtype, value_sum=0.0):
    """What a result of `dtype` may be off by: its own rounding, fp32's (float64: double's) in between, and for the 16-bit types the
    rounding of the weights for the matrix pipe (fp16: values below 2^-14 of the largest, shifted by 2^8, lose bits)."""
    unit = 2.0 ** -53 if dtype is ta.float64 else 2.0 ** -24
    b = HALF[dtype] * np.abs(out) + unit * slack
    if dtype in (ta.float16, ta.bfloat16):
        b = b + HALF[dtype] * (1 + HALF[dtype]) * size
    if dtype is ta.float16:
        b = b + 2.0 ** -25 + 2.0 ** -25 * 2.0 ** -8 * value_sum
    return b


def rounded(x, dtype):
    """`x` as values of `dtype` (float64 array)."""
    return ta.types.to_numeric(ta.types.to_storage(x, dtype), dtype).astype(np.float64)


class Cache:
    """Sequences with `new[s]` tokens behind `context[s]` earlier ones, their pages anywhere in a pool; whatever no token wrote is NaN, and the
    table names pages that do not exist behind a sequence's last."""

    def __init__(self, rng, dtype, device, heads, kv_heads, d, page, new, context, spare=3, columns=1, token_major=False, room=None, width=None):
        self.dtype, self.page, self.new, self.context = dtype, page, list(new), list(context)
        self.heads, self.kv_heads, self.d = heads, kv_heads, d
        have = [-(-(a + b) // page) for a, b in zip(new, context)]
        room = room or sum(have) + spare
        order = rng.permutation(room)
        width = width or max(have + [0]) + columns
        table = np.array([-1, 1 << 30, -(1 << 31), room])[rng.integers(0, 4, (len(new), width))]
        self.k = [rounded(rng.standard_normal((a + b, kv_heads, d)), dtype) for a, b in zip(new, context)]
        self.v = [rounded(rng.standard_normal((a + b, kv_heads, d)), dtype) for a, b in zip(new, context)]
        keys, values = np.full((2, room, kv_heads, page, d), np.nan)
        at = 0
        for s, n in enumerate(have):
            table[s, :n] = order[at:at + n]
            at += n
            for j in range(len(self.k[s])):
                keys[table[s, j // page], :, j % page] = self.k[s][j]
                values[table[s, j // page], :, j % page] = self.v[s][j]
        if token_major:     # (pages of [page, kv heads, d], seen the other way round)
            self.keys, self.values = (ta.tensor(x.transpose(0, 2, 1, 3), dtype, device).transpose(1, 2) for x in (keys, values))
        else:
            self.keys, self.values = ta.tensor(keys, dtype, device), ta.tensor(values, dtype, device)
        self.host_table = table
        self.table = ta.tensor(table, ta.int32, device)
        self.starts = ta.tensor(np.concatenate([[0], np.cumsum(new)]), ta.int32, device)
        self.lengths = ta.tensor(np.array(context), ta.int32, device)
        self.q = rounded(rng.standard_normal((sum(new), heads, d)), dtype)

    def expected(self, scale, missing=()):
        """Result, slack, sum of p |v| and sum of |v| for every token; `missing`: (sequence, column) of pages that are not there."""
        shape = self.q.shape
        out, slack, size, total = np.zeros(shape), np.zeros(shape), np.zeros(shape), np.zeros(shape)
        first, group = 0, self.heads // self.kv_heads
        for s, (n, c) in enumerate(zip(self.new, self.context)):
            live = np.ones(n + c, bool)
            for at, column in missing:
                if at == s:
                    live[column * self.page:(column + 1) * self.page] = False
            for h in range(self.heads):
                rows = slice(first, first + n)
                k, v = self.k[s][:, h // group], self.v[s][:, h // group]
                out[rows, h], slack[rows, h], size[rows, h] = head_attention(self.q[rows, h], k, v, scale, c + 1 + np.arange(n), live)
                total[rows, h] = np.abs(v).sum(0) if n + c else 0.0
            first += n
        return out, slack, size, total


def assert_within(got, want, slack, size, dtype, total=0.0, what=""):
    b = bound(want, slack, size, dtype, total)
    off = np.abs(np.asarray(got, np.float64) - want)
    bad = ~(off <= b)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} off by more than they may; first at {i}: {got[i]} for {want[i]}, bound {b[i]}")
