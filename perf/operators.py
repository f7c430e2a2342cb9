"""What the attention over a paged cache and the operators around it are measured on: the work that a program which serves a
model hands to ``tannic_amd.ops``.

A case is a dict of plain values.  ``listed()`` names twelve, ``draw(rng)`` gives one more of the same ranges; ``prepare`` makes
what a program has in hand before the call, ``run`` is one pass, ``work`` what it cannot do without and ``exact`` what it returns
by the operators' definitions in 64 bits.  With ``own`` the framework's operators run, else the same in elementary operations.

The kinds, and what they stand for:

    attend   queries of new tokens over the pages that hold their sequences' keys and values, those of the new tokens among
             them: one token of every sequence (decoding), or a chunk of a prompt behind what is there already
    append   keys and values of new tokens, rotated by their positions, written into their sequences' pages; the queries rotated
    copy     pages copied inside a cache of several layers: the pages that forked sequences go on writing, or a compaction
    cross    queries of a decoder's tokens over an encoder's states, of another length for every sequence of the batch
"""
import math

import torch

own = False

_DEVICE = torch.device("cuda", 0)
_TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}

# heads, kv heads, head size: the decoder layers of this repository's measurements
_LARGE, _MIDDLE, _SMALL = (32, 8, 128), (16, 4, 128), (16, 4, 64)


def _case(name, kind, dtype, heads, **more):
    return {"name": name, "kind": kind, "dtype": dtype, "heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2], **more}


def listed():
    return [
        # the next token of one sequence: the smallest call, latency
        _case("attend-1-token", "attend", "bfloat16", _LARGE, sequences=1, new_from=1, new=1, context_from=2048, context=2048, page=16),
        # the next token of a batch whose sequences have come differently far
        _case("attend-32-tokens", "attend", "float16", _LARGE, sequences=32, new_from=1, new=1, context_from=64, context=4096, page=16),
        # the next token of a few sequences with very long contexts: the cache's bytes are what counts
        _case("attend-4-long", "attend", "bfloat16", _LARGE, sequences=4, new_from=1, new=1, context_from=32768, context=131072, page=64),
        # short prompts in the front end's default type, pages that no power of two divides, lengths as they fall
        _case("attend-prompts-fp32", "attend", "float32", _SMALL, sequences=3, new_from=17, new=100, context_from=1, context=1000, page=20),
        # a chunk of a prompt behind a first part
        _case("attend-chunk", "attend", "bfloat16", _LARGE, sequences=1, new_from=512, new=512, context_from=4096, context=4096, page=16),
        # a large chunk of a very long prompt: the matrix pipe is what counts
        _case("attend-chunk-long", "attend", "bfloat16", _LARGE, sequences=1, new_from=2048, new=2048, context_from=30720, context=30720, page=64),
        # the same batch's new keys and values
        _case("append-32-tokens", "append", "bfloat16", _LARGE, sequences=32, new_from=1, new=1, context_from=64, context=4096, page=16),
        # prompts of several lengths at once
        _case("append-prompts", "append", "float16", _LARGE, sequences=4, new_from=500, new=4001, context_from=0, context=0, page=16),
        # four sequences forked in the middle of a page, every layer's keys and values
        _case("copy-fork", "copy", "bfloat16", _LARGE, layers=32, pages=256, moved=4, page=16),
        # half of a cache moved together
        _case("copy-compact", "copy", "bfloat16", _LARGE, layers=8, pages=2048, moved=1000, page=16),
        # one decoder token of every sequence over its encoder states
        _case("cross-1-token", "cross", "float16", (16, 16, 64), batch=8, tokens=1, states=1024),
        # whole decoder inputs over theirs (training-shaped batches, scoring)
        _case("cross-prompts", "cross", "bfloat16", (16, 16, 64), batch=8, tokens=700, states=2000),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        kind = rng.choice(["attend", "attend", "attend", "append", "copy", "cross"])
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
        heads = rng.choice([_LARGE, _LARGE, _MIDDLE, _SMALL, (8, 8, 80), (12, 2, 256), (5, 1, 40)])
        page = rng.choice([16, 16, 16, 32, 64, 20, 7])
        c = {"kind": kind, "dtype": dtype, "heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2]}
        if kind in ("attend", "append"):
            most = _log(rng, 16, 65536)
            least = rng.choice([most, max(1, most // 8), _log(rng, 1, most)])
            new = rng.choice([1, 1, _log(rng, 2, 2048)])
            c.update(sequences=_log(rng, 1, 64), new_from=rng.choice([1, new]), new=new, context_from=least, context=most, page=page)
        elif kind == "copy":
            pages = _log(rng, 16, 2048)
            c.update(layers=rng.choice([1, 1, 4, 8, 32]), pages=pages, moved=_log(rng, 1, pages // 2), page=page)
        else:
            c.update(batch=_log(rng, 1, 32), tokens=rng.choice([1, _log(rng, 2, 1024)]), states=_log(rng, 16, 4096))
        w = work(c)
        # (the plain form keeps its scores in memory)
        if w["bytes"] <= 1.2e9 and w["flops"] <= (2e10 if dtype == "float32" else 5e11) and _held(c) <= 6e9:
            return c


def _held(case):
    """Bytes of the plain form's padded scores and values, or of the cache."""
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "cross":
        return 4 * case["batch"] * (heads * case["tokens"] * case["states"] + 2 * kv * case["states"] * d)
    if case["kind"] == "copy":
        return 8 * case["layers"] * case["pages"] * case["page"] * kv * d
    longest = case["context"] + case["new"]
    return 4 * case["sequences"] * (heads * case["new"] * longest + 2 * kv * longest * d)


def _spread(low, high, n):
    """n whole numbers from low to high, evenly apart in their logarithm."""
    if n == 1 or low == high:
        return [high] * n
    a, b = math.log(low + 1), math.log(high + 1)
    return [int(round(math.exp(a + (b - a) * i / (n - 1)))) - 1 for i in range(n)]


def _lengths(case):
    """New tokens and earlier tokens of every sequence; the longest chunk comes with the shortest context."""
    n = case["sequences"]
    return _spread(case["new_from"], case["new"], n), _spread(case["context_from"], case["context"], n)[::-1]


def _states(case):
    return _spread(max(1, case["states"] // 4), case["states"], case["batch"])


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "copy":
        moved = 2 * case["layers"] * case["moved"] * kv * case["page"] * d
        return {"bytes": 2 * size * moved, "flops": 0}
    if case["kind"] == "cross":
        seen = sum(_states(case))
        return {"bytes": size * d * (2 * heads * case["batch"] * case["tokens"] + 2 * kv * seen) + 4 * case["batch"],
                "flops": 4 * heads * d * case["tokens"] * seen}
    new, context = _lengths(case)
    tokens, total = sum(new), sum(new) + sum(context)
    tables = 4 * (2 * len(new) + 1 + sum(-(-(n + c) // case["page"]) for n, c in zip(new, context)))
    if case["kind"] == "append":
        return {"bytes": tokens * d * (size * 2 * (heads + 2 * kv) + 4) + tables, "flops": 3 * tokens * d * (heads + kv)}
    return {"bytes": size * d * (2 * heads * tokens + 2 * kv * total) + tables,
            "flops": 4 * heads * d * sum(n * c + n * (n + 1) // 2 for n, c in zip(new, context))}


# ---- what a program has in hand -----------------------------------------------------------------------------------------
class _Borrowed:
    """Memory of a torch tensor as a buffer of the framework's tensors; keeps it."""

    def __init__(self, tensor, environment):
        self.owner, self.environment, self.array = tensor, environment, None
        self.address, self.nbytes = tensor.data_ptr(), tensor.untyped_storage().nbytes() - tensor.storage_offset() * tensor.element_size()


def _in_hand(tensor, device):
    """The framework's tensor over a torch tensor's memory."""
    import tannic_amd as ta
    t = ta.Tensor(ta.types.BY_NAME[str(tensor.dtype).replace("torch.", "")], tensor.shape, tensor.stride())
    t.buffer = _Borrowed(tensor, device)
    return t


class _Memory:
    """A result's memory as the array interface describes it; keeps the result."""

    def __init__(self, result):
        self.result = result
        # (16-bit results are looked at as 16-bit integers first: the array interface has no bfloat16)
        self.__cuda_array_interface__ = {"shape": result.shape, "typestr": "<f4" if result.dtype.itemsize == 4 else "<i2", "data": (result.address, False), "strides": None, "version": 2}


def _seen(result, dtype):
    view = torch.as_tensor(_Memory(result), device=_DEVICE)
    return view if dtype is torch.float32 else view.view(dtype)


def _angles(positions, d):
    """cos and sin of position * theta^(-2i/d) in fp32, from the angles in 64 bits."""
    inv = 500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=_DEVICE) / d)
    a = torch.arange(positions, dtype=torch.float64, device=_DEVICE)[:, None] * inv
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    dtype, heads, kv, d = _TORCH[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
    g = torch.Generator(device=_DEVICE)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.empty(shape, dtype=dtype, device=_DEVICE).normal_(0.0, 1.0, generator=g)

    s = {"kind": case["kind"], "scale": 1.0 / math.sqrt(d), "dtype": dtype}
    if case["kind"] == "copy":
        s["pool"] = normal(case["layers"], 2, case["pages"], kv, case["page"], d)
        order = torch.randperm(case["pages"], generator=g, device=_DEVICE)
        s["sources"], s["targets"] = order[:case["moved"]].contiguous(), order[case["moved"]:2 * case["moved"]].contiguous()
        # (which pages move is decided on the host)
        s["lists"] = s["sources"].tolist(), s["targets"].tolist()
        names = ["pool"]
    elif case["kind"] == "cross":
        s["q"] = normal(case["batch"], case["tokens"], heads, d)
        s["k"], s["v"] = normal(case["batch"], case["states"], kv, d), normal(case["batch"], case["states"], kv, d)
        at = torch.randperm(case["batch"], generator=g, device=_DEVICE)
        s["lengths"] = torch.tensor(_states(case), dtype=torch.int32, device=_DEVICE)[at]
        names = ["q", "k", "v", "lengths"]
    else:
        new, context = _lengths(case)
        n, page = len(new), case["page"]
        pages = [-(-(a + b) // page) for a, b in zip(new, context)]
        # every sequence's pages lie anywhere in the cache; what is behind a sequence's last page names none
        room = sum(pages) + 8
        order = torch.randperm(room, generator=g, device=_DEVICE).to(torch.int32)
        at = torch.arange(max(pages), device=_DEVICE)[None, :]
        have = torch.tensor(pages, device=_DEVICE)
        first = torch.cumsum(have, 0) - have
        s["table"] = torch.where(at < have[:, None], order[(first[:, None] + at).clamp(max=room - 1)], -1).to(torch.int32).contiguous()
        s["context"] = torch.tensor(context, dtype=torch.int32, device=_DEVICE)
        s["starts"] = torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device=_DEVICE)
        s["longest"], s["chunk"] = max(a + b for a, b in zip(new, context)), max(new)
        s["keys"], s["values"] = normal(room, kv, page, d), normal(room, kv, page, d)
        names = ["q", "keys", "values", "table", "starts", "context"]
        if case["kind"] == "append":
            # columns of one projection's result, as the product leaves them
            s["qkv"] = normal(sum(new), heads + 2 * kv, d)
            s["q"], s["k"], s["v"] = s["qkv"][:, :heads], s["qkv"][:, heads:heads + kv], s["qkv"][:, heads + kv:]
            s["cos"], s["sin"] = _angles(s["longest"], d)
            names += ["k", "v", "cos", "sin"]
        else:
            s["q"] = normal(sum(new), heads, d)
    if own:
        import tannic_amd as ta
        device = ta.Device(0)
        s["hand"] = {name: _in_hand(s[name], device) for name in names}
    return s


# ---- the passes ---------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _OWN[state["kind"]](state, state["hand"])
    return _PLAIN[state["kind"]](state)


def _own_attend(s, t):
    from tannic_amd import ops
    return _seen(ops.attend_pages(t["q"], t["keys"], t["values"], t["table"], t["starts"], t["context"], s["scale"]), s["dtype"])


def _own_append(s, t):
    from tannic_amd import ops
    q = ops.append_pages(t["k"], t["v"], t["keys"], t["values"], t["table"], t["starts"], t["context"], t["cos"], t["sin"], t["q"])
    return _seen(q, s["dtype"]), s["keys"], s["values"]


def _own_copy(s, t):
    from tannic_amd import ops
    ops.copy_pages(t["pool"], *s["lists"])
    return s["pool"]


def _own_cross(s, t):
    from tannic_amd import ops
    return _seen(ops.attend(t["q"], t["k"], t["v"], t["lengths"], s["scale"]), s["dtype"])


_OWN = {"attend": _own_attend, "append": _own_append, "copy": _own_copy, "cross": _own_cross}


def _weights(scores, seen):
    """Softmax over the last axis of the scores that are seen."""
    scores = scores.masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _attention(q, k, v, seen, scale):
    """q [b, n, heads, d], k and v [b, kv heads, length, d], seen [b, n, length]: in fp32."""
    b, n, heads, d = q.shape
    kv, group = k.shape[1], heads // k.shape[1]
    rows = q.float().view(b, n, kv, group, d).transpose(1, 2).reshape(b, kv, n * group, d)
    scores = (rows @ k.float().transpose(-1, -2)) * scale
    p = _weights(scores, seen[:, None].repeat_interleave(group, 2))
    return (p @ v.float()).view(b, kv, n, group, d).transpose(1, 2).reshape(b, n, heads, d)


def _places(s):
    """Sequence of every new token and its number among that sequence's."""
    starts = s["starts"].long()
    token = torch.arange(s["q"].shape[0], device=_DEVICE)
    sequence = torch.searchsorted(starts, token, right=True) - 1
    return sequence, token - starts[sequence]


def _plain_attend(s):
    sequence, number = _places(s)
    n, longest, chunk = s["context"].shape[0], s["longest"], s["chunk"]
    q = torch.zeros((n, chunk) + s["q"].shape[1:], dtype=torch.float32, device=_DEVICE)
    q[sequence, number] = s["q"].float()
    table = s["table"].long().clamp(min=0)
    k, v = (pool[table].transpose(1, 2).flatten(2, 3)[:, :, :longest] for pool in (s["keys"], s["values"]))
    at = torch.arange(longest, device=_DEVICE)
    seen = at <= s["context"].long()[:, None, None] + torch.arange(chunk, device=_DEVICE)[:, None]
    return _attention(q, k, v, seen, s["scale"])[sequence, number].to(s["dtype"])


def _turned(x, cos, sin):
    """The pairs (2i, 2i+1) of x [tokens, heads, d] by their token's angles [tokens, d/2]."""
    x = x.float()
    even, odd, cos, sin = x[..., 0::2], x[..., 1::2], cos[:, None].float(), sin[:, None].float()
    return torch.stack((even * cos - odd * sin, even * sin + odd * cos), -1).flatten(-2)


def _plain_append(s):
    sequence, number = _places(s)
    position = s["context"].long()[sequence] + number
    page = s["keys"].shape[2]
    where, row = s["table"].long()[sequence, position // page], position % page
    cos, sin = s["cos"][position], s["sin"][position]
    s["keys"][where, :, row] = _turned(s["k"], cos, sin).to(s["dtype"])
    s["values"][where, :, row] = s["v"]
    return _turned(s["q"], cos, sin).to(s["dtype"]), s["keys"], s["values"]


def _plain_copy(s):
    s["pool"][:, :, s["targets"]] = s["pool"][:, :, s["sources"]]
    return s["pool"]


def _plain_cross(s):
    at = torch.arange(s["k"].shape[1], device=_DEVICE)
    seen = (at < s["lengths"].long()[:, None])[:, None].expand(-1, s["q"].shape[1], -1)
    return _attention(s["q"], s["k"].transpose(1, 2), s["v"].transpose(1, 2), seen, s["scale"]).to(s["dtype"])


_PLAIN = {"attend": _plain_attend, "append": _plain_append, "copy": _plain_copy, "cross": _plain_cross}


# ---- by definition, in 64 bits ------------------------------------------------------------------------------------------
def _one_head(q, k, v, scale, last):
    """q [n, d] over k, v [length, d] of one head; row i sees the keys up to last[i]."""
    s = (q.double() @ k.double().t().contiguous()) * scale
    s = torch.where(torch.arange(k.shape[0], device=_DEVICE)[None] <= last[:, None], s, torch.full_like(s, -math.inf))
    p = torch.softmax(s, -1)
    return p @ v.double()


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "copy":
        pool = s["pool"].double()
        for a, b in zip(*s["lists"]):
            pool[:, :, b] = pool[:, :, a]
        return pool
    if case["kind"] == "cross":
        if case["batch"] * heads > 4096:
            return None
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEVICE)
        for b, length in enumerate(s["lengths"].tolist()):
            for h in range(heads):
                last = torch.full((case["tokens"],), length - 1, device=_DEVICE)
                out[b, :, h] = _one_head(s["q"][b, :, h], s["k"][b, :length, h * kv // heads], s["v"][b, :length, h * kv // heads], s["scale"], last)
        return out
    starts, context, page = s["starts"].tolist(), s["context"].tolist(), case["page"]
    if case["kind"] == "append":
        positions = torch.cat([torch.arange(starts[i + 1] - starts[i], device=_DEVICE) + c for i, c in enumerate(context)])
        rows = torch.cat([s["table"][i, (torch.arange(starts[i + 1] - starts[i], device=_DEVICE) + c) // page] for i, c in enumerate(context)]).long()
        # (the angles are inputs: the tables in fp32)
        turn = torch.complex(s["cos"][positions].double(), s["sin"][positions].double())[:, None]
        q, k = (torch.view_as_real(torch.view_as_complex(x.double().unflatten(-1, (d // 2, 2)).contiguous()) * turn).flatten(-2) for x in (s["q"], s["k"]))
        keys, values = s["keys"].double(), s["values"].double()
        for h in range(kv):
            keys[rows, h, positions % page], values[rows, h, positions % page] = k[:, h], s["v"][:, h].double()
        return q, keys, values
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEVICE)
    for i, c in enumerate(context):
        n = starts[i + 1] - starts[i]
        pages = s["table"][i, :-(-(c + n) // page)].long()
        last = c + torch.arange(n, device=_DEVICE)
        for h in range(heads):
            k, v = (pool[pages, h * kv // heads].reshape(-1, d)[:c + n] for pool in (s["keys"], s["values"]))
            out[starts[i]:starts[i + 1], h] = _one_head(s["q"][starts[i]:starts[i + 1], h], k, v, s["scale"], last)
    return out
