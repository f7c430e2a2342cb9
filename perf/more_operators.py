"""What the operators around products of 8-bit integers are measured on: the work that a program which serves a model with quantised
weights hands to ``tannic_amd.ops``.

A case is a dict of plain values.  ``listed()`` names twelve, ``draw(rng)`` gives one more of the same ranges; ``prepare`` makes
what a program has in hand before the call, ``run`` is one pass, ``work`` what it cannot do without and ``exact`` what it returns
by the operators' definitions in 64 bits.  With ``own`` the framework's operators run, else the same in elementary operations.

The kinds, and what they stand for:

    norm      a layer's activations and what the part before adds to them: their sum, and its root-mean-square norm in the
              model's type or in 8 bits with a scale for each token
    quantize  rows in 8 bits with a scale each: the attention's results, or a matrix of weights when a model is loaded
    swiglu    the gated activation of two halves of one projection, in 8 bits with a scale for each token
    product   tokens in 8 bits times weights in 8 bits, with a scale for each token and each channel, in the model's type

What is in 8 bits leaves a pass as the values that it stands for (integer times scale, in the model's type).
"""
import math

import torch

own = False

_DEVICE = torch.device("cuda", 0)
_TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
# a row whose largest value is smaller is quantised as if it were this: 127 divided by it is finite, it divided by 127 no subnormal
_LEAST = 2.0 ** -119


def _rows(name, kind, dtype, rows, width, **more):
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "width": width, **more}


def _product(name, dtype, rows, columns, inner):
    return {"name": name, "kind": "product", "dtype": dtype, "rows": rows, "columns": columns, "inner": inner}


def listed():
    return [
        # the next token of one sequence: the smallest call, latency
        _rows("norm-1-token", "norm", "bfloat16", 1, 4096, bits=8, residual=True),
        # the last norm of a model, before the products with its vocabulary: a batch's tokens, in the model's type
        _rows("norm-512-typed", "norm", "bfloat16", 512, 4096, bits=16, residual=True),
        # prompts, an odd number of tokens
        _rows("norm-prompts", "norm", "float16", 8001, 5120, bits=8, residual=True),
        # the attention's results of a batch of single tokens
        _rows("quantize-32-tokens", "quantize", "bfloat16", 32, 4096),
        # the largest matrix of a layer, when a model is loaded: its two projections into the feed-forward part
        _rows("quantize-weights", "quantize", "float16", 28672, 4096),
        # the next token of one sequence
        _rows("swiglu-1-token", "swiglu", "bfloat16", 1, 14336),
        # prompts
        _rows("swiglu-prompts", "swiglu", "bfloat16", 4096, 14336),
        # the next token of one sequence: the weights' bytes are what counts
        _product("product-1-token", "bfloat16", 1, 28672, 4096),
        # the next tokens of a batch
        _product("product-32-tokens", "bfloat16", 32, 4096, 14336),
        # the front end's default type, rows that start anywhere, sizes that no tile divides
        _product("product-odd-fp32", "float32", 77, 2049, 1030),
        # a chunk of a prompt
        _product("product-512-tokens", "bfloat16", 512, 6144, 4096),
        # prompts together: the matrix pipe is what counts
        _product("product-8192-tokens", "bfloat16", 8192, 28672, 4096),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        kind = rng.choice(["norm", "norm", "quantize", "swiglu", "product", "product", "product"])
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
        if kind == "product":
            # (rows of 16-byte pieces, of whole lines, or of any length)
            step = rng.choice([1, 16, 16, 128, 128])
            c = {"kind": kind, "dtype": dtype, "rows": rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192)]), "columns": _log(rng, 16, 28672),
                 "inner": max(1, _log(rng, 32, 14336) // step) * step}
            if 2.0 * c["rows"] * c["columns"] * c["inner"] <= 1.5e12:
                return c
            continue
        step = rng.choice([1, 8, 8, 256])
        c = {"kind": kind, "dtype": dtype, "rows": _log(rng, 1, 8192), "width": max(1, _log(rng, 16, 16384) // step) * step}
        if kind == "norm":
            c.update(bits=rng.choice([8, 8, 16]), residual=rng.choice([True, True, True, False]))
        if kind == "swiglu" and dtype == "float32":
            c["dtype"] = "float16"
        if c["rows"] * c["width"] <= 40_000_000:
            return c


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    rows = case["rows"]
    if case["kind"] == "product":
        columns, inner = case["columns"], case["inner"]
        return {"bytes": (rows + columns) * (inner + 4) + size * rows * columns, "flops": 2 * rows * columns * inner}
    width = case["width"]
    elements = rows * width
    if case["kind"] == "quantize":
        return {"bytes": elements * (size + 1) + 4 * rows, "flops": 3 * elements}
    if case["kind"] == "swiglu":
        return {"bytes": elements * (2 * size + 1) + 4 * rows, "flops": 8 * elements}
    moved = size * (width + elements * (3 if case["residual"] else 1))
    return {"bytes": moved + (elements + 4 * rows if case["bits"] == 8 else size * elements), "flops": 7 * elements}


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


def _integers(x):
    """A matrix in 8 bits and a scale for each row."""
    most = x.abs().amax(-1, keepdim=True)
    return torch.round(x * (127.0 / most)).to(torch.int8), (most / 127.0)[:, 0].contiguous()


def prepare(case, seed):
    dtype, rows = _TORCH[case["dtype"]], case["rows"]
    g = torch.Generator(device=_DEVICE)
    g.manual_seed(seed)

    def normal(*shape, deviation=1.0):
        return torch.empty(shape, dtype=torch.float32, device=_DEVICE).normal_(0.0, deviation, generator=g)

    def activations(width):
        # a few channels are much larger than the others, as in trained models
        x = normal(rows, width)
        channels = torch.randperm(width, generator=g, device=_DEVICE)[:max(1, width // 500)]
        x[:, channels] *= 12.0
        return x

    s = {"kind": case["kind"], "dtype": dtype}
    if case["kind"] == "product":
        s["a"], s["a_scales"] = _integers(activations(case["inner"]))
        # weights lie as [channels, inner], a scale for each channel
        s["w"], s["w_scales"] = _integers(normal(case["columns"], case["inner"], deviation=0.02))
        names = ["a", "a_scales", "w", "w_scales"]
    elif case["kind"] == "swiglu":
        # columns of one projection's result, as the product leaves them
        s["both"] = normal(rows, 2 * case["width"], deviation=1.5).to(dtype)
        s["gate"], s["up"] = s["both"][:, :case["width"]], s["both"][:, case["width"]:]
        names = ["gate", "up"]
    else:
        s["x"] = activations(case["width"]).to(dtype) if rows <= 8192 else normal(rows, case["width"], deviation=0.02).to(dtype)
        names = ["x"]
        if case["kind"] == "norm":
            s["bits"], s["eps"] = case["bits"], 1e-5
            s["gain"] = (1.0 + 0.1 * normal(case["width"])).to(dtype)
            s["residual"] = normal(rows, case["width"], deviation=2.0).to(dtype) if case["residual"] else None
            names += ["gain"] + (["residual"] if case["residual"] else [])
    if own:
        import tannic_amd as ta
        device = ta.Device(0)
        s["hand"] = {"residual": None, **{name: _in_hand(s[name], device) for name in names}}
        if case["kind"] == "product":
            s["hand"]["w"] = s["hand"]["w"].transpose()
            s["type"] = ta.types.BY_NAME[case["dtype"]]
    return s


# ---- the passes ---------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _OWN[state["kind"]](state, state["hand"])
    return _PLAIN[state["kind"]](state)


def _own_values(s, t, values, scales):
    from tannic_amd import ops
    return _seen(ops.dequantize(values, scales, t.dtype), s["dtype"]), _seen(scales, torch.float32)


def _own_norm(s, t):
    from tannic_amd import ops
    if s["bits"] == 8:
        values, scales, total = ops.add_rms_norm_quantized(t["x"], t["residual"], t["gain"], s["eps"])
        outputs = _own_values(s, t["x"], values, scales)
    else:
        normed, total = ops.add_rms_norm(t["x"], t["residual"], t["gain"], s["eps"])
        outputs = (_seen(normed, s["dtype"]),)
    # (without a residual the sum is the input itself)
    return outputs if s["residual"] is None else outputs + (_seen(total, s["dtype"]),)


def _own_quantize(s, t):
    from tannic_amd import ops
    return _own_values(s, t["x"], *ops.quantize(t["x"]))


def _own_swiglu(s, t):
    from tannic_amd import ops
    return _own_values(s, t["gate"], *ops.swiglu_quantized(t["gate"], t["up"]))


def _own_product(s, t):
    from tannic_amd import ops
    return _seen(ops.matmul_quantized(t["a"], t["a_scales"], t["w"], t["w_scales"], s["type"]), s["dtype"])


_OWN = {"norm": _own_norm, "quantize": _own_quantize, "swiglu": _own_swiglu, "product": _own_product}


def _in_8_bits(u, factor, dtype):
    """The values that u * factor (a factor for each row) stands for in 8 bits, and the rows' scales: the factor cancels in the integers."""
    most = u.abs().amax(-1, keepdim=True).clamp(min=_LEAST)
    integers = torch.round(u * (127.0 / most))
    scales = most * factor / 127.0
    return (integers * scales).to(dtype), scales[..., 0]


def _plain_norm(s):
    total = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["dtype"])
    x = total.float()
    factor = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
    if s["bits"] == 8:
        outputs = _in_8_bits(x * s["gain"].float(), factor, s["dtype"])
    else:
        outputs = ((x * factor * s["gain"].float()).to(s["dtype"]),)
    return outputs if s["residual"] is None else outputs + (total,)


def _plain_quantize(s):
    return _in_8_bits(s["x"].float(), 1.0, s["dtype"])


def _plain_swiglu(s):
    gate = s["gate"].float()
    return _in_8_bits(gate / (1.0 + torch.exp(-gate)) * s["up"].float(), 1.0, s["dtype"])


def _plain_product(s):
    sums = s["a"].float() @ s["w"].float().t()
    return (sums * s["a_scales"][:, None] * s["w_scales"]).to(s["dtype"])


_PLAIN = {"norm": _plain_norm, "quantize": _plain_quantize, "swiglu": _plain_swiglu, "product": _plain_product}


# ---- by definition, in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "product":
        # (a block of tokens at a time)
        w = s["w"].double().t().contiguous()
        out = torch.empty((case["rows"], case["columns"]), dtype=torch.float64, device=_DEVICE)
        for i in range(0, case["rows"], 1024):
            out[i:i + 1024] = torch.mm(s["a"][i:i + 1024].double(), w)
        return out.mul_(s["a_scales"].double()[:, None]).mul_(s["w_scales"].double())
    total = None
    if case["kind"] == "swiglu":
        gate, up = s["gate"].double(), s["up"].double()
        y = gate * torch.sigmoid(gate) * up
    elif case["kind"] == "quantize":
        y = s["x"].double()
    else:
        y = s["x"].double()
        if case["residual"]:
            # (what is normed is the sum as it is kept)
            total = y + s["residual"].double()
            y = total.to(s["dtype"]).double()
        y = y / torch.sqrt(torch.sum(y * y, -1, keepdim=True) / case["width"] + s["eps"]) * s["gain"].double()
        if case["bits"] != 8:
            return (y,) if total is None else (y, total)
    scale = torch.linalg.vector_norm(y, ord=math.inf, dim=-1, keepdim=True) / 127
    values = torch.round(y / scale) * scale
    return (values, scale[:, 0]) if total is None else (values, scale[:, 0], total)
