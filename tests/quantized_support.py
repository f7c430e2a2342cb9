"""The operators on rows of 8-bit integers restated in numpy: by their definition in 64 bits, and step by step in fp32 where the steps are whole-number or single roundings."""
import numpy as np

import tannic_amd as ta

HALF = {ta.float16: 2.0 ** -11, ta.bfloat16: 2.0 ** -8, ta.float32: 2.0 ** -24}     # of a rounding, relative
TINY = {ta.float16: 2.0 ** -25, ta.bfloat16: 0.0, ta.float32: 0.0}                  # and absolute, below the smallest normal number
LEAST = np.float32(2.0 ** -119)


def rounded(x, dtype):
    """x as a tensor of the type holds it, in fp32."""
    return ta.tensor(np.asarray(x), dtype).numpy().astype(np.float32)


def integers_of(u):
    """values, largest and whether finite, of rows u in fp32: every step is one rounding."""
    u = np.asarray(u, np.float32)
    most = np.abs(u).max(-1, initial=0.0, keepdims=True) if u.shape[-1] else np.zeros(u.shape[:-1] + (1,), np.float32)
    finite = np.isfinite(u).all(-1, keepdims=True)
    largest = np.maximum(np.where(finite, most, 1.0), LEAST).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        values = np.rint(np.where(finite, u, 0.0).astype(np.float32) * (np.float32(127) * (np.float32(1) / largest))).astype(np.int8)
    return values, largest[..., 0], finite[..., 0]


def assert_stands_for(values, scales, want, slack, what=""):
    """values * scales are the rows `want` (64 bits): every element is off by half a scale at most, and by what its u (relative to the row's largest) and the scale are off by: `slack`,
    and 2^-22 for the factor, its product with u, the scale and a tie.  The largest is 127 scales, to the same 2^-22 and `slack`."""
    values, scales = values.astype(np.float64), scales.astype(np.float64)[..., None]
    most = np.maximum(np.abs(want).max(-1, initial=0.0, keepdims=True), float(LEAST))
    assert (np.abs(values) <= 127).all(), what
    assert (np.abs(scales * 127 - most) <= (slack + 2.0 ** -22) * most).all(), what
    bound = 0.5 * scales + (2 * slack + 2.0 ** -21) * most
    assert (np.abs(values * scales - want) <= bound).all(), (what, float((np.abs(values * scales - want) / bound).max()))


def product(a, a_scales, b, b_scales):
    """The product in fp32 as it is defined: the exact sums rounded, times both scales, each once."""
    sums = (a.astype(np.float64) @ b.astype(np.float64))        # (exact: below 2^53)
    return sums.astype(np.float32) * a_scales[..., :, None].astype(np.float32) * b_scales[..., None, :].astype(np.float32)
