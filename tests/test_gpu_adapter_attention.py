"""The C++ nodes of the attention and the cache on the device, over a stand-in of the front end, against the definition in 64 bits."""
import subprocess

import numpy as np
import pytest

import adapter_build
import tannic_amd as ta
from attention_support import assert_within, head_attention

pytestmark = pytest.mark.gpu


def attention(q, k, v, scale, seen):
    """q [n, heads, d] over k, v [length, kv heads, d]: result, slack, sum of p |v|."""
    out = [head_attention(q[:, h], k[:, h // 2], v[:, h // 2], scale, seen) for h in range(q.shape[1])]
    return [np.stack([o[i] for o in out], 1) for i in range(3)]


def test_the_nodes_on_the_device(tmp_path):
    binary = adapter_build.build(str(tmp_path))
    rng = np.random.default_rng(90)
    shapes = [(2, 3, 4, 16), (2, 9, 2, 16), (2, 9, 2, 16), (6, 2, 4, 16), (6, 2, 4, 16), (5, 2, 16), (5, 2, 16), (5, 4, 16), (8, 8), (8, 8)]
    given = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    (tmp_path / "in").write_bytes(b"".join(x.tobytes() for x in given))
    done = subprocess.run([binary, str(tmp_path / "in"), str(tmp_path / "out")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout + done.stderr
    raw = (tmp_path / "out").read_bytes()
    got, at = [], 0
    for shape in [shapes[0], shapes[0], shapes[3], shapes[3], shapes[7], shapes[3], shapes[3], shapes[7], shapes[3]]:
        n = 4 * int(np.prod(shape))
        got.append(np.frombuffer(raw[at:at + n], np.float32).reshape(shape))
        at += n
    assert at == len(raw)
    q, k, v, keys, values, new_k, new_v, new_q, cos, sin = (x.astype(np.float64) for x in given)
    for result, scale, lengths in ((got[0], 0.25, (9, 9)), (got[1], -0.5, (9, 4))):
        for b in (0, 1):
            want, slack, size = attention(q[b], k[b], v[b], scale, [lengths[b]] * 3)
            assert_within(result[b], want, slack, size, ta.float32)
    # the new tokens' places: (page, row) behind 2 and 4 of tables 1 3 and 0 4
    places, positions = [(1, 2), (1, 3), (3, 0), (4, 0), (4, 1)], [2, 3, 4, 4, 5]
    for (page, row), x, y in zip(places, new_k, new_v):
        keys[page, :, row], values[page, :, row] = x, y
    assert np.array_equal(got[2], keys) and np.array_equal(got[3], values)

    def turned(x):
        c, s, out = cos[positions][:, None], sin[positions][:, None], np.empty_like(x)
        out[..., 0::2], out[..., 1::2] = x[..., 0::2] * c - x[..., 1::2] * s, x[..., 0::2] * s + x[..., 1::2] * c
        # (both products and their sum are rounded)
        size = np.empty_like(x)
        size[..., 0::2], size[..., 1::2] = np.abs(x[..., 0::2] * c) + np.abs(x[..., 1::2] * s), np.abs(x[..., 0::2] * s) + np.abs(x[..., 1::2] * c)
        return out, 2 * 2.0 ** -24 * (1 + 2.0 ** -24) * size

    want, off = turned(new_q)
    assert (np.abs(got[4] - want) <= off).all()
    want, off = turned(new_k)
    for i, (page, row) in enumerate(places):
        assert (np.abs(got[5][page, :, row] - want[i]) <= off[i]).all()
        keys[page, :, row] = got[5][page, :, row]
    assert np.array_equal(got[5], keys) and np.array_equal(got[6], values)
    for tokens, pages, context in ((slice(0, 3), [1, 3], 2), (slice(3, 5), [0, 4], 4)):
        mine_k, mine_v = (np.concatenate([pool[p].transpose(1, 0, 2) for p in pages]) for pool in (keys, values))
        want, slack, size = attention(new_q[tokens], mine_k, mine_v, 0.125, context + 1 + np.arange(tokens.stop - tokens.start))
        assert_within(got[7][tokens], want, slack, size, ta.float32)
    keys[5] = keys[1]
    keys[2] = keys[5]
    assert np.array_equal(got[8], keys)
