"""The C++ functions of rows in 8-bit integers on the device, over a stand-in of the front end: what the Python functions give, bit for bit."""
import subprocess

import numpy as np
import pytest

import adapter_quantized_build
import tannic_amd as ta
from tannic_amd import ops

pytestmark = pytest.mark.gpu


def test_the_functions_on_the_device(tmp_path, device):
    binary = adapter_quantized_build.build(str(tmp_path))
    rng = np.random.default_rng(95)
    given = [rng.standard_normal(s).astype(np.float32) for s in ((2, 3, 40), (2, 3, 40), (40,), (40, 40))]
    (tmp_path / "in").write_bytes(b"".join(x.tobytes() for x in given))
    done = subprocess.run([binary, str(tmp_path / "in"), str(tmp_path / "out")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout + done.stderr
    x, residual, gain, w = (ta.tensor(t, ta.float32, device) for t in given)
    q, scales = ops.quantize(x)
    weights, channels = ops.quantize(w)
    want = [scales, ops.dequantize(q, scales, ta.float32), ops.matmul_quantized(q, scales, weights, channels, ta.float32), ops.dequantize(*ops.swiglu_quantized(x, residual), ta.float32),
            ops.dequantize(*ops.add_rms_norm_quantized(x, None, gain, 0.5)[:2], ta.float32), *ops.add_rms_norm(x, residual, gain, 0.25)]
    in_8_bits = ops.add_rms_norm_quantized(x, residual, gain, 0.25)
    want += [ops.dequantize(*in_8_bits[:2], ta.float32), in_8_bits[2]]
    assert (tmp_path / "out").read_bytes() == b"".join(np.ascontiguousarray(t.numpy()).tobytes() for t in want)
