"""The C++ functions of rows in 8-bit integers hand every operand to its place: compiled over a stand-in of the front end, with the library's entry points replaced."""
import subprocess

import adapter_quantized_build


def test_the_functions_hand_over_what_they_were_given(tmp_path):
    binary = adapter_quantized_build.build(str(tmp_path), "-DRECORD")
    (tmp_path / "none").write_bytes(b"")
    done = subprocess.run([binary, str(tmp_path / "none"), str(tmp_path / "out")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr
    # x residual gain w: 1 .. 4; the integers and scales of x 5 and 6, of w 7 and 8; types 2: 8-bit integers, 8: float
    assert done.stdout.splitlines() == [
        "quantize 1:8[2,3,40] 5:2[2,3,40] 6:8[2,3] stream 77",
        "quantize 4:8[40,40] 7:2[40,40] 8:8[40] stream 77",
        "dequantize 5:2[2,3,40] 6:8[2,3] 9:8[2,3,40] stream 77",
        "gemm_quantized 5:2[2,3,40] 6:8[2,3] 7:2[40,40] 8:8[40] 10:8[2,3,40] stream 77",
        "swiglu_quantize 1:8[2,3,40] 2:8[2,3,40] 11:2[2,3,40] 12:8[2,3] stream 77",
        "dequantize 11:2[2,3,40] 12:8[2,3] 13:8[2,3,40] stream 77",
        "add_rms_norm 1:8[2,3,40] - 3:8[40] - 14:2[2,3,40] 15:8[2,3] stream 77 eps 0.5",
        "dequantize 14:2[2,3,40] 15:8[2,3] 16:8[2,3,40] stream 77",
        "add_rms_norm 1:8[2,3,40] 2:8[2,3,40] 3:8[40] 17:8[2,3,40] 18:8[2,3,40] - stream 77 eps 0.25",
        "add_rms_norm 1:8[2,3,40] 2:8[2,3,40] 3:8[40] 21:8[2,3,40] 19:2[2,3,40] 20:8[2,3] stream 77 eps 0.25",
        "dequantize 19:2[2,3,40] 20:8[2,3] 22:8[2,3,40] stream 77",
        "host: quantize: implemented by the device backend only (move the operands to a Device)",
        "mixed: swiglu_quantized: operands live in different environments",
        "scalar: operands have rank >= 1",
        "ranks: Inputs must have rank >= 2",
        "inner: Inner dimensions must match for matmul",
        "add_rms_norm 1:8[2,3,40] 2:8[2,3,40] 3:8[40] 26:8[2,3,40] 27:8[2,3,40] - stream 77 eps 1",
        "types: add_rms_norm: unsupported dtype",
        "dequantize 1:8[2,3,40] 2:8[2,3,40] 28:8[2,3,40] stream 77",
        "refused: dequantize: rejected by the device backend (shapes or dtypes do not fit)",
    ]
