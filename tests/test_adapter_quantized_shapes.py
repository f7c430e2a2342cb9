"""What shape a product of 8-bit integers has in the C++ front end: that of the Python operators, an empty batch over one matrix included (a target of another extent is refused by the device)."""
import os
import subprocess

from adapter_build import CSRC, HEADERS, ROOT, TESTS


def test_shapes(tmp_path):
    os.makedirs(tmp_path / "runtime", exist_ok=True)
    for name in HEADERS:
        (tmp_path / name).write_text('#include "frontend_standin.hpp"\n')
    binary = str(tmp_path / "shapes")
    done = subprocess.run(["g++", "-std=c++20", "-O0", "-Wall", "-I", str(tmp_path), "-I", TESTS, "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CSRC, "adapter"),
                           os.path.join(TESTS, "adapter_quantized_shapes.cpp"), os.path.join(CSRC, "adapter", "adapter.cpp"), "-L", CSRC, "-ltannic_hip", f"-Wl,-rpath,{CSRC}", "-o", binary],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-4000:]
    out = subprocess.run([binary], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.split() == ["[4,5]", "[2,3,4,5]", "[3,4,5]", "[2,3,4,5]", "[0,4,5]", "[0,4,5]", "[0,4,5]", "[2,0,4,5]", "[0,3,4,5]"], out.stdout
