"""Builds tests/adapter_attention.cpp over the stand-in of the front end."""
import os
import subprocess

TESTS = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(TESTS)
CSRC = os.path.join(ROOT, "tannic_amd", "csrc")
HEADERS = ["callback.hpp", "concepts.hpp", "exceptions.hpp", "expressions.hpp", "indexing.hpp", "operations.hpp", "reductions.hpp", "tensor.hpp", "runtime/resources.h",
           "runtime/status.h", "runtime/streams.h", "runtime/tensor.h", "runtime/types.h"]


def build(where, *flags):
    os.makedirs(os.path.join(where, "runtime"), exist_ok=True)
    for name in HEADERS:
        with open(os.path.join(where, name), "w") as f:
            f.write('#include "frontend_standin.hpp"\n')
    binary = os.path.join(where, "adapter_attention")
    done = subprocess.run(["g++", "-std=c++20", "-O0", "-Wall", *flags, "-I", str(where), "-I", TESTS, "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CSRC, "adapter"),
                           os.path.join(TESTS, "adapter_attention.cpp"), os.path.join(CSRC, "adapter", "adapter.cpp"), "-L", CSRC, "-ltannic_hip", f"-Wl,-rpath,{CSRC}", "-o", binary],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-4000:]
    return binary
