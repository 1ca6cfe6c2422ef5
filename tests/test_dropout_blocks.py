"""The block of an element as the kernels form it, the upper half once for a CTA and the lower one for each thread, on the CPU: element / 4
wherever a CTA begins, past 2^34 elements too, where the counter's second word is no longer 0."""
import ctypes
import os
import subprocess

import pytest

from conftest import PKG_DIR

SOURCE = """
#include "dfa3d_philox.cuh"
extern "C" long long wrong(unsigned long long base, uint32_t width) {
  long long n = 0;
  for (uint32_t e = 0; e < width; e += 4) n += dfa3d::block_of(base, e) != (base + e) / 4;
  return n;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("blocks")
    (d / "blocks.cpp").write_text(SOURCE)
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "blocks.cpp"), "-o", str(d / "blocks.so")], check=True)
    lib = ctypes.CDLL(str(d / "blocks.so"))
    lib.wrong.argtypes, lib.wrong.restype = [ctypes.c_uint64, ctypes.c_uint32], ctypes.c_longlong
    return lib


@pytest.mark.parametrize("width", [2048, 4096])
@pytest.mark.parametrize("around", [0, 2 ** 31, 2 ** 33, 2 ** 34, 3 * 2 ** 34, 2 ** 40, 2 ** 42])
def test_block_is_element_by_four(lib, width, around):
    for k in range(-3, 4):
        base = around + k * width
        if base >= 0:
            assert lib.wrong(base, width) == 0, base
