"""What a dropout keeps, on the CPU: the generator against published vectors and against its definition, the rule that p makes."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import row_reference as R
from conftest import PKG_DIR

SOURCE = """
#include "dfa3d_philox.cuh"
using namespace dfa3d;
extern "C" void words(unsigned long long block, uint32_t site, uint64_t seed, uint32_t *out) {
  const PhiloxWords w = philox_words(block, site, DropKey{(uint32_t)seed, (uint32_t)(seed >> 32)});
  out[0] = w.x; out[1] = w.y; out[2] = w.z; out[3] = w.w;
}
extern "C" int rule(double p, uint32_t *last, float *scale) {
  const DropRule r = drop_rule(p, nullptr, 0);
  *last = r.last; *scale = r.scale;
  return r.rng;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("philox")
    (d / "philox.cpp").write_text(SOURCE)
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "philox.cpp"), "-o", str(d / "philox.so")], check=True)
    lib = ctypes.CDLL(str(d / "philox.so"))
    lib.words.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint64, ctypes.POINTER(ctypes.c_uint32)]
    lib.rule.argtypes = [ctypes.c_double, ctypes.POINTER(ctypes.c_uint32), ctypes.POINTER(ctypes.c_float)]
    return lib


def words(lib, block, site, seed):
    out = (ctypes.c_uint32 * 4)()
    lib.words(block, site, seed & (2 ** 64 - 1), out)
    return list(out)


def test_generator_gives_the_published_vector_of_seven_rounds(lib):
    assert words(lib, 0, 0, 0) == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]


@pytest.mark.parametrize("seed,site", [(0, 0), (-1, 5), (123456789, 2 ** 31 - 1), (-2 ** 63, 1)])
def test_generator_gives_its_definition(lib, seed, site):
    want = R.philox_words(400, seed, site).reshape(-1, 4)
    for block in range(100):
        assert words(lib, block, site, seed) == want[block].tolist()


def test_blocks_past_32_bits_differ_from_those_below(lib):
    a, b = words(lib, 7, 3, 99), words(lib, 7 + (1 << 32), 3, 99)
    assert all(x != y for x, y in zip(a, b))


@pytest.mark.parametrize("p", [2.0 ** -33, 1e-9, 0.1, 0.5, 0.9, 1 - 1e-9, 1 - 2.0 ** -34, 1.0])
def test_rule_drops_what_p_says(lib, p):
    last, scale = ctypes.c_uint32(), ctypes.c_float()
    assert lib.rule(p, last, scale) == 1
    assert last.value == int(p * 2 ** 32 + 0.5) - 1
    assert scale.value == (np.float32(1 / (1 - p)) if p < 1 else 0)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -34])
def test_rule_needs_no_words_where_nothing_is_dropped(lib, p):
    last, scale = ctypes.c_uint32(), ctypes.c_float()
    assert lib.rule(p, last, scale) == 0
    assert scale.value == 1.0
