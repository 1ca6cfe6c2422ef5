"""How the rows of a feature pyramid are cut up for the group norm (csrc/dfa3d_segments.h), on the CPU: whatever the level table says,
the segments are disjoint and cover the rows, pieces have numbers of their own."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import PKG_DIR

SOURCE = """
#include "dfa3d_segments.h"
using namespace dfa3d;
extern "C" int segments(const int64_t *shapes, int stride, const int64_t *start, int L, int N, int *end) {
  SegmentTable t;
  make_segments(t, shapes, stride, start, L, N);
  for (int i = 0; i < t.count; ++i) end[i] = t.end[i];
  return t.count;
}
extern "C" int divided(int n, uint32_t d) { return quotient(n, make_divisor(d)); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("segments")
    (d / "segments.cpp").write_text(SOURCE)
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "segments.cpp"), "-o", str(d / "segments.so")], check=True)
    return ctypes.CDLL(str(d / "segments.so"))


def segments(lib, shapes, start, N, stride=2):
    L = len(start)
    flat = [v for s in shapes for v in (list(s) + [77])[:stride]]
    a, b, end = (ctypes.c_int64 * len(flat))(*flat), (ctypes.c_int64 * L)(*start), (ctypes.c_int * (2 * L + 1))()
    assert lib.segments(a, stride, b, L, N, end) == 2 * L + 1
    return list(end)


def test_ordinary_table(lib):
    assert segments(lib, [(4, 5), (2, 3), (1, 1)], [0, 20, 26], 27) == [0, 20, 20, 26, 26, 27, 27]
    assert segments(lib, [(4, 5), (2, 3), (1, 1)], [0, 20, 26], 27, stride=3) == [0, 20, 20, 26, 26, 27, 27]


def test_one_level_without_a_table(lib):
    end = (ctypes.c_int * 3)()
    assert lib.segments(None, 0, None, 1, 55, end) == 3 and list(end) == [0, 55, 55]


def test_gaps_and_rows_behind_the_last_level(lib):
    assert segments(lib, [(2, 2), (1, 3)], [1, 7], 12) == [1, 5, 7, 10, 12]


@pytest.mark.parametrize("shapes,start,N,want", [
    ([(4, 5)], [0], 10, [0, 10, 10]),                               # past the end
    ([(4, 5)], [-3], 40, [0, 20, 40]),                              # before the beginning
    ([(4, 5), (2, 2)], [0, 10], 40, [0, 20, 20, 20, 40]),           # the second lies in the first
    ([(4, 5), (2, 3)], [0, 18], 40, [0, 20, 20, 24, 40]),           # and sticks out of it
    ([(-1, 5), (2, 0)], [0, 4], 9, [0, 0, 4, 4, 9]),                # no rows
    ([(2 ** 40, 2 ** 40)], [2 ** 62], 9, [9, 9, 9]),
    ([(2 ** 62, 2 ** 62)], [0], 9, [0, 9, 9]),
    ([(3, 3), (3, 3)], [9, 0], 18, [9, 18, 18, 18, 18]),            # backwards: the second has no rows left
])
def test_tables_that_do_not_fit_are_cut(lib, shapes, start, N, want):
    assert segments(lib, shapes, start, N) == want


def test_any_table_gives_disjoint_ascending_segments(lib):
    rng = random.Random(3)
    for _ in range(2000):
        L, N = rng.randint(1, 6), rng.randint(1, 50)
        big = rng.choice((8, 60, 2 ** 31, 2 ** 62))
        shapes = [(rng.randint(-2, big), rng.randint(-2, big)) for _ in range(L)]
        end = segments(lib, shapes, [rng.randint(-big, big) for _ in range(L)], N)
        assert all(0 <= a <= b for a, b in zip([0] + end, end)) and end[-1] == N


def test_pieces_have_their_own_numbers(lib):
    rng = random.Random(4)
    for _ in range(300):
        n, R = rng.randint(1, 200), rng.randint(1, 60)
        cuts = sorted(rng.randint(0, n) for _ in range(6))
        segment = [sum(r >= c for c in cuts) for r in range(n)]
        numbers = {}
        for r in range(n):
            piece = (lib.divided(r, R), segment[r])
            assert numbers.setdefault(sum(piece), piece) == piece
            assert sum(piece) < -(-n // R) + 7


def test_division_by_a_number_of_the_host(lib):
    rng = random.Random(6)
    numbers = [1, 2, 3, 5, 7, 10, 375, 920, 30825, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1]
    for d in numbers + [rng.randint(1, 2 ** 31 - 1) for _ in range(200)] + [rng.randint(1, 1000) for _ in range(200)]:
        for n in [0, 1, d - 1, d, min(2 * d - 1, 2 ** 31 - 1), 2 ** 31 - 1] + [rng.randint(0, 2 ** 31 - 1) for _ in range(50)]:
            assert lib.divided(n, d) == n // d
