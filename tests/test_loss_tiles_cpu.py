"""How a head's two gradient products are dealt out to the SMs (csrc/loss_plan.h), compiled by itself: against a search over all
ways, and in a time that does not grow with the tiles."""
import ctypes
import os
import random
import shutil
import subprocess
import time

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnabla_b200", "csrc")

PROGRAM = r"""
#include "loss_plan.h"
extern "C" int64_t extra(int64_t first, int64_t second, int64_t first_cycles, int64_t second_cycles, int64_t units) {
  return nb200::extra_tiles(first, second, first_cycles, second_cycles, units);
}
"""


@pytest.fixture(scope="module")
def extra(tmp_path_factory):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("tiles")
    (d / "tiles.cpp").write_text(PROGRAM)
    subprocess.run([cc, "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + CSRC, str(d / "tiles.cpp"), "-o", str(d / "tiles.so")],
                   check=True)
    lib = ctypes.CDLL(str(d / "tiles.so"))
    lib.extra.restype = ctypes.c_int64
    return lambda *a: lib.extra(*[ctypes.c_int64(v) for v in a])


def search(first, second, first_cycles, second_cycles, units):
    more = first % units
    if more == 0 or second == 0:
        return 0
    best, at = None, 0
    for n in range((second + more - 1) // more + 1):
        rest = max(0, second - more * n)
        t = max(first_cycles + n * second_cycles, -(-rest // (units - more)) * second_cycles)
        if best is None or t < best:
            best, at = t, n
    return at


def test_the_last_unit_ends_first(extra):
    rng = random.Random(3)
    for _ in range(20000):
        units = rng.choice([74, 148, 66, 1, 2, 10])
        first, second = rng.randint(0, 3 * units), rng.choice([0, rng.randint(1, 40), rng.randint(1, 4000)])
        args = (first, second, rng.randint(2000, 200000), rng.randint(2000, 200000), units)
        assert extra(*args) == search(*args), args


def test_many_tiles_take_no_time(extra):
    t = time.perf_counter()
    for _ in range(1000):
        extra(149, 1 << 30, 2000, 2000, 148)
    assert time.perf_counter() - t < 1.0  # (a search over all of them is 2^30 steps a call)
