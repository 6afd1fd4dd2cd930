"""CPU: index arithmetic of the cache attention kernels that must stay in bounds
after a wait that gave up (csrc/cache_bounds.h), compiled with the host compiler."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "burn_image_b200", "csrc")
SOURCE = """
#include "cache_bounds.h"
extern "C" void slots(int from, int to, int range, int grid, int* out) {
  const bq4::CacheSlots s = bq4::cache_slots(from, to, range, grid);
  out[0] = s.first, out[1] = s.count;
}
extern "C" int pending(int j, int mine, int stages) { return bq4::cache_pending(j, mine, stages); }
"""


@pytest.fixture(scope="module")
def bounds(tmp_path_factory):
    at = tmp_path_factory.mktemp("bounds")
    (at / "b.cc").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(at / "b.so"),
                    str(at / "b.cc")], check=True)
    return ctypes.CDLL(str(at / "b.so"))


def slots(lib, *a):
    out = (ctypes.c_int * 2)()
    lib.slots(*a, out)
    return tuple(out)


def test_written_slots_are_kept(bounds):
    for grid in (1, 5, 592):
        for a in {0, grid // 3, grid - 1}:
            for z in {a, (a + grid) // 2, grid - 1}:
                assert slots(bounds, a, z, 11, grid) == (a + 11, z - a + 1)


def test_whatever_the_workspace_holds_the_slots_exist(bounds):
    rng = random.Random(3)
    odd = [-2 ** 31, -1, 0, 1, 2 ** 31 - 1, 0x7f800000, 0x7fc00000 - 2 ** 31]
    for grid in (1, 2, 444, 592):
        for range_ in (0, 7, 0x3fffffff):
            some = odd + [grid - 1, grid, -grid] + [rng.randrange(-2 ** 31, 2 ** 31) for _ in range(40)]
            for a in some:
                for z in some:
                    first, count = slots(bounds, a, z, range_, grid)
                    assert range_ <= first and 1 <= count and first + count <= range_ + grid


def test_every_copy_under_way_is_waited_for(bounds):
    # the ring as the kernel drives it: stages - 1 fetches ahead, one more at the start of each step
    for stages in range(2, 9):
        for mine in range(20):
            for fails in range(mine + 1):
                issued = min(mine, stages - 1)
                waited = 0
                for j in range(mine):
                    if j + stages - 1 < mine:
                        issued += 1
                    if j == fails:
                        break
                    waited += 1
                assert bounds.pending(fails, mine, stages) == issued - waited
