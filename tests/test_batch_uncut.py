"""Which rows attention over pages leaves uncut (csrc/batch_rules.h, compiled here by
itself): as many blocks as the units allow, whatever leaves the rows that short. CPU
only."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
NONE = 0xFFFFFFFF
UNITS = 256  # compute units

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "batch_rules.h"
using namespace frz::rules;
int main(int argc, char** argv) {
  uint32_t a[7];
  for (int i = 0; i < 7 && i + 1 < argc; ++i) a[i] = strtoul(argv[i + 1], 0, 10);
  const uint64_t blocks = most_row_blocks(a[0], a[1], a[2]);
  std::printf("%llu %d\n", (unsigned long long)blocks, (int)uncut(blocks, a[3], a[4], a[5], a[6]));
}
"""


@pytest.fixture(scope="module")
def uncut(tmp_path_factory):
    d = tmp_path_factory.mktemp("uncut")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I",
                    str(ROOT / "frizzle_amd" / "csrc"), str(d / "main.cpp"), "-o",
                    str(d / "uncut")], check=True)

    def run(capacity, window, dim, i8, units, sinks=0):
        got = subprocess.run([str(d / "uncut"), *map(str, (capacity, window, sinks, dim, int(i8),
                                                           units, UNITS))],
                             check=True, capture_output=True, text=True).stdout.split()
        return int(got[0]), bool(int(got[1]))
    return run


@pytest.mark.parametrize("units", [96, 130, 200, 255, 256, 257, 300, 512, 4096])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 100, 512, 900, 1000, 1500, 2000, 4000, 8000])
@pytest.mark.parametrize("sinks", [0, 5])
def test_16_bits_as_without_a_window(uncut, units, dim, window, sinks):
    # 1 MB of keys and values a workgroup at most, so 26 us by the 40 GB/s that a compute
    # unit takes in: younger requests' rows than the longest are over long before. A table
    # of as many blocks is cut, or not, alike.
    blocks, whole = uncut(8192, window, dim, False, units, sinks)
    assert whole == (blocks * 32 * dim * 2 * 2 <= 1 << 20)
    if blocks <= 255:
        assert uncut(32 * blocks, NONE, dim, False, units) == (blocks, whole)


@pytest.mark.parametrize("units", [1, 16, 61, 95])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 100, 256, 512, 1000, 2000])
def test_16_bits_where_units_are_few(uncut, units, dim, window):
    blocks, whole = uncut(8192, window, dim, False, units)
    assert whole == (blocks * dim <= 2048)


@pytest.mark.parametrize("units,most", [(1, 16), (32, 16), (95, 16), (96, 36), (300, 36),
                                        (4096, 36)])
@pytest.mark.parametrize("window", [1, 250, 400, 460, 600, 900, 1000, 1080, 1200, 2000, 4000])
def test_8_bits_by_their_blocks(uncut, units, most, window):
    blocks, whole = uncut(65536, window, 256, True, units)
    assert whole == (blocks <= most)
    assert uncut(32 * blocks, NONE, 256, True, units) == (blocks, whole)


@pytest.mark.parametrize("dim", [64, 128])
def test_8_bits_of_narrow_heads_as_16(uncut, dim):
    for units, most in ((32, 2048), (300, 8192)):
        for window in (300, 400, 1000, 2000, 4000, 8000):
            blocks, whole = uncut(65536, window, dim, True, units)
            assert whole == (blocks * dim <= most)
