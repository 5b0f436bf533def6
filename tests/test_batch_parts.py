"""A row's parts as the attention kernel counts them, by a quotient in F32
(csrc/batch_rules.h, compiled here by itself), against whole numbers. CPU only."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "batch_rules.h"
using namespace frz::rules;

static uint32_t whole(uint32_t blocks, uint32_t chunk) {
  return chunk ? (blocks + chunk - 1) / chunk : 0;
}

// How often the count is off for blocks of [from, to) by `step`.
int main(int argc, char** argv) {
  if (argc != 5) return 1;
  const uint32_t chunk = strtoul(argv[1], 0, 10), from = strtoul(argv[2], 0, 10),
                 to = strtoul(argv[3], 0, 10), step = strtoul(argv[4], 0, 10);
  const float each = 1.0f / (float)(chunk ? chunk : 1);
  uint32_t off = 0;
  for (uint32_t b = from; b < to; b += step)
    off += row_parts(b, chunk, each) != whole(b, chunk);
  // What a reciprocal off by one ulp either way would give.
  for (uint32_t b = from; b < to; b += step)
    off += row_parts(b, chunk, each * (1.0f + 0x1p-23f)) != whole(b, chunk);
  for (uint32_t b = from; b < to; b += step)
    off += row_parts(b, chunk, each * (1.0f - 0x1p-24f)) != whole(b, chunk);
  std::printf("%u\n", off);
}
"""


@pytest.fixture(scope="module")
def off(tmp_path_factory):
    d = tmp_path_factory.mktemp("parts")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I",
                    str(ROOT / "frizzle_amd" / "csrc"), str(d / "main.cpp"), "-o",
                    str(d / "parts")], check=True)
    return lambda *a: int(subprocess.run([str(d / "parts"), *map(str, a)], check=True,
                                         capture_output=True, text=True).stdout)


# All rows of up to 2^19 blocks (2^24 keys) and one, by every small chunk and some
# of the larger ones that a batch's even shares give.
@pytest.mark.parametrize("chunks", [range(1, 13), (16, 28, 100, 404, 1020, 1024, 1028, 4096),
                                    (5460, 8188, 43692, 65536, 174764, 524288)])
def test_parts_are_the_blocks_over_the_chunk_rounded_up(off, chunks):
    for chunk in chunks:
        assert off(chunk, 0, (1 << 19) + 2, 1) == 0, chunk


def test_rows_up_to_the_limit(off):
    for chunk in (1, 2, 4, 12, 1000, 700000):
        assert off(chunk, 0, 1 << 20, 37) == 0 and off(chunk, (1 << 20) - 999, 1 << 20, 1) == 0


def test_no_chunk_no_parts(off):
    # A batch of no rows: its chunk is none, and so are its parts.
    assert off(0, 0, 1, 1) == 0
