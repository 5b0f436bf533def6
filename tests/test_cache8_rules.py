"""The rules of first keys and of blocks' scales (csrc/batch_rules.h, compiled here by
itself): every key of a row in one block as counted, and the least power of two. CPU
only."""
import math
import struct
import subprocess
from pathlib import Path

import pytest

from _cache8 import block_scale

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>
#include "batch_rules.h"
using namespace frz::rules;

// Rows whose blocks hold other keys than theirs, or one twice, and rows of more
// blocks than the most.
static int wrong(uint32_t window, uint32_t sinks, uint32_t capacity, uint32_t to) {
  int off = 0;
  for (uint32_t p = 0; p < to; ++p) {
    const KeyRange r = key_range(p, window, capacity, sinks);
    const uint32_t n = row_blocks(r);
    std::set<uint32_t> got, want;
    size_t count = 0;
    for (uint32_t i = 0; i < n; ++i) {
      const BlockKeys b = block_keys(r, i);
      for (uint32_t j = b.block * kBlockKeys; j < (b.block + 1) * kBlockKeys; ++j)
        if (j >= b.first && j < b.end) {
          got.insert(j);
          ++count;
        }
    }
    for (uint32_t j = 0; j <= p && j < capacity; ++j)
      if (j < sinks || p - j < window) want.insert(j);
    off += got != want || count != got.size() || n > most_row_blocks(capacity, window, sinks);
  }
  return off;
}

// Rows whose parts, cut as evenly as fours leave them, are not as many as the chunk's,
// none empty and none longer.
static int uneven(uint32_t chunk, uint32_t to) {
  int off = 0;
  for (uint32_t n = 1; n < to; ++n) {
    const uint32_t parts = row_parts(n, chunk, 1.0f / chunk), each = row_chunk(n, parts, chunk);
    off += each > chunk || parts * each < n || (parts - 1) * each >= n;
  }
  return off;
}

int main(int argc, char** argv) {
  if (argc == 3) {
    std::printf("%d\n", uneven(strtoul(argv[1], 0, 10), strtoul(argv[2], 0, 10)));
    return 0;
  }
  if (argc == 5)
    std::printf("%d\n", wrong(strtoul(argv[1], 0, 10), strtoul(argv[2], 0, 10),
                              strtoul(argv[3], 0, 10), strtoul(argv[4], 0, 10)));
  for (int i = 1; argc != 5 && i < argc; ++i)
    std::printf("%u\n", block_scale_bits(strtoul(argv[i], 0, 10)));
  return 0;
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules8")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I",
                    str(ROOT / "frizzle_amd" / "csrc"), str(d / "main.cpp"), "-o",
                    str(d / "rules")], check=True)
    return lambda *a: [int(x) for x in subprocess.run([str(d / "rules"), *map(str, a)],
                                                      check=True, capture_output=True,
                                                      text=True).stdout.split()]


@pytest.mark.parametrize("sinks", [0, 1, 4, 31, 32, 33, 64, 100, 0xFFFFFFFF])
@pytest.mark.parametrize("window", [1, 16, 32, 33, 100, 0xFFFFFFFF])
@pytest.mark.parametrize("capacity", [0, 16, 96, 400])
def test_every_key_in_one_block(rules, sinks, window, capacity):
    assert rules(window, sinks, capacity, 450) == [0]


@pytest.mark.parametrize("chunk", [1, 2, 4, 8, 12, 16, 44, 84, 132, 1000, 4096])
def test_parts_of_a_row_are_even(rules, chunk):
    assert rules(chunk, 20000) == [0]


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


def number(b):
    return struct.unpack("<f", struct.pack("<I", b))[0]


def test_scales_are_the_least_powers_of_two(rules):
    values = [0.0, 2.0 ** -149, 1e-40, 2.0 ** -126, 127 * 2.0 ** -126, 1.0, 126.99999, 127.0,
              127.00001, 128.0, 253.9, 254.0, 254.1, 1e-3, 0.7, 5.5, 1e30, number(0x7F7FFFFF)]
    for x, got in zip(values, rules(*map(bits, values))):
        scale = number(got)
        if x == 0:
            assert scale == 0
            continue
        assert math.frexp(scale)[0] == 0.5 and 2.0 ** -126 <= scale <= 2.0 ** 121
        assert x <= 127 * scale or scale == 2.0 ** 121
        assert scale == 2.0 ** -126 or x > 127 * scale / 2
        assert scale == block_scale(number(bits(x)))


def test_scales_past_the_range_are_the_last(rules):
    assert [number(b) for b in rules(bits(math.inf), bits(3.4e38), bits(math.inf))] == [
        2.0 ** 121] * 3
