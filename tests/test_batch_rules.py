"""The rules by which a batch of requests finds its pages and cuts its
attention into parts (csrc/batch_rules.h, compiled here by itself): every block
of every row in one part, within the grid and the workspace that the launcher
sizes. CPU only."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "batch_rules.h"
using namespace frz::rules;

// A batch's cut as the kernel makes it.
static void cut(const std::vector<uint32_t>& lengths, uint32_t window, uint32_t capacity,
                uint32_t head_blocks, uint32_t at_once) {
  const uint32_t units = lengths.size() * head_blocks;
  std::vector<uint32_t> blocks;
  uint64_t all = 0;
  for (uint32_t n : lengths) {
    const uint32_t b = n ? row_blocks(key_range(n - 1, window, capacity)) : 0;
    blocks.push_back(b);
    all += b;
  }
  const uint32_t chunk = part_chunk(all * head_blocks, units, at_once, [&](uint32_t c) {
    uint32_t n = 0;
    for (uint32_t b : blocks) n += c ? (b + c - 1) / c : 0;
    return n * head_blocks;
  });
  uint64_t parts = 0, joined = 0;
  bool covered = true;
  for (uint32_t b : blocks) {
    const uint32_t p = chunk ? (b + chunk - 1) / chunk : 0;
    uint64_t sum = 0;
    for (uint32_t i = 0; i < p; ++i) {
      const uint32_t to = (i + 1) * chunk < b ? (i + 1) * chunk : b;
      covered = covered && to > i * chunk;
      sum += to - i * chunk;
    }
    covered = covered && sum == b;
    parts += (uint64_t)p * head_blocks;
    if (p > 1) joined += (uint64_t)p * head_blocks;
  }
  std::printf("%u %llu %u %llu %u %d\n", chunk, (unsigned long long)parts,
              most_parts(units, at_once), (unsigned long long)joined,
              most_joined_parts(units, at_once), (int)covered);
}

int main(int argc, char** argv) {
  if (argc == 4) {
    const KeyRange r = key_range(strtoul(argv[1], 0, 10), strtoul(argv[2], 0, 10),
                                 strtoul(argv[3], 0, 10));
    std::printf("%u %u %u\n", r.first, r.end, row_blocks(r));
    return 0;
  }
  if (argc == 1) {  // pages: a table of two rows of three over a pool of 7
    const uint32_t table[6] = {3, 6, kNone, 7, 0, 4000000000u};
    for (uint32_t s = 0; s < 4; ++s)
      for (uint32_t i = 0; i < 5; ++i) std::printf("%u ", page_at(table, 2, 3, 7, s, i));
    std::printf("%u\n", page_at(table, 2, 3, 7, kNone, kNone));
    return 0;
  }
  std::vector<uint32_t> lengths;
  for (int i = 5; i < argc; ++i) lengths.push_back(strtoul(argv[i], 0, 10));
  cut(lengths, strtoul(argv[1], 0, 10), strtoul(argv[2], 0, 10), strtoul(argv[3], 0, 10),
      strtoul(argv[4], 0, 10));
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I",
                    str(ROOT / "frizzle_amd" / "csrc"), str(d / "main.cpp"), "-o",
                    str(d / "rules")], check=True)

    def run(*args):
        return subprocess.run([str(d / "rules"), *map(str, args)], check=True,
                              capture_output=True, text=True).stdout.split()
    return run


NONE = 0xFFFFFFFF


def test_pages_outside_the_pool_or_the_table_are_none(rules):
    got = list(map(int, rules()))
    want = [3, 6, NONE, NONE, NONE] + [NONE, 0, NONE, NONE, NONE] + [NONE] * 10 + [NONE]
    assert got == want


@pytest.mark.parametrize("position,window,capacity,want", [
    (0, NONE, 4096, (0, 1, 1)), (31, NONE, 4096, (0, 32, 1)), (32, NONE, 4096, (0, 33, 2)),
    (0, 1, 4096, (0, 1, 1)), (500, 1, 4096, (500, 501, 1)), (511, 512, 4096, (0, 512, 16)),
    (512, 512, 4096, (1, 513, 17)), (100, 33, 4096, (68, 101, 2)),
    # past the table: what it holds of the window, and nothing of none
    (5000, NONE, 4096, (0, 4096, 128)), (5000, 1000, 4096, (4001, 4096, 3)),
    (9000, 1000, 4096, (4096, 4096, 1)), (7, NONE, 0, (0, 0, 1)),
    (NONE - 1, NONE, 4096, (0, 4096, 128)), (NONE - 1, 5, 4096, (4096, 4096, 1)),
])
def test_keys_that_a_row_reads(rules, position, window, capacity, want):
    assert tuple(map(int, rules(position, window, capacity))) == want


RAGGED = [1 + 37 * i % 8192 for i in range(61)]


@pytest.mark.parametrize("lengths,window,capacity,head_blocks,at_once", [
    ([1], NONE, 16, 1, 256), ([5004], NONE, 8192, 1, 256), ([0, 0, 0], NONE, 64, 1, 256),
    ([0, 1, 0], NONE, 64, 8, 512), ([1 << 24], NONE, 1 << 24, 1, 512),
    ([1 << 24] * 512, NONE, 1 << 24, 1024, 512), (RAGGED, NONE, 8192, 1, 256),
    (RAGGED, NONE, 8192, 8, 512), (RAGGED, 512, 8192, 64, 512),
    ([100000] + [3] * 511, NONE, 1 << 17, 1, 512), ([100000] + [3] * 127, NONE, 1 << 17, 1, 256),
    ([100000] + [3] * 128, NONE, 1 << 17, 1, 256), ([4000] * 512, NONE, 8192, 64, 512),
    ([129] * 3, NONE, 8192, 85, 512), ([129] * 256, NONE, 8192, 1, 512),
    ([129] * 257, NONE, 8192, 1, 512), (list(range(1, 513)), 700, 512, 3, 512),
])
def test_every_block_in_one_part_within_the_grid(rules, lengths, window, capacity, head_blocks,
                                                 at_once):
    chunk, parts, most, joined, most_joined, covered = map(
        int, rules(window, capacity, head_blocks, at_once, *lengths))
    assert covered == 1
    assert chunk % 4 == 0 or chunk <= 2
    assert parts <= most
    # The workspace holds the parts of rows that have several.
    assert joined <= most_joined <= 3 * at_once
    if any(lengths):
        assert chunk >= 1
