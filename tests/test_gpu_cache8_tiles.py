"""Appends to caches of 8 bits of so many rows and heads that a workgroup takes a tile of
two to four rows (csrc/paged_cache.hip): every number and scale of the pool as defined."""
import numpy as np
import pytest

from _batch import NONE
from test_gpu_cache8_append import Cache

pytestmark = pytest.mark.gpu

AT_ONCE = 1024  # rows' key-value heads that go a workgroup each


def tile_of(rows, kv):
    """(rows of a tile, tiles, whether one was added to make them odd)."""
    tile = min(4, -(-rows * kv // AT_ONCE))
    tiles = -(-rows // tile)
    more = tile > 1 and tiles % 2 == 0
    return tile, tiles + more, more


SIZES = [(300, 4), (300, 8), (350, 8), (410, 5), (507, 5), (507, 8), (510, 6), (512, 8),
         (512, 4), (506, 4)]


def test_the_sizes_are_of_every_tile():
    got = {(tile, more) for tile, _, more in (tile_of(*s) for s in SIZES)}
    assert got == {(t, m) for t in (2, 3, 4) for m in (False, True)}
    # Tiles that are not full, too.
    assert {t for r, k in SIZES for t, n, _ in [tile_of(r, k)] if r % n} == {2, 3, 4}


def prompts(rng, rows, shuffled):
    """Rows of three prompts that begin inside a block, a few of them at no position."""
    each = -(-rows // 3)
    at = [(q, start + i) for q, start in enumerate((0, 5, 40)) for i in range(each)][:rows]
    if shuffled:
        at = [at[i] for i in rng.permutation(rows)]
    positions = np.array([p for _, p in at])
    positions[rng.random(rows) < 0.03] = NONE
    return np.array([q for q, _ in at]), positions


def scattered(rng, rows):
    """Rows anywhere, some of one position, of requests that are not there, past the table."""
    positions = rng.integers(0, 260, rows)
    positions[rng.random(rows) < 0.1] = NONE
    return rng.integers(0, 6, rows), positions


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,kv", SIZES)
def test_tiles_of_rows(device, rows, kv, dim):
    rng = np.random.default_rng(rows + kv + dim)
    cache = Cache(device, rng, [230, 200, 233, 48], kv, dim, 32, wide=1)
    for requests, positions in (prompts(rng, rows, False), prompts(rng, rows, True),
                                scattered(rng, rows), scattered(rng, rows)):
        q, k, v = cache.random(rows, kv, 10.0 ** rng.uniform(-2, 2, rows))
        cache.step(positions, q, k, v, kv, requests)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,kv", [(512, 8), (350, 8), (300, 4)])
def test_a_token_of_each_request(device, rows, kv, dim):
    # A decode step: each row begins a workgroup's block, some at no position.
    rng = np.random.default_rng(dim)
    lengths = [int(n) for n in rng.integers(1, 40, rows)]
    cache = Cache(device, rng, lengths, kv, dim, 16)
    positions = np.array(lengths) - 1
    positions[rng.random(rows) < 0.05] = NONE
    order = rng.permutation(rows)
    for requests in (None, order):
        at = positions if requests is None else positions[order]
        cache.step(at, *cache.random(rows, kv), kv, requests)
