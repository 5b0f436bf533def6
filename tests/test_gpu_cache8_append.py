"""Appends to caches of 8 bits: every number and scale of the pool, those not written
among them, as defined from the keys that frz_op_rope_paged gives in F32, and the keys
themselves in 64 bits."""
import numpy as np
import pytest

import frizzle_amd as fz
from _batch import F16, NONE, Paged, rope, rope_exact
from _cache8 import BLOCK, Paged8, append

pytestmark = pytest.mark.gpu


def gains(rng, dim):
    return [(1 + 0.1 * rng.normal(0, 1, dim)).astype(np.float32) for _ in range(2)]


class Cache:
    """A pool of 8 bits and one of 16 whose op turns keys as queries, in F32."""

    def __init__(self, device, rng, lengths, kv, dim, slots, **more):
        self.device, self.rng = device, rng
        self.paged = Paged8(device, rng, lengths, kv, dim, slots, **more)
        self.gains, self.turns = gains(rng, dim), fz.rope_turns(1e4, dim)

    def turned(self, positions, key, requests):
        """The keys that the op quantises: the same rows turned as queries."""
        kv, dim = self.paged.kv, self.paged.dim
        other = Paged(self.device, self.rng, [0] * len(self.paged.table), kv, dim, 16, F16)
        g = self.gains[1]
        out = rope(self.device, other, positions, self.turns, (g, g), key, key, key, kv, requests)
        return out.reshape(-1, kv, dim)

    def step(self, positions, query, key, value, heads, requests=None, **more):
        """One step on the device and by definition; all of both pools compared."""
        kv, dim = self.paged.kv, self.paged.dim
        got = rope(self.device, self.paged, positions, self.turns, self.gains, query, key, value,
                   heads, requests, **more)
        append(self.paged, positions, self.turned(positions, key, requests),
               value.reshape(-1, kv, dim), requests)
        want = self.paged.pools + self.paged.scale_pools
        for name, g, w in zip(("keys", "values", "key scales", "value scales"),
                              self.paged.download(), want):
            assert np.array_equal(g, w, equal_nan=g.dtype == np.float32), name
        return got

    def random(self, rows, heads, sizes=1.0):
        kv, dim = self.paged.kv, self.paged.dim
        sizes = np.broadcast_to(np.asarray(sizes, np.float32), (rows,))[:, None]
        return [(self.rng.normal(0, 1.5, (rows, n * dim)) * sizes).astype(np.float32)
                for n in (heads, kv, kv)]


SHAPES = [(4, 1, 256, 16), (4, 1, 256, 64), (6, 2, 128, 48), (32, 8, 128, 16), (5, 5, 64, 32),
          (16, 1, 64, 16)]


@pytest.mark.parametrize("heads,kv,dim,slots", SHAPES)
def test_a_conversation(device, heads, kv, dim, slots):
    # A prompt in ragged steps, then single tokens, of growing and shrinking sizes.
    rng = np.random.default_rng(heads + dim)
    cache = Cache(device, rng, [120, 7], kv, dim, slots)
    at = 0
    for n, size in ((3, 1.0), (40, 0.3), (1, 5.0), (1, 0.01), (2, 100.0), (1, 90.0), (17, 1.0),
                    (1, 1e-3), (1, 1e4)):
        positions = list(range(at, at + n)) + [NONE]
        q, k, v = cache.random(n + 1, heads, size)
        cache.step(positions, q, k, v, heads, [0] * n + [1])
        at += n


@pytest.mark.parametrize("heads,kv,dim,slots", SHAPES)
def test_queries_are_frz_op_rope_pageds(device, heads, kv, dim, slots):
    rng = np.random.default_rng(3)
    cache = Cache(device, rng, [50, 31, 200, 1], kv, dim, slots, pad=32)
    q, k, v = cache.random(4, heads)
    positions = [49, NONE, 199, 0]
    other = Paged(device, rng, [50, 31, 200, 1], kv, dim, slots, F16)
    for more in (dict(), dict(in_place=True), dict(out_width=heads * dim + 8, extra=4)):
        got = cache.step(positions, q, k, v, heads, **more)
        want = rope(device, other, positions, cache.turns, cache.gains, q, k, v, heads, **more)
        assert np.array_equal(got[:, :heads * dim], want[:, :heads * dim])


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 300, 512])
def test_rows_in_any_order_the_last_of_a_position_kept(device, rows):
    rng = np.random.default_rng(rows)
    cache = Cache(device, rng, [64, 200, 33, 48], 2, 64, 32, wide=1)
    requests = rng.integers(0, 6, rows)  # two are past the table
    positions = rng.integers(0, 260, rows)
    positions[rng.random(rows) < 0.1] = NONE
    q, k, v = cache.random(rows, 4, 10.0 ** rng.uniform(-2, 2, rows))
    for _ in range(2):
        cache.step(positions, q, k, v, 4, requests)


def test_a_block_begun_anew(device):
    # A page that another request left: large numbers, and scales that are none.
    rng = np.random.default_rng(8)
    cache = Cache(device, rng, [64, 64, 64, 64, 64, 64], 1, 128, 64, powers=(20, 20))
    for request, scale in enumerate((np.nan, 0.0, -1.0, np.inf, -np.inf)):
        for pool in cache.paged.scales():
            pool[cache.paged.page(request, 0)] = scale
    cache.paged.upload()
    q, k, v = cache.random(12, 2)
    # From a first slot, and from one further on.
    cache.step([16, 35] * 6, q, k, v, 2, [r for r in range(6) for _ in range(2)])
    scale = cache.paged.scales()[1]
    assert scale[cache.paged.page(5, 0), 2, 0] == 2.0 ** 20  # held
    assert scale[cache.paged.page(5, 0), 1, 0] < 1
    for request in range(6):
        assert (cache.paged.codes()[0][cache.paged.page(request, 0), 17:32] == 0).all()


def test_scales_that_are_no_powers_of_two(device):
    rng = np.random.default_rng(9)
    cache = Cache(device, rng, [64], 2, 64, 64)
    for pool in cache.paged.scales():
        pool[cache.paged.page(0, 0)] = rng.uniform(0.001, 0.1, pool.shape[1:])
    cache.paged.upload()
    for p in (5, 22, 40, 41, 63):
        cache.step([p], *cache.random(1, 2), 2)


@pytest.mark.parametrize("values", [
    [0.0], [-0.0, 1e-45], [1e-38, 1e-40], [127.0, 63.5, -0.5], [127.00001, 1.5, 2.5],
    [254.0, -254.00003, 1.0], [3.4028235e38, 1.0], [np.inf, 1.0, -np.inf], [np.nan, 2.0],
    [np.nan], [1e38, np.nan, -1e37], [126.5, 0.5, 1.5], [2.0 ** -126 * 127, 2.0 ** -149]])
@pytest.mark.parametrize("first", [0, 3])
def test_values_at_the_borders(device, values, first):
    rng = np.random.default_rng(10)
    cache = Cache(device, rng, [32], 1, 64, 16, powers=(-149, -140))
    q, k, v = cache.random(2, 1)
    v[:] = np.resize(np.asarray(values, np.float32), v.shape)
    v[1] = 0
    cache.step([first, first + 1], q, k, v, 1, [0, 0])


def test_keys_that_are_no_number(device):
    rng = np.random.default_rng(11)
    cache = Cache(device, rng, [32, 32], 2, 128, 32)
    q, k, v = cache.random(3, 2)
    k[0, 5], k[1, 200] = np.nan, np.inf  # NaN all through their heads, 0 in the cache
    cache.step([0, 1, 17], q, k, v, 2, [0, 0, 1])


def test_pages_and_positions_that_are_not_there(device):
    rng = np.random.default_rng(12)
    cache = Cache(device, rng, [64, 64, 64], 1, 256, 16)
    cache.paged.table[0, 1] = NONE
    cache.paged.table[1, 2] = cache.paged.pages
    cache.paged.table[2, 3] = 4000000000
    cache.paged.upload()
    positions = [15, 16, 33, 47, 63, 64, 1 << 24, NONE - 1]
    requests = [0, 0, 1, 1, 2, 2, 0, 0]
    cache.step(positions, *cache.random(8, 4), 4, requests)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_numbers_are_near_the_keys(device, dim):
    # Half a scale of this step's rows, less than one of those before; keys of F32's
    # arithmetic are off by 2^-18 of the largest at most besides.
    rng = np.random.default_rng(13)
    cache = Cache(device, rng, [32], 1, dim, 16)
    far = {}
    for p in range(32):
        q, k, v = cache.random(1, 1, 1.0 + 0.3 * (p % BLOCK))
        cache.step([p], q, k, v, 1)
        x, size = rope_exact(k, cache.gains[1], cache.turns, p)
        far[p] = (x[0], v[0].astype(np.float64), 2.0 ** -18 * size.max())
        for j, (key, value, slack) in far.items():
            if j // BLOCK != p // BLOCK:
                continue
            got = [g[0][0] for g in cache.paged.held(0, [j])]
            scales = [s[cache.paged.page(0, j), 0, 0] for s in cache.paged.scales()]
            part = 0.5 if j == p else 1.0
            assert (abs(got[0] - key) <= part * scales[0] + slack).all()
            assert (abs(got[1] - value) <= part * scales[1]).all()


def test_the_most_heads(device):
    rng = np.random.default_rng(14)
    cache = Cache(device, rng, [40, 33], 1024, 64, 16)
    cache.step([39, 32], *cache.random(2, 1024), 1024)


def test_pools_past_32_bits(device):
    # The last of pages 2^31 numbers and 2^30 scales apart.
    rng = np.random.default_rng(15)
    from frizzle_amd import _lib
    dim, pages, stride, scale_stride = 128, 3, 1 << 31, 1 << 30
    big = fz.runtime.DeviceArray(device, stride * (pages - 1) + 32 * dim, np.uint8, (1,))
    scales = fz.runtime.DeviceArray(device, 4 * (scale_stride * (pages - 1) + 4), np.uint8, (1,))
    table, positions = device.array(np.array([[2]], np.uint32)), device.array(
        np.array([0], np.uint32))
    g, turns = device.array(np.ones(dim, np.float32)), device.array(fz.rope_turns(1e4, dim))
    x = rng.normal(0, 1, (1, dim)).astype(np.float32)
    dx, do = device.array(x), device.array(np.zeros((1, dim), np.float32))
    c = fz.Pages(big.ptr, big.ptr + 16 * dim, 24, 1, dim, 16, pages, stride, table.ptr, 1, 1,
                 scales.ptr, scales.ptr + 8, scale_stride)
    _lib.check(fz.load().frz_op_rope_paged(device.handle, c, None, positions.ptr, turns.ptr, g.ptr,
                                           g.ptr, dx.ptr, dx.ptr, dx.ptr, dim, dim, do.ptr, dim, 1,
                                           1e-6, 1))
    out = [device.array(np.zeros((1, dim), np.float32)) for _ in range(2)]
    _lib.check(fz.load().frz_op_read_paged(device.handle, c, None, positions.ptr, 0, out[0].ptr,
                                           out[1].ptr, dim, 1))
    device.sync()
    got = [o.numpy()[0] for o in out]
    big.free()
    scales.free()
    assert (abs(got[1] - x[0]) <= 2.0 ** -6 * abs(x).max()).all() and abs(got[1]).max() > 1
    assert (abs(got[0] - do.numpy()[0]) <= 2.0 ** -6 * abs(got[0]).max()).all()
