"""Attention over caches of 8 bits at the ends of F32's range, against 64 bits: queries,
scales and blocks' scales that balance one another."""
import numpy as np
import pytest

from _batch import NONE
from _cache8 import BLOCK, Paged8, check

pytestmark = pytest.mark.gpu


def batch(device, seed, lengths, heads, kv, dim, slots, **more):
    rng = np.random.default_rng(seed)
    paged = Paged8(device, rng, lengths, kv, dim, slots, **more)
    query = rng.normal(0, 1.5, (len(lengths), heads * dim)).astype(np.float32)
    return paged, query, [n - 1 if n else NONE for n in lengths]


# Scores of some units from numbers of which each product but the last is out of F32's
# normal range, or next to it. Tolerances are check()'s: what is held of a query (2^-30 of
# its largest, so these lie above 2^-108, of which 2^-139 is less) and F32's sums.
@pytest.mark.parametrize("dim,heads,kv", [(256, 4, 1), (128, 8, 1), (64, 12, 1)])
@pytest.mark.parametrize("keys", [0, 16384])
@pytest.mark.parametrize("query_size,key_power,scale", [
    (2.0 ** -107, 120, 1.3 * 2.0 ** -19), (2.0 ** -107, 117, 2.0 ** -14 / 3),
    (2.0 ** -104, 119, -1.7 * 2.0 ** -21), (2.0 ** -100, 100, 1.1 * 2.0 ** -6),
    (2.0 ** -60, 119, 1.9 * 2.0 ** -65), (2.0 ** -30, 120, 0.9 * 2.0 ** -96),
    (2.0 ** 100, -126, 1.3 * 2.0 ** 11), (2.0 ** 118, -140, 1.3 * 2.0 ** 11),
    (2.0 ** 122, -5, 1.5 * 2.0 ** -123), (2.0 ** 122, -1, 1.5 * 2.0 ** -126)])
def test_numbers_that_balance(device, dim, heads, kv, keys, query_size, key_power, scale):
    paged, query, positions = batch(device, 31, [150, 33, 700], heads, kv, dim, 16,
                                    wide=keys // 16)
    keys_scales, _ = paged.scales()
    keys_scales[:] = np.ldexp(np.float32(1), key_power) * np.where(np.isnan(keys_scales), np.nan, 1)
    paged.upload()
    query = (query * np.float32(query_size)).astype(np.float32)
    check(device, paged, positions, query, heads, NONE, float(np.float32(scale)))


# A block whose numbers are all 0 holds no value, however large its scale, and so does one
# of whose keys those that are not 0 lie outside the window: the others' outputs keep
# check()'s bound, of the largest value that is read.
@pytest.mark.parametrize("dim,heads,kv", [(256, 4, 1), (128, 8, 1), (128, 6, 2), (64, 12, 1)])
@pytest.mark.parametrize("keys", [0, 16384])
@pytest.mark.parametrize("power", [18, 30, 60, 121, 127])
def test_scales_of_blocks_of_zeros(device, dim, heads, kv, keys, power):
    lengths = [150, 33, 700, 16, 4000]
    paged, query, positions = batch(device, 32, lengths, heads, kv, dim, 16, wide=keys // 16)
    codes, scales = paged.codes()[1], paged.scales()[1]
    rng = np.random.default_rng(33)
    for r, n in enumerate(lengths):
        for j in range(0, n, BLOCK):
            if r == 3 or rng.random() < 0.4:
                page, head = paged.page(r, j), rng.integers(0, kv)
                codes[page, :, head] = 0
                scales[page, 0, head] = 2.0 ** power
    paged.upload()
    for window, sinks in ((NONE, 0), (100, 0), (70, 20)):
        check(device, paged, positions, query, heads, window, dim ** -0.5, sinks=sinks)


@pytest.mark.parametrize("dim,heads,kv", [(256, 4, 1), (128, 8, 1), (64, 12, 1)])
@pytest.mark.parametrize("keys", [0, 16384])
def test_scales_of_keys_outside_the_window(device, dim, heads, kv, keys):
    # The window's first key is the second of its block; what gave the block its scale was
    # the first, as an append writes it: the others are 0 beside it.
    lengths = [57 + BLOCK, 200, 713]
    paged, query, positions = batch(device, 34, lengths, heads, kv, dim, 16, wide=keys // 16)
    window = 40
    for r, n in enumerate(lengths):
        first = n - window
        page = paged.page(r, first)
        codes, scales = paged.codes()[1], paged.scales()[1]
        codes[page, :first % BLOCK + 1] = 127
        codes[page, first % BLOCK:] = 0
        scales[page] = 2.0 ** 40
    paged.upload()
    check(device, paged, positions, query, heads, window, dim ** -0.5)
    check(device, paged, positions, query, heads, window, dim ** -0.5, sinks=3)


def test_values_of_zeros_alone(device):
    paged, query, positions = batch(device, 35, [150, 700], 4, 1, 256, 16)
    paged.codes()[1][:] = 0
    paged.scales()[1][:] = 2.0 ** 100
    paged.upload()
    got = check(device, paged, positions, query, 4, NONE, 1 / 16)
    assert (got == 0.0).all()
