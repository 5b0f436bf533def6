"""Attention over a request's first keys and a window, over caches of every format,
against 64 bits."""
import numpy as np
import pytest

from _batch import BF16, F16, NONE, attention as plain
from _cache8 import I8, any_pool, attention, check

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("fmt", [F16, BF16, I8])


def batch(device, seed, lengths, heads, kv, dim, slots, fmt, wide=0):
    rng = np.random.default_rng(seed)
    paged = any_pool(device, rng, lengths, kv, dim, slots, fmt, wide=wide)
    query = rng.normal(0, 1.5, (len(lengths), heads * dim)).astype(np.float32)
    return paged, query, [n - 1 if n else NONE for n in lengths]


@FORMATS
@pytest.mark.parametrize("wide", [0, 1000])
@pytest.mark.parametrize("sinks", [1, 4, 16, 31, 32, 33, 70, 200])
@pytest.mark.parametrize("window", [1, 17, 32, 100])
def test_sinks_and_windows(device, fmt, wide, sinks, window):
    # First keys and windows apart, in one block, touching, overlapping, past the row.
    lengths = [1, 2, 5, 33, 34, 49, 64, 101, 102, 130, 0, 133, 170, 233, 300, 301, 1000]
    paged, query, positions = batch(device, sinks, lengths, 4, 1, 128, 16, fmt, wide)
    check(device, paged, positions, query, 4, window, 128 ** -0.5, sinks=sinks)


@FORMATS
@pytest.mark.parametrize("dim,heads,kv", [(256, 4, 1), (64, 18, 3), (128, 16, 1), (256, 16, 2)])
def test_heads(device, fmt, dim, heads, kv):
    paged, query, positions = batch(device, dim, [900, 3, 64, 250], heads, kv, dim, 32, fmt)
    check(device, paged, positions, query, heads, 90, dim ** -0.5, sinks=37)
    check(device, paged, positions, query, heads, 600, dim ** -0.5, sinks=5)


@FORMATS
def test_rows_of_several_parts(device, fmt):
    paged, query, positions = batch(device, 4, [30000, 7, 9000, 6000, 0], 4, 1, 128, 64, fmt)
    check(device, paged, positions, query, 4, 5000, 0.09, sinks=3000)
    check(device, paged, positions, query, 4, 8999, 0.09, sinks=1)


@FORMATS
def test_many_rows(device, fmt):
    rng = np.random.default_rng(6)
    lengths = [int(n) for n in rng.integers(0, 400, 300)]
    paged, query, positions = batch(device, 7, lengths, 4, 2, 64, 16, fmt)
    check(device, paged, positions, query, 4, 60, 0.125, sinks=18)


# Rows of a wide table that a window leaves short: a workgroup each.
@FORMATS
@pytest.mark.parametrize("rows,heads,kv,dim,window,sinks", [
    (150, 4, 1, 256, 900, 10), (33, 4, 1, 256, 300, 4), (100, 8, 4, 128, 1900, 33),
    (70, 40, 2, 64, 2500, 1)])
def test_many_rows_of_a_window(device, fmt, rows, heads, kv, dim, window, sinks):
    rng = np.random.default_rng(rows)
    lengths = [int(n) for n in rng.integers(0, 2 * window, rows)]
    paged, query, positions = batch(device, rows, lengths, heads, kv, dim, 32, fmt, wide=200)
    check(device, paged, positions, query, heads, window, dim ** -0.5, sinks=sinks)


@FORMATS
def test_pages_between_that_are_gone_or_hold_anything(device, fmt):
    # What lies between first keys and window is other requests', or nothing: also the
    # rest of a page, a tile and a scale's block that first keys or window end in.
    paged, query, positions = batch(device, 8, [500, 333, 200], 4, 1, 256, 32, fmt)
    sinks, window = 21, 50
    for r, n in enumerate((500, 333, 200)):
        gone = range(sinks, n - window)
        for j in gone:
            page = paged.page(r, j)
            if fmt == I8:
                for codes in paged.codes():
                    codes[page, j % 32] = -128
            else:
                paged.keys[page, j % 32] = paged.values[page, j % 32] = 0x7FC0  # NaN of both
        paged.table[r, 1:(n - window) // 32] = [NONE, paged.pages, 4000000000][r]
    if fmt == I8:
        for scales in paged.scales():
            for r, n in enumerate((500, 333, 200)):
                for j in range(32, (n - window) // 16 * 16, 16):
                    if paged.page(r, j) is not None:
                        scales[paged.page(r, j), j % 32 // 16] = np.nan
    paged.upload()
    check(device, paged, positions, query, 4, window, 1 / 16, sinks=sinks)


@FORMATS
def test_no_sinks_and_all_keys(device, fmt):
    paged, query, positions = batch(device, 9, [500, 33, 0, 200], 4, 1, 256, 16, fmt)
    for window in (70, NONE):
        want = plain(device, paged, positions, query, 4, window, 1 / 16)
        assert np.array_equal(attention(device, paged, positions, query, 4, window, 1 / 16), want)
    # First keys that reach the window are all keys.
    for window, sinks in ((70, 430), (70, NONE), (1, 499), (NONE, 3)):
        got = check(device, paged, positions, query, 4, window, 1 / 16, sinks=sinks)
        assert np.isfinite(got[[0, 1, 3]]).all()


@FORMATS
def test_positions_past_the_table_and_requests_that_are_not_there(device, fmt):
    paged, query, _ = batch(device, 10, [64, 64, 64, 64, 64, 64], 4, 1, 128, 16, fmt)
    positions, requests = [63, 70, 5000, NONE - 1, 30, 30], [0, 1, 2, 3, 9, NONE]
    for window, sinks in ((10, 5), (32, 40), (1, 64), (20, 1000)):
        got = check(device, paged, positions, query, 4, window, 0.1, requests, sinks)
        assert (got[4:] == 0.0).all()


@FORMATS
def test_missing_first_pages(device, fmt):
    paged, query, positions = batch(device, 11, [300, 300, 300], 4, 1, 256, 16, fmt)
    paged.table[0, 0] = NONE
    paged.table[1, 0:19] = NONE
    paged.table[2, 1:] = NONE  # nothing but first keys
    paged.upload()
    got = check(device, paged, positions, query, 4, 40, 1 / 16, sinks=20)
    assert (got[1] == 0.0).all() and (got[2] != 0.0).any()
