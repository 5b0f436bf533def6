"""Caches read back by request and position, from and to every format: the formats'
own rounding of what is held, bit for bit."""
import numpy as np
import pytest

from _batch import BF16, F16, F32, NONE, Paged, of_format, to_format
from _cache8 import I8, Paged8, any_pool, read

pytestmark = pytest.mark.gpu


def expected(paged, requests, positions, fmt, stride, start=7.0):
    """What the op leaves in its rows, keys and values."""
    size = paged.kv * paged.dim
    out = [np.full((len(positions), stride), start) for _ in range(2)]
    for row, p in enumerate(positions):
        if p == NONE:
            continue
        request = row if requests is None else requests[row]
        page, slot = paged.page(request, int(p)), int(p) % paged.slots
        for which in (0, 1):
            if page is None:
                x = np.zeros(size)
            elif isinstance(paged, Paged8):
                x = paged.held(request, [int(p)])[which][0].reshape(-1)
            else:
                x = of_format((paged.keys, paged.values)[which][page, slot], paged.fmt).reshape(-1)
            if fmt == F16:
                x = np.clip(x, -65504, 65504)
            out[which][row, :size] = x
    return [to_format(o, fmt) for o in out]


def check(device, paged, requests, positions, fmt, stride=None):
    stride = stride or paged.kv * paged.dim
    got = read(device, paged, requests, positions, fmt, stride)
    for g, w in zip(got, expected(paged, requests, positions, fmt, stride)):
        assert np.array_equal(g, w, equal_nan=g.dtype == np.float32)


@pytest.mark.parametrize("fmt", [F32, F16, BF16])
@pytest.mark.parametrize("cache", [I8, F16, BF16])
@pytest.mark.parametrize("kv,dim,slots", [(1, 256, 16), (3, 64, 48), (8, 128, 32), (1, 64, 16)])
def test_formats(device, fmt, cache, kv, dim, slots):
    rng = np.random.default_rng(kv + dim)
    lengths = [100, 1, 77, 30]
    paged = any_pool(device, rng, lengths, kv, dim, slots, cache)
    requests = rng.integers(0, 4, 130)
    positions = [int(rng.integers(0, lengths[r])) for r in requests]
    check(device, paged, requests, positions, fmt)
    check(device, paged, requests, positions, fmt, stride=kv * dim + 24)


@pytest.mark.parametrize("cache", [I8, F16])
def test_rows_that_are_none_and_keys_that_are_not_there(device, cache):
    rng = np.random.default_rng(2)
    paged = any_pool(device, rng, [64, 64], 2, 128, 16, cache)
    paged.table[0, 1], paged.table[1, 3] = NONE, paged.pages
    paged.upload()
    requests = [0, 0, 1, 1, 7, 0, NONE, 1, 0]
    positions = [0, 17, 63, NONE, 3, 64, 5, NONE - 1, 63]
    check(device, paged, requests, positions, F32)
    check(device, paged, requests, positions, BF16, stride=2 * 128 + 8)


def test_each_row_its_own_request(device):
    rng = np.random.default_rng(3)
    paged = Paged8(device, rng, [5, 40, 17], 1, 64, 16, pad=16)
    check(device, paged, None, [4, 39, NONE], F32)


@pytest.mark.parametrize("rows,kv,dim", [(70001, 1, 64), (3001, 5, 256), (40, 1024, 64)])
def test_many_rows(device, rows, kv, dim):
    rng = np.random.default_rng(rows)
    paged = Paged8(device, rng, [700], kv, dim, 64) if kv < 1024 else Paged8(
        device, rng, [40], kv, dim, 16)
    positions = np.arange(rows) % paged.lengths[0]
    got = read(device, paged, np.zeros(rows, np.uint32), positions, F16)
    keys, values = paged.rows(0, 0, paged.lengths[0])
    for g, w in zip(got, (keys, values)):
        w = to_format(w.reshape(len(w), -1), F16)
        assert np.array_equal(g, w[positions])


@pytest.mark.parametrize("cache,fmt,kv,dim,rows", [
    (I8, BF16, 2, 128, 40001), (I8, F32, 1, 256, 20003), (F16, F16, 3, 64, 50001),
    (I8, F16, 1024, 64, 150)])
def test_more_than_the_caches_hold(device, cache, fmt, kv, dim, rows):
    # Over 32 MB of outputs, rows of no position and keys of no page among them.
    rng = np.random.default_rng(rows)
    paged = any_pool(device, rng, [90, 300], kv, dim, 16, cache)
    paged.table[1, 2] = NONE
    paged.upload()
    requests = rng.integers(0, 2, rows)
    positions = np.where(requests == 0, rng.integers(0, 90, rows), rng.integers(0, 300, rows))
    positions[rng.random(rows) < 0.1] = NONE
    got = read(device, paged, requests, positions, fmt, stride=kv * dim + 8)
    every = [expected(paged, np.full(n, r), np.arange(n), fmt, kv * dim + 8)
             for r, n in enumerate((90, 300))]
    for which, g in enumerate(got):
        w = np.concatenate([every[0][which], every[1][which], to_format(np.full(
            (1, kv * dim + 8), 7.0), fmt)])
        w = w[np.where(positions == NONE, 390, positions + 90 * requests)]
        assert np.array_equal(g, w, equal_nan=g.dtype == np.float32)


@pytest.mark.parametrize("cache", [I8, BF16])
def test_wide_rows_as_f32_past_the_caches(device, cache):
    test_more_than_the_caches_hold(device, cache, F32, 1024, 64, 75)


def test_the_ends_of_the_range(device):
    rng = np.random.default_rng(4)
    paged = Paged8(device, rng, [48], 1, 64, 16)
    for pool in paged.scales():
        for j, scale in enumerate((2.0 ** 121, 2.0 ** -126, 0.3)):
            pool[paged.page(0, 16 * j)] = scale
    paged.upload()
    for fmt in (F32, F16, BF16):
        check(device, paged, [0] * 48, list(range(48)), fmt)
    paged = Paged(device, rng, [32], 1, 64, 16, BF16, scale=1e30)  # past F16
    check(device, paged, [0] * 32, list(range(32)), F16)
