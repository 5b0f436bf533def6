"""Attention over caches of 8 bits against 64 bits, over what the pages hold: head
layouts, lengths, pages, strides, scales of any size."""
import threading

import numpy as np
import pytest

import frizzle_amd as fz
from _batch import NONE
from _cache8 import BLOCK, Paged8, attention, check, exact

pytestmark = pytest.mark.gpu


def batch(device, seed, lengths, heads, kv, dim, slots, **more):
    rng = np.random.default_rng(seed)
    paged = Paged8(device, rng, lengths, kv, dim, slots, **more)
    query = rng.normal(0, 1.5, (len(lengths), heads * dim)).astype(np.float32)
    return paged, query, [n - 1 if n else NONE for n in lengths]


TABLES = pytest.mark.parametrize("keys", [0, 16384])


@TABLES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (5, 1), (8, 1), (9, 1), (16, 1), (17, 1),
                                      (40, 1), (6, 2), (8, 8), (24, 3)])
def test_heads(device, dim, heads, kv, keys):
    paged, query, positions = batch(device, heads + dim, [70, 1, 0, 33, 150], heads, kv, dim, 16,
                                    wide=keys // 16)
    check(device, paged, positions, query, heads, NONE, dim ** -0.5)


@TABLES
@pytest.mark.parametrize("slots", [16, 48, 64, 256])
@pytest.mark.parametrize("window", [1, 15, 33, 512, NONE])
def test_lengths_and_windows(device, slots, window, keys):
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 100, 127, 129, 300, 513, 1000]
    paged, query, positions = batch(device, slots, lengths, 4, 1, 256, slots, wide=keys // slots)
    check(device, paged, positions, query, 4, window, 1 / 16)


@pytest.mark.parametrize("lengths,heads,kv,dim,slots", [
    ([20000], 4, 1, 256, 64), ([9000, 0, 5, 129, 4000], 4, 1, 256, 16),
    ([30000] + [3] * 100, 5, 1, 128, 32), ([2000] + [10] * 200, 12, 4, 64, 16),
    ([70000], 2, 2, 64, 256), ([200, 300] * 70, 18, 1, 64, 16), ([5000, 700], 16, 1, 256, 16)])
def test_rows_of_several_parts(device, lengths, heads, kv, dim, slots):
    paged, query, positions = batch(device, sum(lengths), lengths, heads, kv, dim, slots)
    check(device, paged, positions, query, heads, NONE, dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 6, 12, 17])
@pytest.mark.parametrize("window", [40, NONE])
def test_many_short_rows(device, dim, group, window):
    rng = np.random.default_rng(dim + group)
    lengths = [int(n) for n in rng.integers(0, 100, 270)]
    lengths[100] = 4097 if dim == 128 and window == NONE else 1
    paged, query, positions = batch(device, group, lengths, 4 * group, 4, dim, 16)
    check(device, paged, positions, query, 4 * group, window, dim ** -0.5)


# As many units as waves run at once, and fewer of fewer blocks: a wave each.
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,group,kv,most", [(512, 1, 8, 90), (500, 6, 8, 40), (512, 12, 8, 33),
                                                (300, 3, 4, 31), (400, 2, 1, 32)])
def test_rows_of_a_wave_each(device, dim, rows, group, kv, most):
    rng = np.random.default_rng(dim + rows)
    lengths = [int(n) for n in rng.integers(0, most + 1, rows)]
    paged, query, positions = batch(device, group, lengths, kv * group, kv, dim, 16)
    check(device, paged, positions, query, kv * group, NONE, dim ** -0.5)


@TABLES
def test_rows_of_a_request_in_any_order_and_requests_that_are_not_there(device, keys):
    rng = np.random.default_rng(9)
    paged, _, _ = batch(device, 10, [700, 0, 333, 64], 4, 1, 256, 16, wide=keys // 16)
    requests = [2, 0, 3, 0, 2, 0, 9, 1, NONE]
    positions = [332, 699, 63, 5, 100, NONE, 20, 10, 4]
    query = rng.normal(0, 1, (9, 1024)).astype(np.float32)
    got = check(device, paged, positions, query, 4, 400, 1 / 16, requests)
    assert (got[6:] == 0.0).all()


@TABLES
def test_pages_that_are_not_there(device, keys):
    paged, query, positions = batch(device, 11, [400, 400, 400, 400, 90], 4, 1, 256, 16,
                                    wide=keys // 16)
    paged.table[0, 3] = NONE
    paged.table[0, 24] = paged.pages
    paged.table[1, :] = 4000000000
    paged.table[2, 0:21] = NONE
    paged.table[3, 10:] = NONE
    paged.table[4, 0::2] = NONE
    paged.upload()
    got = check(device, paged, positions, query, 4, NONE, 1 / 16)
    assert (got[1] == 0.0).all()
    check(device, paged, positions, query, 4, 70, 1 / 16)


def test_strides_and_positions_past_the_table(device):
    paged, query, _ = batch(device, 13, [200, 64, 77, 16], 12, 3, 128, 16, pad=48)
    check(device, paged, [199, 5000, 76, NONE - 1], query, 12, NONE, 128 ** -0.5, width=1600,
          out_width=1540)
    check(device, paged, [199, 230, 76, NONE - 1], query, 12, 60, 128 ** -0.5)


@pytest.mark.parametrize("near", [0, 1])
def test_scales_that_rise_fall_and_vanish(device, near):
    # By 2^40 and more between blocks, so that a wave's outputs change their unit;
    # negative ones, zeros, and no powers of two.
    paged, query, positions = batch(device, 14, [640, 200, 40], 4, 1, 256, 16)
    rng = np.random.default_rng(14)
    keys, values = paged.scales()
    for r, n in enumerate((640, 200, 40)):
        for j in range(0, n, BLOCK):
            at = paged.page(r, j), j % 16 // BLOCK, 0
            values[at] = rng.choice([-1.0, 1.0]) * rng.uniform(1, 2) * (
                2.0 ** rng.integers(-3, 3) if near else 2.0 ** (j // BLOCK - 20))
            keys[at] *= rng.choice([-1.0, 1.0, 0.0]) * rng.uniform(0.5, 1)
    values[paged.page(1, 0)] = 0.0
    paged.upload()
    check(device, paged, positions, query, 4, NONE, 1 / 16)
    check(device, paged, positions, query, 4, 100, 1 / 16)


@TABLES
@pytest.mark.parametrize("query_size,key_power,value_power", [
    (1e4, -20, 0), (1e-30, 60, 0), (3e6, -30, 0), (0.0, -5, 0), (1.0, -5, 120), (1.0, -5, -126),
    (1e30, -110, 0), (1e-20, 60, 60), (30.0, -5, -5), (1e-33, 105, -5)])
def test_queries_scales_and_values_of_any_size(device, query_size, key_power, value_power, keys):
    paged, query, positions = batch(device, 15, [150, 33, 1], 4, 1, 256, 16, wide=keys // 16)
    for pool, power in zip(paged.scales(), (key_power, value_power)):
        pool[:] = np.ldexp(np.float32(1), power) * np.where(np.isnan(pool), np.nan, 1)
    paged.upload()
    query = (query * query_size).astype(np.float32)
    size = query_size * 2.0 ** key_power * 30
    check(device, paged, positions, query, 4, NONE, 1 / (16 * max(1.0, min(size, 256))))


def test_a_head_whose_queries_differ_in_size(device):
    # Whole numbers of the largest: what is 2^-26 of it has four bits, as the bound says.
    paged, query, positions = batch(device, 16, [150, 33, 1], 4, 1, 256, 16)
    query[:, ::7] *= 2.0 ** -26
    query[:, 256] = 100.0
    check(device, paged, positions, query, 4, NONE, 1 / 16)
    check(device, paged, positions, query, 4, NONE, -0.3)
    check(device, paged, positions, query, 4, NONE, 0.0)


def test_rising_scores(device):
    paged, query, positions = batch(device, 17, [640], 4, 1, 256, 16)
    query[:] = 1.0
    codes = paged.codes()[0]
    for j in range(640):
        codes[paged.page(0, j), j % 16, 0] = j // 6
    paged.scales()[0][:] = 1 / 16
    paged.upload()
    check(device, paged, positions, query, 4, NONE, 1 / 16)


@pytest.mark.parametrize("length", [200, 3000])
def test_a_query_that_is_no_number_stays_in_its_row_and_head(device, length):
    paged, query, positions = batch(device, 18, [100, 100, length], 4, 1, 256, 16)
    bad = query.copy()
    bad[1, 300] = np.nan
    bad[2, 1000] = np.inf
    got = attention(device, paged, positions, bad, 4, NONE, 1 / 16)
    want, far = exact(paged, positions, query, 4, NONE, 1 / 16)
    for row, sound in ((0, [0, 1, 2, 3]), (1, [0, 2, 3]), (2, [0, 1, 2])):
        for h in range(4):
            at = slice(256 * h, 256 * h + 256)
            if h in sound:
                assert (abs(got[row, at] - want[row][at]) <= far[row][at]).all()
            else:
                assert np.isnan(got[row, at]).all()


# As of 16 bits: 4.1e-7 of the scores, 2.7e-7 of the sums.
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 256), (8, 1, 128), (16, 1, 256), (6, 3, 64)])
@pytest.mark.parametrize("lengths,wide", [([300, 77, 16], 0), ([2000, 700, 1300], 0),
                                          ([300, 77, 16], 500)])
def test_in_the_mean(device, heads, kv, dim, lengths, wide):
    paged, query, positions = batch(device, heads + dim, lengths, heads, kv, dim, 32, wide=wide)
    check(device, paged, positions, query, heads, NONE, dim ** -0.5, near=8e-7)


def test_the_same_bits_every_time_and_from_threads(device):
    sets = [batch(device, 19, [5000, 20, 0, 900], 4, 1, 256, 64),
            batch(device, 20, [64, 7000], 6, 2, 128, 16)]
    args = [(sets[0][0], sets[0][2], sets[0][1], 4, NONE, 1 / 16),
            (sets[1][0], sets[1][2], sets[1][1], 6, 300, 0.1)]
    want = [attention(device, *a) for a in args]
    bad = []

    def work(i):
        for _ in range(20):
            if not np.array_equal(attention(device, *args[i]), want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i % 2,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_the_most_rows_and_heads(device):
    rng = np.random.default_rng(5)
    lengths = [int(n) for n in rng.integers(0, 90, 512)]
    paged, query, positions = batch(device, 6, lengths, 4, 2, 64, 16)
    check(device, paged, positions, query, 4, 64, 0.125)
    paged, query, positions = batch(device, 7, [33, 0, 150], 1024, 512, 64, 16)
    check(device, paged, positions, query, 1024, NONE, 0.125)


def test_a_pool_past_32_bits(device):
    # Pages 2^31 numbers and 2^29 scales apart: the last begin at 2^32 and 2^32 bytes.
    from frizzle_amd import _lib
    rng = np.random.default_rng(22)
    dim, slots, pages, stride, scale_stride = 256, 16, 3, 1 << 31, 1 << 29
    lib = fz.load()
    big = fz.runtime.DeviceArray(device, stride * (pages - 1) + 2 * slots * dim, np.uint8, (1,))
    far = fz.runtime.DeviceArray(device, 4 * (scale_stride * (pages - 1) + 2), np.uint8, (1,))
    codes = rng.integers(-127, 128, (pages, 2, slots, dim)).astype(np.int8)
    scales = np.exp2(rng.integers(-7, -4, (pages, 2))).astype(np.float32)
    for p in range(pages):
        _lib.check(lib.frz_write(device.handle, big.ptr + stride * p,
                                 np.ascontiguousarray(codes[p]).ctypes.data, codes[p].nbytes))
        _lib.check(lib.frz_write(device.handle, far.ptr + 4 * scale_stride * p,
                                 np.ascontiguousarray(scales[p]).ctypes.data, scales[p].nbytes))
    table = device.array(np.array([[2, 0, 1]], np.uint32))
    positions = device.array(np.array([44], np.uint32))
    query = rng.normal(0, 1.5, (1, 1024)).astype(np.float32)
    dq, do = device.array(query), device.empty((1, 1024), np.float32)
    c = fz.Pages(big.ptr, big.ptr + slots * dim, 24, 1, dim, slots, pages, stride, table.ptr, 1, 3,
                 far.ptr, far.ptr + 4, scale_stride)
    _lib.check(lib.frz_op_attention_paged(device.handle, c, None, positions.ptr, dq.ptr, 1024,
                                          do.ptr, 1024, 4, NONE, 1 / 16, 1))
    device.sync()
    got = do.numpy()[0].reshape(4, dim)
    big.free()
    far.free()
    order = [2, 0, 1]
    k, v = ((codes[order, i].astype(np.float64) * scales[order, i][:, None, None])
            .reshape(-1, dim)[:45] for i in (0, 1))
    s = query.astype(np.float64).reshape(4, dim) @ k.T / 16
    w = np.exp(s - s.max(1, keepdims=True))
    want = w / w.sum(1, keepdims=True) @ v
    assert np.linalg.norm(got - want) <= 5e-6 * np.linalg.norm(want)
