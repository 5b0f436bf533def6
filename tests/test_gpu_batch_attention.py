"""Attention of a batch's rows over caches in pages (frz_op_attention_paged)
against its values in 64 bits."""
import threading

import numpy as np
import pytest

from _batch import (BF16, F16, NONE, Paged, attention, attention_exact, check_attention, of_format,
                    to_format)

pytestmark = pytest.mark.gpu

EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 500]


def batch(device, seed, lengths, heads, kv, dim, slots, fmt, **more):
    rng = np.random.default_rng(seed)
    paged = Paged(device, rng, lengths, kv, dim, slots, fmt, **more)
    query = rng.normal(0, 1.5, (len(lengths), heads * dim)).astype(np.float32)
    positions = [n - 1 if n else NONE for n in lengths]
    return paged, query, positions


# Tables of no more pages than the rows have, whose rows go uncut, a workgroup
# each; and of LONG keys, which could hold rows that are cut into parts.
LONG = 20000
TABLES = pytest.mark.parametrize("keys", [0, LONG])


# Every compiled shape, groups that leave columns free and such that take two
# head blocks.
@pytest.mark.parametrize("heads,kv,dim", [
    (4, 1, 256), (1, 1, 64), (3, 3, 128), (6, 2, 128), (8, 1, 256), (9, 1, 64), (10, 2, 256),
    (16, 1, 128), (32, 2, 256), (20, 1, 64), (66, 2, 128), (40, 8, 64), (17, 1, 256)])
@pytest.mark.parametrize("fmt", [F16, BF16])
@TABLES
def test_head_layouts(device, heads, kv, dim, fmt, keys):
    lengths = [1, 40, 0, 130, 17, 300]
    paged, query, positions = batch(device, heads + dim, lengths, heads, kv, dim, 32, fmt,
                                    wide=keys // 32)
    check_attention(device, paged, positions, query, heads, NONE, dim ** -0.5)


@pytest.mark.parametrize("slots", [16, 48, 64, 1024])
@pytest.mark.parametrize("window", [1, 31, 33, 100, 512, NONE])
@TABLES
def test_lengths_windows_and_pages(device, slots, window, keys):
    paged, query, positions = batch(device, slots + window % 1000, EDGES, 4, 1, 256, slots, F16,
                                    wide=keys // slots)
    check_attention(device, paged, positions, query, 4, window, 1 / 16)


@pytest.mark.parametrize("dim,fmt", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("window", [40, NONE])
@TABLES
def test_lengths_of_other_widths(device, dim, fmt, window, keys):
    paged, query, positions = batch(device, dim + window % 999, EDGES, 6, 2, dim, 16, fmt,
                                    wide=keys // 16)
    check_attention(device, paged, positions, query, 6, window, dim ** -0.5)


# One long row among short ones: parts joined by the second launch, at its
# widths and at more parts than its threads.
@pytest.mark.parametrize("lengths,heads,kv,dim,slots,fmt", [
    ([20000], 4, 1, 256, 64, F16), ([9000, 0, 5, 129, 4000], 4, 1, 256, 16, F16),
    ([30000] + [3] * 100, 5, 1, 128, 32, BF16), ([2000] + [10] * 200, 12, 4, 64, 16, F16),
    ([70000], 2, 2, 64, 256, F16), ([200, 300] * 70, 18, 1, 64, 16, BF16)])
def test_rows_of_several_parts(device, lengths, heads, kv, dim, slots, fmt):
    paged, query, positions = batch(device, sum(lengths), lengths, heads, kv, dim, slots, fmt)
    check_attention(device, paged, positions, query, heads, NONE, dim ** -0.5)


@pytest.mark.parametrize("heads,kv", [(1024, 1024), (1024, 2), (1024, 1), (1008, 63)])
@TABLES
def test_the_most_heads(device, heads, kv, keys):
    paged, query, positions = batch(device, heads + kv, [33, 0, 150, 1, 18], heads, kv, 64, 16, F16,
                                    wide=keys // 16)
    check_attention(device, paged, positions, query, heads, 100, 0.125)


# More rows and key-value heads than workgroups run at once: a wave each.
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group,fmt", [(1, F16), (6, F16), (12, F16), (17, F16), (4, BF16),
                                       (7, BF16), (16, BF16)])
@pytest.mark.parametrize("window", [40, NONE])
def test_many_short_rows(device, dim, group, fmt, window):
    rng = np.random.default_rng(dim + group)
    lengths = [int(n) for n in rng.integers(0, 100, 270)]
    paged, query, positions = batch(device, group, lengths, 4 * group, 4, dim, 16, fmt)
    check_attention(device, paged, positions, query, 4 * group, window, dim ** -0.5)


# The same over long tables: more units than parts run at once, several parts.
@pytest.mark.parametrize("dim,fmt,window", [(256, F16, NONE), (128, BF16, 1100), (64, F16, NONE)])
def test_many_rows_some_long(device, dim, fmt, window):
    rng = np.random.default_rng(dim)
    lengths = [int(n) for n in rng.integers(0, 60, 270)]
    lengths[7], lengths[100], lengths[269] = 9000, 4097, 1500
    paged, query, positions = batch(device, dim, lengths, 4, 4, dim, 16, fmt)
    check_attention(device, paged, positions, query, 4, window, dim ** -0.5)


def test_the_most_rows(device):
    rng = np.random.default_rng(5)
    lengths = [int(n) for n in rng.integers(0, 90, 512)]
    paged, query, positions = batch(device, 6, lengths, 4, 2, 64, 16, F16)
    check_attention(device, paged, positions, query, 4, 64, 0.125)


def test_no_row_after_rows_of_several_parts(device):
    # The second launch must not join what an earlier call left.
    paged, query, positions = batch(device, 8, [6000, 5000], 4, 1, 256, 64, F16)
    check_attention(device, paged, positions, query, 4, NONE, 1 / 16)
    got = attention(device, paged, [NONE, NONE], query, 4, NONE, 1 / 16)
    assert (got == 7.0).all()


@TABLES
def test_several_rows_of_a_request_in_any_order(device, keys):
    rng = np.random.default_rng(9)
    paged, _, _ = batch(device, 10, [700, 0, 333, 64], 4, 1, 256, 16, F16, wide=keys // 16)
    requests = [2, 0, 3, 0, 2, 0, 9, 1, NONE]
    positions = [332, 699, 63, 5, 100, NONE, 20, 10, 4]
    query = rng.normal(0, 1, (9, 1024)).astype(np.float32)
    # Requests past the table and one without pages read nothing.
    got = check_attention(device, paged, positions, query, 4, 400, 1 / 16, requests)
    assert (got[6:] == 0.0).all()


@TABLES
def test_pages_that_are_not_there(device, keys):
    paged, query, positions = batch(device, 11, [400, 400, 400, 400, 90], 4, 1, 256, 16, F16,
                                    wide=keys // 16)
    paged.table[0, 3] = NONE           # a hole
    paged.table[0, 24] = paged.pages   # the last page, and so the row's own key
    paged.table[1, :] = 4000000000     # none at all
    paged.table[2, 0:21] = NONE        # all but the last few
    paged.table[3, 10:] = NONE         # the end
    paged.table[4, 0::2] = NONE        # half of each block
    paged.upload()
    got = check_attention(device, paged, positions, query, 4, NONE, 1 / 16)
    assert (got[1] == 0.0).all()
    check_attention(device, paged, positions, query, 4, 70, 1 / 16)


def test_positions_past_the_table(device):
    paged, query, _ = batch(device, 12, [64, 64, 64, 64], 4, 1, 256, 16, F16)
    positions = [63, 70, 5000, NONE - 1]
    check_attention(device, paged, positions, query, 4, 32, 1 / 16)
    check_attention(device, paged, positions, query, 4, NONE, 1 / 16)


@pytest.mark.parametrize("fmt", [F16, BF16])
def test_strides_and_interleaved_pools(device, fmt):
    lengths = [200, 0, 77, 16]
    for more in (dict(pad=8), dict(interleaved=True), dict(interleaved=True, pad=64, wide=3)):
        paged, query, positions = batch(device, 13, lengths, 12, 3, 128, 16, fmt, **more)
        check_attention(device, paged, positions, query, 12, NONE, 128 ** -0.5, width=1600,
                        out_width=1540)


def test_shared_prefix_pages(device):
    paged, query, positions = batch(device, 14, [300, 300, 300], 4, 1, 256, 64, F16)
    paged.table[1, :4] = paged.table[0, :4]
    paged.table[2, :2] = paged.table[0, :2]
    paged.upload()
    check_attention(device, paged, positions, query, 4, NONE, 1 / 16)


@TABLES
@pytest.mark.parametrize("fmt", [F16, BF16])
@pytest.mark.parametrize("query_scale,key_scale", [
    (1e4, 1e-4), (1e-30, 1.0), (3e6, 1e-6), (0.0, 1.0), (1.0, 1e-5), (30.0, 1.0)])
def test_queries_and_keys_of_any_size(device, fmt, query_scale, key_scale, keys):
    # F16 keys of 1e-5 and 1e-6 are subnormal; scores of 30 make peaked weights.
    paged, query, positions = batch(device, 15, [150, 33, 1], 4, 1, 256, 16, fmt, scale=key_scale,
                                    wide=keys // 16)
    query = (query * query_scale).astype(np.float32)
    check_attention(device, paged, positions, query, 4, NONE, 1 / 16)


@pytest.mark.parametrize("fmt,query_scale,key_scale,value_scale", [
    (F16, 1e36, 1e-4, 1.0), (F16, 1.0, 1.0, 1e4), (BF16, 1e36, 1e-25, 1e25),
    (BF16, 1e-30, 1e30, 1.0), (BF16, 1.0, 1.0, 1e34), (BF16, 1.0, 1e36, 1e-6)])
def test_values_near_the_ends_of_the_range(device, fmt, query_scale, key_scale, value_scale):
    # Largest queries, keys and values whose products and sums F32 still holds.
    paged, query, positions = batch(device, 20, [150, 33, 1], 4, 1, 256, 16, fmt, scale=key_scale)
    query = (query * query_scale).astype(np.float32)
    paged.values[:] = to_format(of_format(paged.values, fmt) * value_scale, fmt)
    paged.upload()
    check_attention(device, paged, positions, query, 4, NONE,
                    1 / (16 * max(1.0, query_scale * key_scale)))


def test_negative_and_zero_scale(device):
    paged, query, positions = batch(device, 16, [150, 33, 1], 4, 1, 256, 16, F16)
    for scale in (-0.3, 0.0):
        check_attention(device, paged, positions, query, 4, NONE, scale)


def test_rising_scores(device):
    # Each key beats the one before, so the running maximum moves at every step.
    paged, query, positions = batch(device, 17, [640], 4, 1, 256, 16, F16)
    query[:] = 1.0
    for j in range(640):
        paged.keys[paged.page(0, j), j % 16, 0] = to_format(np.full(256, j / 64), F16)
    paged.upload()
    check_attention(device, paged, positions, query, 4, NONE, 1 / 16)


@pytest.mark.parametrize("length", [200, 3000])
def test_a_query_that_is_no_number_stays_in_its_row(device, length):
    paged, query, positions = batch(device, 18, [100, 100, length], 4, 1, 256, 16, F16)
    bad = query.copy()
    bad[1, 300] = np.nan
    bad[2, 1000] = np.inf
    got = attention(device, paged, positions, bad, 4, NONE, 1 / 16)
    want, far = attention_exact(paged, positions, query, 4, NONE, 1 / 16)
    for row, sound in ((0, [0, 1, 2, 3]), (1, [0, 2, 3]), (2, [0, 1, 2])):
        for h in range(4):
            at = slice(256 * h, 256 * h + 256)
            if h in sound:
                assert (abs(got[row, at] - want[row][at]) <= far[row][at]).all()
            else:
                assert np.isnan(got[row, at]).all()


def test_the_same_bits_every_time_and_from_threads(device):
    paged, query, positions = batch(device, 19, [5000, 20, 0, 900], 4, 1, 256, 64, F16)
    other, query2, positions2 = batch(device, 20, [64, 7000], 6, 2, 128, 16, BF16)
    want = attention(device, paged, positions, query, 4, NONE, 1 / 16)
    want2 = attention(device, other, positions2, query2, 6, 300, 0.1)
    bad = []

    def work(args, expected):
        for _ in range(20):
            if not np.array_equal(attention(device, *args), expected):
                bad.append(args)

    threads = [threading.Thread(target=work, args=x) for x in
               (((paged, positions, query, 4, NONE, 1 / 16), want),
                ((other, positions2, query2, 6, 300, 0.1), want2)) * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_two_handles_of_one_device_at_once(device):
    # Each has its own stream and workspace.
    import frizzle_amd as fz
    other = fz.Device(0)
    try:
        sets = [(d, *batch(d, 24 + i, [5000 + 300 * i, 20, 0, 900], 4, 1, 256, 64, F16))
                for i, d in enumerate((device, other))]
        want = [attention(d, p, at, q, 4, NONE, 1 / 16) for d, p, q, at in sets]
        bad = []

        def work(i):
            d, p, q, at = sets[i]
            for _ in range(30):
                if not np.array_equal(attention(d, p, at, q, 4, NONE, 1 / 16), want[i]):
                    bad.append(i)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not bad
        sets.clear()
    finally:
        other.close()


def test_batch_does_not_change_a_row_much(device):
    # A row's cut goes by the batch, so its bits may; its values stay in bounds.
    paged, query, positions = batch(device, 21, [3000] * 40, 4, 1, 256, 64, F16)
    full = check_attention(device, paged, positions, query, 4, NONE, 1 / 16)
    alone = attention(device, paged, positions[:1], query[:1], 4, NONE, 1 / 16)
    _, far = attention_exact(paged, positions[:1], query[:1], 4, NONE, 1 / 16)
    assert (abs(alone[0] - full[0]) <= 2 * far[0]).all()


def test_a_pool_past_32_bits(device):
    # Pages 2^31 values apart: byte offsets to 2^33, value offsets past 2^32.
    import frizzle_amd as fz
    from frizzle_amd import _lib
    rng = np.random.default_rng(22)
    dim, slots, pages, stride = 256, 16, 3, 1 << 31
    pool = device.empty((1,), np.uint8)
    big = fz.runtime.DeviceArray(device, 2 * (stride * (pages - 1) + 2 * slots * dim), np.uint8, (1,))
    keys = to_format(rng.normal(0, 1, (pages, 2, slots, dim)), F16)
    for p in range(pages):
        _lib.check(fz.load().frz_write(device.handle, big.ptr + 2 * stride * p,
                                       np.ascontiguousarray(keys[p]).ctypes.data, keys[p].nbytes))
    table, positions = device.array(np.array([[2, 0, 1]], np.uint32)), device.array(
        np.array([44], np.uint32))
    query = rng.normal(0, 1.5, (1, 1024)).astype(np.float32)
    dq, do = device.array(query), device.empty((1, 1024), np.float32)
    c = fz.Pages(big.ptr, big.ptr + 2 * slots * dim, F16, 1, dim, slots, pages, stride, table.ptr,
                 1, 3)
    _lib.check(fz.load().frz_op_attention_paged(device.handle, c, None, positions.ptr, dq.ptr, 1024,
                                                do.ptr, 1024, 4, NONE, 1 / 16, 1))
    device.sync()
    got = do.numpy()[0].reshape(4, dim)
    big.free()
    pool.free()
    k = keys.view(np.float16).astype(np.float64)[[2, 0, 1]]
    kk, vv = k[:, 0].reshape(-1, dim)[:45], k[:, 1].reshape(-1, dim)[:45]
    s = query.astype(np.float64).reshape(4, dim) @ kk.T / 16
    w = np.exp(s - s.max(1, keepdims=True))
    want = w / w.sum(1, keepdims=True) @ vv
    assert np.linalg.norm(got - want) <= 5e-6 * np.linalg.norm(want)
