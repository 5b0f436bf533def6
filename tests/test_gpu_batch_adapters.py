"""Low-rank adapters beside a shared projection (frz_op_adapters) against their
values in 64 bits, and one layer's attention half of a batch's step through all
of the ops over requests."""
import threading

import numpy as np
import pytest

import frizzle_amd as fz
from _batch import (BF16, F16, F32, NONE, Paged, Pool, adapters, adapters_exact, attention_exact,
                    check_adapters, of_format, rope_exact, to_format)
from frizzle_amd import _lib
from helpers import q4_blocks

pytestmark = pytest.mark.gpu


def inputs(rng, tokens, pool):
    return (rng.normal(0, 1, (tokens, pool.cols)).astype(np.float32),
            rng.normal(0, 1, (tokens, pool.rows)).astype(np.float32))


@pytest.mark.parametrize("fmt", [F32, F16, BF16])
@pytest.mark.parametrize("rank,cols,rows", [
    (8, 8, 1), (16, 1152, 1536), (24, 40, 99), (64, 264, 257), (128, 1000, 130), (40, 6912, 64),
    (32, 1152, 1030)])
def test_shapes(device, fmt, rank, cols, rows):
    rng = np.random.default_rng(rank + cols)
    pool = Pool(device, rng, 5, rank, cols, rows, fmt, ranks=[rank, 1, rank - 3, 0, 7],
                scales=[1.0, -0.5, 2.0, 3.0, 0.0])
    which = [0, 0, 1, NONE, 2, 3, 4, 1, 2, 5, 0] + [2] * 20
    x, base = inputs(rng, len(which), pool)
    check_adapters(device, pool, which, x, base)


# Runs that end, begin and cross at sixteens, a token each, none, all.
@pytest.mark.parametrize("which", [
    [0], [NONE], [2] * 16, [1] * 17, [0] * 15 + [1] * 2, [0, 1] * 20, list(range(6)) * 11,
    [NONE] * 40, [0] * 512, [i // 100 for i in range(512)], [i % 7 for i in range(512)],
    [NONE] * 30 + [3] * 3 + [NONE] * 30, [4] * 33 + [NONE, 5, NONE] + [4] * 31])
def test_runs(device, which):
    rng = np.random.default_rng(len(which))
    pool = Pool(device, rng, 6, 16, 64, 300, F16)
    x, base = inputs(rng, len(which), pool)
    check_adapters(device, pool, which, x, base)


@pytest.mark.parametrize("cols", [8, 16, 24, 32, 40, 120, 128, 136, 248, 256, 264, 504, 8184, 8200,
                                  12288])
def test_columns_at_the_splits(device, cols):
    rng = np.random.default_rng(cols)
    pool = Pool(device, rng, 2, 24, cols, 20, BF16, ranks=[24, 17])
    which = [0, 1, 1, 0, NONE]
    x, base = inputs(rng, 5, pool)
    check_adapters(device, pool, which, x, base)


# Calls that read over 128 MB a token at a time, or over 600 kB of one token's D,
# go by runs of tokens with one adapter, in two launches: each compiled number of ranks (1, 2 or 4 tiles of D,
# 2, 4 or 8 of U) and run length (16, 32 and 64), K in one split and in up to 32,
# the last of them short or without columns.
@pytest.mark.parametrize("fmt,tokens,rank,cols,rows", [
    (F16, 512, 16, 264, 8100), (BF16, 450, 24, 6912, 300), (F32, 512, 40, 264, 4300),
    (BF16, 333, 64, 8200, 101), (F16, 512, 64, 40, 4500), (F16, 300, 128, 1152, 1901),
    (F32, 200, 128, 8, 2600), (BF16, 512, 128, 1000, 5002), (F32, 480, 24, 1504, 2200),
    (BF16, 512, 8, 14400, 2100), (F16, 511, 128, 200, 2300), (F32, 500, 64, 96, 2100),
    (F16, 300, 40, 6920, 515), (BF16, 16, 128, 8224, 1000), (F16, 9, 128, 65536, 24),
    (F32, 40, 16, 30008, 900), (F16, 1, 128, 4280, 701), (BF16, 3, 64, 9000, 130),
    (F32, 17, 128, 2304, 1), (F16, 2, 16, 20000, 257), (F32, 1, 8, 19400, 33)])
@pytest.mark.parametrize("pattern", ["one", "requests", "mixed"])
def test_runs_of_large_calls(device, fmt, tokens, rank, cols, rows, pattern):
    rng = np.random.default_rng(rank + cols)
    pool = Pool(device, rng, 5, rank, cols, rows, fmt, ranks=[rank, 1, rank - 3, 0, 7],
                scales=[1.0, -0.5, 2.0, 3.0, 0.25])
    if pattern == "one":
        which = [2] * tokens
    elif pattern == "requests":
        which = [(NONE, 0, 1, 2, 3, 4, 0)[i * 7 // tokens] for i in range(tokens)]
    else:
        which = [int(i) for i in rng.choice([0, 0, 1, 2, 4, 9], tokens)]
    x, base = inputs(rng, tokens, pool)
    check_adapters(device, pool, which, x, base)


@pytest.mark.parametrize("fmt,tokens,rank,cols,rows", [
    (F16, 300, 128, 1152, 1901), (BF16, 333, 64, 8200, 101), (F32, 500, 64, 96, 2100),
    (F16, 20, 16, 264, 500), (BF16, 20, 16, 264, 500)])
def test_tokens_of_any_size(device, fmt, tokens, rank, cols, rows):
    # Tokens of 10^-25 to 10^25 side by side, one of zeros, and a column 2^15 times
    # the others whose weights are zeros: it must cost them none of their bits.
    rng = np.random.default_rng(rows)
    pool = Pool(device, rng, 2, rank, cols, rows, fmt)
    pool.down[:, :, 3] = 0
    pool.dev[0] = device.array(pool.down)
    x, base = inputs(rng, tokens, pool)
    x[1::3, 3] = 2.0 ** 15
    size = (10.0 ** rng.uniform(-25, 25, (tokens, 1))).astype(np.float32)
    size[1] = 0.0
    which = [int(i) for i in np.sort(rng.integers(0, 2, tokens))]
    check_adapters(device, pool, which, x * size, base * size)


def test_runs_in_place_and_strided(device):
    rng = np.random.default_rng(8)
    pool = Pool(device, rng, 2, 64, 1152, 1538, F16, ranks=[64, 33])
    assert 512 * 64 * (1152 + 1538) * 2 > 128 << 20
    which = [0] * 100 + [1] * 200 + [NONE] * 70 + [0] * 142
    x, base = inputs(rng, 512, pool)
    plain = check_adapters(device, pool, which, x, base)[:, :1538]
    wide = check_adapters(device, pool, which, x, base, x_width=1160, base_width=1544, y_width=1600)
    assert np.array_equal(wide[:, :1538], plain)
    there = check_adapters(device, pool, which, x, base, in_place=True)
    assert np.array_equal(there[:, :1538], plain)


def test_strides_in_place_and_rows_behind(device):
    rng = np.random.default_rng(3)
    pool = Pool(device, rng, 3, 16, 128, 98, F16, scales=[0.5, 1, 2])
    which = [1, 1, NONE, 0, 2]
    x, base = inputs(rng, 5, pool)
    plain = check_adapters(device, pool, which, x, base)[:, :98]
    wide = check_adapters(device, pool, which, x, base, x_width=200, base_width=144, y_width=112)
    assert np.array_equal(wide[:, :98], plain)
    there = check_adapters(device, pool, which, x, base, base_width=116, in_place=True)
    assert np.array_equal(there[:, :98], plain)
    # Nothing past the tokens is written.
    d = [device.array(a) for a in (np.asarray(which, np.uint32), x)]
    y = device.array(np.full((9, 100), 7.0, np.float32))
    b = device.array(np.zeros((5, 100), np.float32))
    _lib.check(fz.load().frz_op_adapters(device.handle, pool.c(), d[0].ptr, d[1].ptr, 128, b.ptr,
                                         100, y.ptr, 100, 5))
    device.sync()
    assert (y.numpy()[5:] == 7.0).all()


def test_ranks_past_the_pool_and_an_empty_pool_entry(device):
    rng = np.random.default_rng(4)
    pool = Pool(device, rng, 3, 8, 64, 40, F32, ranks=[4000000000, 0, 8])
    x, base = inputs(rng, 4, pool)
    got = check_adapters(device, pool, [0, 1, 2, 1], x, base)
    assert np.array_equal(got[1], base[1]) and np.array_equal(got[3], base[3])


@pytest.mark.parametrize("tokens,rank,cols,rows", [(4, 16, 96, 50), (500, 64, 96, 2100)])
def test_a_token_that_is_no_number_stays_in_its_row(device, tokens, rank, cols, rows):
    rng = np.random.default_rng(5)
    pool = Pool(device, rng, 2, rank, cols, rows, F16, ranks=[13, rank])
    which = [0] * (tokens - 1) + [1]
    x, base = inputs(rng, tokens, pool)
    want, far = adapters_exact(pool, which, x, base)
    x[1, 3], x[-1, 95] = np.nan, np.inf
    got = adapters(device, pool, which, x, base)[:, :rows]
    sound = [0] + list(range(2, tokens - 1))
    assert (abs(got[sound] - want[sound]) <= far[sound]).all()
    assert np.isnan(got[1]).all() and not np.isfinite(got[-1]).any()


def test_the_same_bits_every_time_and_from_threads(device):
    rng = np.random.default_rng(6)
    sets = []
    # One launch, and two over runs.
    for rank, cols, rows, fmt, tokens in ((16, 1152, 1536, F16, 70), (128, 2504, 1500, BF16, 200)):
        pool = Pool(device, rng, 4, rank, cols, rows, fmt)
        which = [int(i) for i in rng.integers(0, 5, tokens)]
        x, base = inputs(rng, tokens, pool)
        sets.append((pool, which, x, base))
    want = [adapters(device, *s) for s in sets]
    bad = []

    def work(i):
        for _ in range(20):
            if not np.array_equal(adapters(device, *sets[i]), want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i % 2,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("tokens", [3, 300])
def test_a_pool_past_32_bits(device, tokens):
    # Down matrices of 2^23 values: the last adapter's lie past 2^32 of them.
    rng = np.random.default_rng(7)
    count, rank, cols, rows = 514, 128, 1 << 16, 24
    big = fz.runtime.DeviceArray(device, 2 * count * rank * cols, np.uint8, (1,))
    down = to_format(rng.normal(0, cols ** -0.5, (rank, cols)), F16)
    up = np.full((count, rows, rank), 0x7E00, np.uint16)  # NaN
    up[513] = to_format(rng.normal(0, rank ** -0.5, (rows, rank)), F16)
    _lib.check(fz.load().frz_write(device.handle, big.ptr + 2 * 513 * rank * cols,
                                   down.ctypes.data, down.nbytes))
    dev_up, which = device.array(up), device.array(np.full(tokens, 513, np.uint32))
    x = rng.normal(0, 1, (tokens, cols)).astype(np.float32)
    base = rng.normal(0, 1, (tokens, rows)).astype(np.float32)
    dx, db = device.array(x), device.array(base)
    p = fz.Adapters(F16, count, rank, cols, rows, big.ptr, dev_up.ptr, None, None)
    _lib.check(fz.load().frz_op_adapters(device.handle, p, which.ptr, dx.ptr, cols, db.ptr, rows,
                                         db.ptr, rows, tokens))
    device.sync()
    got = db.numpy()
    big.free()
    d, u = of_format(down, F16), of_format(up[513], F16)
    want = base + x.astype(np.float64) @ d.T @ u.T
    far = (abs(x).astype(np.float64) @ abs(d).T @ abs(u).T) * (cols + rank + 8) * 2.0 ** -24
    assert (abs(got - want) <= far + 2.0 ** -22 * abs(want)).all()
    assert np.linalg.norm(got - want) <= 3e-6 * np.linalg.norm(want)


# ---- together ------------------------------------------------------------------


def test_a_batch_of_requests_steps_through_a_layer(device):
    """Five requests' tokens through Q/K/V with adapters, rope and append, attention
    over pages, O with adapters, for three steps; every op enqueued, one wait a
    step; each step against 64 bits from the device's own products."""
    rng = np.random.default_rng(7)
    heads, kv, dim, hidden = 4, 1, 256, 1152
    qkv_rows = (heads + 2 * kv) * dim
    lengths = [100, 700, 1, 64, 0]
    steps = 3
    paged = Paged(device, rng, [n + steps for n in lengths], kv, dim, 64, F16)
    weights = {}
    for name, rows, cols in (("qkv", qkv_rows, hidden), ("o", hidden, heads * dim)):
        codes, scales = fz.block_split(fz.Q4_0, q4_blocks(rng, rows, cols))
        weights[name] = (device.array(codes), device.array(scales), rows, cols)
    pools = {"qkv": Pool(device, rng, 3, 16, hidden, qkv_rows, F16, ranks=[16, 9, 4]),
             "o": Pool(device, rng, 3, 16, heads * dim, hidden, F16, ranks=[16, 9, 4])}
    which = [2, NONE, 0, 1, 0]
    rows = len(lengths)
    gains = (1 + 0.1 * rng.normal(0, 1, (2, dim))).astype(np.float32)
    turns = fz.rope_turns(1e6, dim)
    dt, dqg, dkg = device.array(turns), device.array(gains[0]), device.array(gains[1])
    dw = device.array(np.asarray(which, np.uint32))
    lib = fz.load()
    for step in range(steps):
        # The last request is idle in the second step.
        positions = [n + step for n in lengths]
        if step == 1:
            positions[4] = NONE
        live = [r for r in range(rows) if positions[r] != NONE]
        dp = device.array(np.asarray(positions, np.uint32))
        x = rng.normal(0, 1, (rows, hidden)).astype(np.float32)
        dx = device.array(x)
        product, out = device.empty((rows, qkv_rows), np.float32), device.empty((rows, hidden),
                                                                                 np.float32)
        qkv = device.empty((rows, qkv_rows), np.float32)
        mixed = device.array(np.zeros((rows, heads * dim), np.float32))
        done = device.empty((rows, hidden), np.float32)
        codes, scales, n, k = weights["qkv"]
        _lib.check(lib.frz_op_gemv(device.handle, codes.ptr, scales.ptr, n, k, dx.ptr, k,
                                   product.ptr, n, rows, 0))
        _lib.check(lib.frz_op_adapters(device.handle, pools["qkv"].c(), dw.ptr, dx.ptr, hidden,
                                       product.ptr, qkv_rows, qkv.ptr, qkv_rows, rows))
        q = heads * dim
        _lib.check(lib.frz_op_rope_paged(
            device.handle, paged.c(), None, dp.ptr, dt.ptr, dqg.ptr, dkg.ptr, qkv.ptr,
            qkv.ptr + 4 * q, qkv.ptr + 4 * (q + dim), qkv_rows, qkv_rows, qkv.ptr, qkv_rows, heads,
            1e-6, rows))
        _lib.check(lib.frz_op_attention_paged(
            device.handle, paged.c(), None, dp.ptr, qkv.ptr, qkv_rows, mixed.ptr, q, heads, 512,
            1 / 16, rows))
        codes, scales, n, k = weights["o"]
        _lib.check(lib.frz_op_gemv(device.handle, codes.ptr, scales.ptr, n, k, mixed.ptr, k,
                                   out.ptr, n, rows, 0))
        _lib.check(lib.frz_op_adapters(device.handle, pools["o"].c(), dw.ptr, mixed.ptr, k, out.ptr,
                                       n, done.ptr, n, rows))
        device.sync()
        # Q/K/V from the shared product on, each op from what the one before left.
        full, _ = adapters_exact(pools["qkv"], which, x, product.numpy())
        got = qkv.numpy()
        keys, values, _ = paged.read()
        for r in live:
            want, size = rope_exact(full[r, :q].reshape(heads, dim), gains[0], turns, positions[r])
            assert abs(got[r, :q].reshape(heads, dim) - want).max() <= 4e-6 * size.max()
            at = paged.page(r, positions[r]), positions[r] % 64
            want, size = rope_exact(full[r, q:q + dim].reshape(1, dim), gains[1], turns,
                                    positions[r])
            k = of_format(keys[at], F16)
            assert (abs(k - want) <= 2.0 ** -11 * abs(want) + 4e-6 * size + 2.0 ** -25).all()
            v = of_format(values[at], F16).ravel()
            assert np.allclose(v, full[r, q + dim:], rtol=2.0 ** -10, atol=1e-5)
            # The host's caches go on with what the device appended.
            paged.keys[at], paged.values[at] = keys[at], values[at]
        want, far = attention_exact(paged, positions, got[:, :q], heads, 512, 1 / 16)
        a = mixed.numpy()
        for r in live:
            assert (abs(a[r] - want[r]) <= far[r]).all()
        if step == 1:
            assert (a[4] == 0.0).all()
        y, far = adapters_exact(pools["o"], which, a, out.numpy())
        assert (abs(done.numpy() - y) <= far).all()
