"""The ops over requests at the ends of their operands' ranges, and beside
values far larger than the ones that count, against values in 64 bits."""
import numpy as np
import pytest

from _batch import (BF16, F16, F32, NONE, Paged, Pool, adapters, adapters_exact, check_adapters,
                    check_attention, of_format, to_format)

pytestmark = pytest.mark.gpu


def batch(device, seed, lengths, heads, kv, dim, fmt, **more):
    rng = np.random.default_rng(seed)
    paged = Paged(device, rng, lengths, kv, dim, 16, fmt, **more)
    query = rng.normal(0, 1.0, (len(lengths), heads * dim)).astype(np.float32)
    return paged, query, [n - 1 for n in lengths]


# Ten thousand BF16 values near the type's largest (3.4e38), alike and of either
# sign, whose weights are about the same: their sum is far out of F32's range, the
# output, a mean of them, is in it.
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 64), (16, 2, 128), (12, 1, 256)])
@pytest.mark.parametrize("lengths", [[200, 31, 1], [10000, 700]])
@pytest.mark.parametrize("spread", [0.1, 2.0])
def test_sums_of_the_largest_values(device, heads, kv, dim, lengths, spread):
    paged, query, positions = batch(device, dim, lengths, heads, kv, dim, BF16, scale=0.02)
    values = of_format(paged.values, BF16) / 0.02
    values = np.clip(2e38 * (1.0 if spread < 1 else 0.0) + 5e37 * spread * values, -3e38, 3e38)
    paged.values[:] = to_format(values, BF16)
    paged.upload()
    check_attention(device, paged, positions, query, heads, NONE, dim ** -0.5)


# Small queries over BF16 keys near the type's largest (3.4e38): products and
# their sums fit F32, though those of a query of ordinary size would not.
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 64), (8, 1, 128), (16, 1, 256), (3, 3, 256)])
@pytest.mark.parametrize("query_scale", [1e-3, 1e-20, 1e-37])
def test_small_queries_over_the_largest_keys(device, heads, kv, dim, query_scale):
    paged, query, positions = batch(device, dim, [150, 33, 1], heads, kv, dim, BF16, scale=6e37)
    query = (query * query_scale).astype(np.float32)
    check_attention(device, paged, positions, query, heads, NONE,
                    1 / (dim ** 0.5 * query_scale * 6e37))


# One dimension of the query far above all others, over keys that are zero there:
# it counts for nothing, and costs the others none of their bits.
@pytest.mark.parametrize("fmt", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 256), (3, 3, 64), (8, 1, 128), (12, 1, 64),
                                          (16, 1, 256)])
@pytest.mark.parametrize("times", [2.0 ** 24, 2.0 ** 29])
def test_a_query_beside_a_dimension_of_no_key(device, fmt, heads, kv, dim, times):
    paged, query, positions = batch(device, heads, [150, 700, 1], heads, kv, dim, fmt)
    query.reshape(3, heads, dim)[:, :, dim // 3] *= times
    paged.keys[..., dim // 3] = 0
    paged.upload()
    check_attention(device, paged, positions, query, heads, NONE, dim ** -0.5, near=2e-6)


# Calls by tokens, and over runs of 16, 32 and 64: one and two tiles of ranks a
# workgroup, and four over long rows of 16-bit weights.
SHAPES = pytest.mark.parametrize("tokens,rank,cols,rows", [
    (20, 16, 264, 500), (300, 16, 20008, 515), (333, 64, 1152, 3001), (300, 40, 6920, 515),
    (511, 128, 200, 2300), (512, 64, 264, 4200)])


def adapters_of(device, rng, fmt, tokens, rank, cols, rows):
    pool = Pool(device, rng, 2, rank, cols, rows, fmt)
    # A column that no adapter takes.
    pool.down[:, :, 3] = 0
    pool.dev[0] = device.array(pool.down)
    which = [int(i) for i in np.sort(rng.integers(0, 2, tokens))]
    return pool, which, rng.normal(0, 1, (tokens, cols)).astype(np.float32)


# The column far above a token's others costs them none of their bits. A value of
# the others that is 2^-20 of them is off by 2^-51 of the column at most, which is
# 2^-23 of the others' size, as F32's own roundings of their sum are.
@pytest.mark.parametrize("fmt", [F32, F16, BF16])
@SHAPES
@pytest.mark.parametrize("times", [2.0 ** 20, 2.0 ** 24, 2.0 ** 28])
def test_tokens_beside_a_column_of_no_weight(device, fmt, tokens, rank, cols, rows, times):
    rng = np.random.default_rng(rows)
    pool, which, x = adapters_of(device, rng, fmt, tokens, rank, cols, rows)
    x[:, 3] *= times
    check_adapters(device, pool, which, x, np.zeros((tokens, rows), np.float32), near=1e-6)


# Small tokens keep their bits in every form. Parts of BF16, of x over BF16 weights
# and of the low-rank sums over all, end at 2^-134, so that 2^-23 of 2^-103 (1e-31)
# is still held, and of the low-rank sums of 1e-36 with weights 1,024 times as large
# as 1 / sqrt(cols), about 2^-110.
@pytest.mark.parametrize("fmt,size", [(F32, 1e-31), (BF16, 1e-28), (BF16, 1e-31), (F16, 1e-28),
                                      (F16, 1e-31), (F16, 1e-36)])
@SHAPES
def test_the_smallest_tokens(device, fmt, tokens, rank, cols, rows, size):
    rng = np.random.default_rng(rows)
    pool, which, x = adapters_of(device, rng, fmt, tokens, rank, cols, rows)
    for i, w in enumerate((pool.down, pool.up)):
        w[:] = to_format(of_format(w, fmt) * 1024, fmt)
        pool.dev[i] = device.array(w)
    check_adapters(device, pool, which, (x * size).astype(np.float32),
                   np.zeros((tokens, rows), np.float32), near=1e-6)


# Values between BF16's largest, 3.3895e38, and F32's, 3.4028e38, which F32 sums take
# like any other: x, a low-rank sum, a weight.
@pytest.mark.parametrize("fmt,place", [(f, p) for f in (F32, F16, BF16) for p in ("x", "low")]
                         + [(F32, "up")])
@SHAPES
def test_values_past_the_largest_of_16_bits(device, fmt, place, tokens, rank, cols, rows):
    rng = np.random.default_rng(rows)
    pool, which, x = adapters_of(device, rng, fmt, tokens, rank, cols, rows)
    down, up = of_format(pool.down, fmt), of_format(pool.up, fmt)
    if place == "x":
        x[:, 5] = 3.4e38 * rng.choice([-1, 1], tokens)
        down *= 2.0 ** -16
    elif place == "low":
        x[:] = 0
        x[:, 5] = 1.7e38 * rng.choice([-1, 1], tokens)
        down[:, :, 5], up = 2.0, up * 2.0 ** -8
    else:
        x *= 1e-3
        up = 3.4e38 * np.sign(up)
        down *= 1e-3
    for i, w in enumerate((down, up)):
        bits = to_format(w, fmt)
        (pool.down, pool.up)[i][:] = bits
        pool.dev[i] = device.array(bits)
    check_adapters(device, pool, which, x, np.zeros((tokens, rows), np.float32), near=1e-6)


# An infinite x, whichever form a call takes: infinite outputs of its weights' signs
# where one rank counts, no number where infinities of both signs meet.
@pytest.mark.parametrize("fmt", [F32, F16, BF16])
@SHAPES
def test_infinite_tokens(device, fmt, tokens, rank, cols, rows):
    rng = np.random.default_rng(rows)
    x = rng.normal(0, 1, (tokens, cols)).astype(np.float32)
    pool = Pool(device, rng, 2, rank, cols, rows, fmt, ranks=[1, rank])
    for i, w in enumerate((pool.down, pool.up)):  # no zeros
        w[of_format(w, fmt) == 0] = to_format(np.array([0.5]), fmt)[0]
        pool.dev[i] = device.array(w)
    which = [0] * (tokens // 2) + [1] * (tokens - tokens // 2)
    base = rng.normal(0, 1, (tokens, rows)).astype(np.float32)
    at = rng.choice(tokens, 5, replace=False)
    x[at, rng.integers(0, cols, 5)] = np.inf
    x[at[0]] *= -1
    want, far = adapters_exact(pool, which, np.where(np.isinf(x), 0, x), base)
    got = adapters(device, pool, which, x, base)[:, :rows]
    for t, a in enumerate(which):
        if not np.isinf(x[t]).any():
            assert (abs(got[t] - want[t]) <= far[t]).all(), t
            continue
        k = int(np.flatnonzero(np.isinf(x[t]))[0])
        r = pool.own(a)
        low = np.sign(of_format(pool.down[a, :r, k], fmt)) * np.sign(x[t, k])
        signs = np.sign(of_format(pool.up[a, :, :r], fmt)) * low
        one = abs(signs.sum(1)) == r
        assert np.array_equal(got[t, one], np.inf * signs[one, 0]), t
        assert np.isnan(got[t, ~one]).all(), t
