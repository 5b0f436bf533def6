"""The ops over requests at the ends of their operands' ranges, and beside
values far larger than the ones that count, against values in 64 bits."""
import numpy as np
import pytest

from _batch import BF16, F16, NONE, Paged, check_attention, of_format, to_format

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
