"""How near the ops over requests come to 64 bits in the mean, for operands of
ordinary size: bounds that a loss of two bits anywhere would pass.

A rounding to F32 is off by 2^-24 / sqrt(3) at most in the mean, half of that as a
rule, 2.4e-8. The partial sums of n random terms grow like a random walk, so that
their roundings come to 2.4e-8 sqrt(n / 2) of the sum. What is added one after
another is at most a lane's or a wave's share of it, an eighth, and one more
addition a wave."""
import numpy as np
import pytest

from _batch import BF16, F16, F32, NONE, Paged, Pool, check_adapters, check_attention

pytestmark = pytest.mark.gpu


# Chains of up to 1,152 / 8 columns (2.0e-7) and of 128 ranks (1.9e-7): 2.8e-7
# together, and what parts leave out.
@pytest.mark.parametrize("fmt", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,rank,cols,rows", [
    (1, 16, 1152, 1536), (48, 32, 1152, 1100), (333, 64, 1152, 3001), (512, 128, 1152, 1300),
    (512, 128, 264, 4300), (400, 40, 1152, 5000)])
def test_adapters(device, fmt, tokens, rank, cols, rows):
    rng = np.random.default_rng(tokens + rank)
    pool = Pool(device, rng, 4, rank, cols, rows, fmt)
    which = [i * 4 // tokens for i in range(tokens)]
    x = rng.normal(0, 1, (tokens, cols)).astype(np.float32)
    check_adapters(device, pool, which, x, np.zeros((tokens, rows), np.float32), near=4e-7)


# Scores of about 1.5 from up to 256 products (2.7e-7 each), so weights to 4.1e-7;
# their sums' chains are an eighth of the keys at most, 2.4e-8 sqrt(250 / 2) = 2.7e-7.
@pytest.mark.parametrize("fmt", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 256), (8, 1, 128), (16, 1, 256), (6, 3, 64)])
@pytest.mark.parametrize("lengths,wide", [([300, 77, 16], 0), ([2000, 700, 1300], 0),
                                          ([300, 77, 16], 500)])
def test_attention(device, fmt, heads, kv, dim, lengths, wide):
    rng = np.random.default_rng(heads + dim)
    paged = Paged(device, rng, lengths, kv, dim, 32, fmt, wide=wide)
    query = rng.normal(0, 1.5, (len(lengths), heads * dim)).astype(np.float32)
    check_attention(device, paged, [n - 1 for n in lengths], query, heads, NONE, dim ** -0.5,
                    near=8e-7)
