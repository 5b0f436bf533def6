"""Norm, rope and the append to pages (frz_op_rope_paged): bit for bit
frz_op_rope where that op has the layout, and against values in 64 bits."""
import numpy as np
import pytest

import frizzle_amd as fz
from _batch import BF16, F16, NONE, Paged, of_format, rope, rope_exact, to_format
from frizzle_amd import _lib

pytestmark = pytest.mark.gpu


def inputs(rng, rows, heads, kv, dim):
    return (rng.normal(0, 2, (rows, heads * dim)).astype(np.float32),
            rng.normal(0, 2, (rows, kv * dim)).astype(np.float32),
            rng.normal(0, 2, (rows, kv * dim)).astype(np.float32),
            (1 + 0.1 * rng.normal(0, 1, (2, dim))).astype(np.float32))


@pytest.mark.parametrize("heads,kv,dim,base", [
    (4, 1, 256, 1e6), (4, 1, 256, 1e4), (2, 2, 128, 1e4), (8, 4, 128, 1e6), (16, 8, 64, 1e4),
    (1, 1, 64, 1e6)])
def test_rows_equal_frz_op_rope(device, heads, kv, dim, base):
    # Each row against a call of frz_op_rope of its own, whose ring holds the
    # position's slot.
    rng = np.random.default_rng(heads * dim)
    lengths = [1, 300, 0, 5004, 8192, 17]
    paged = Paged(device, rng, lengths, kv, dim, 64, F16)
    positions = [n - 1 if n else NONE for n in lengths]
    query, key, value, gains = inputs(rng, len(lengths), heads, kv, dim)
    turns = fz.rope_turns(base, dim)
    before = [p.copy() for p in paged.pools]
    got = rope(device, paged, positions, turns, gains, query, key, value, heads)
    keys, values, raw = paged.read()
    for row, p in enumerate(positions):
        if p == NONE:
            assert (got[row] == 7.0).all()
            continue
        dq = device.array(query[row])
        dk, dv = device.array(key[row]), device.array(value[row])
        ck, cv = (device.empty((kv * dim,), np.uint16) for _ in range(2))
        dt, dqg, dkg = device.array(turns), device.array(gains[0]), device.array(gains[1])
        _lib.check(fz.load().frz_op_rope(
            device.handle, dt.ptr, dqg.ptr, dkg.ptr, dq.ptr, dk.ptr, dv.ptr, heads * dim, kv * dim,
            ck.ptr, cv.ptr, 1, dim, heads, kv, 1e-6, p, 1))
        assert np.array_equal(got[row].view(np.uint32), dq.numpy().view(np.uint32)), row
        at = paged.page(row, p), p % 64
        assert np.array_equal(keys[at].ravel(), ck.numpy()), row
        assert np.array_equal(values[at].ravel(), cv.numpy()), row
        # Where the append went, for the comparison of all the rest.
        for now, was in zip((keys, values), before):
            page = np.lib.stride_tricks.as_strided(was, now.shape, now.strides)
            page[at] = now[at]
    for now, was in zip(raw, before):
        assert np.array_equal(now, was), "a slot of no row was written"


# Norm and turn in F32: the mean's sum and root, two products and the rotation
# are under 16 roundings of 2^-24, the angle (under pi, rounded once, its sine and
# cosine to 2^-23) another 8 of the pair.
def near(x):
    return 24 * 2.0 ** -24 * x


@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (5, 5, 64), (48, 3, 256), (7, 1, 128)])
@pytest.mark.parametrize("fmt", [F16, BF16])
def test_layouts_against_64_bits(device, heads, kv, dim, fmt):
    rng = np.random.default_rng(heads + dim)
    lengths = [3, 0, 40, 16, 4001]
    paged = Paged(device, rng, lengths, kv, dim, 16, fmt, interleaved=True, pad=8)
    positions = [n - 1 if n else NONE for n in lengths]
    query, key, value, gains = inputs(rng, len(lengths), heads, kv, dim)
    turns = fz.rope_turns(1e6, dim)
    got = rope(device, paged, positions, turns, gains, query, key, value, heads, extra=12,
               out_width=heads * dim + 8)
    assert (got[:, heads * dim:] == 7.0).all()
    keys, values, _ = paged.read()
    step = 2.0 ** -11 if fmt == F16 else 2.0 ** -8
    for row, p in enumerate(positions):
        if p == NONE:
            continue
        want, size = rope_exact(query[row].reshape(heads, dim), gains[0], turns, p)
        assert (abs(got[row, :heads * dim].reshape(heads, dim) - want) <= near(size)).all()
        want, size = rope_exact(key[row].reshape(kv, dim), gains[1], turns, p)
        at = paged.page(row, p), p % 16
        k = of_format(keys[at], fmt)
        assert (abs(k - want) <= step * abs(want) + (1 + step) * near(size) + 2.0 ** -25).all()
        assert np.array_equal(values[at].ravel(), to_format(value[row], fmt))


def test_in_place_and_requests_in_any_order(device):
    rng = np.random.default_rng(4)
    paged = Paged(device, rng, [100, 40, 64], 1, 256, 16, F16)
    requests, positions = [1, 0, 2, 0, 0], [39, 5, 63, 6, 99]
    query, key, value, gains = inputs(rng, 5, 4, 1, 256)
    turns = fz.rope_turns(1e4, 256)
    apart = rope(device, paged, positions, turns, gains, query, key, value, 4, requests)
    first = paged.read()
    paged.upload()
    there = rope(device, paged, positions, turns, gains, query, key, value, 4, requests,
                 in_place=True)
    assert np.array_equal(there[:, :1024], apart)
    # The keys and values beside the queries are left as they were.
    assert np.array_equal(there[:, 1024:1280], key) and np.array_equal(there[:, 1280:], value)
    for a, b in zip(first[:2], paged.read()[:2]):
        assert np.array_equal(a, b)
    for row, (r, p) in enumerate(zip(requests, positions)):
        got = first[1][paged.page(r, p), p % 16]
        assert np.array_equal(got.ravel(), to_format(value[row], F16))


@pytest.mark.parametrize("rows", [2, 65, 150, 512])
def test_the_last_of_rows_at_one_position_stays(device, rows):
    rng = np.random.default_rng(5)
    paged = Paged(device, rng, [64, 64, 64], 2, 64, 16, F16)
    # All at one request's position but a few, which come to be alone or last.
    requests, positions = np.zeros(rows, np.uint32), np.full(rows, 50, np.uint32)
    last = {(0, 50): rows - 1}
    if rows > 2:
        requests[2], last[1, 50] = 1, 2
        positions[3] = NONE
        positions[5] = positions[rows - 2] = 51
        last[0, 51] = rows - 2
    query, key, value, gains = inputs(rng, rows, 4, 2, 64)
    rope(device, paged, positions, fz.rope_turns(1e4, 64), gains, query, key, value, 4, requests)
    keys, values, _ = paged.read()
    for (request, p), row in last.items():
        at = paged.page(request, p), p % 16
        assert np.array_equal(values[at].ravel(), to_format(value[row], F16)), row
        want, size = rope_exact(key[row].reshape(2, 64), gains[1], fz.rope_turns(1e4, 64), p)
        k = of_format(keys[at], F16)
        assert (abs(k - want) <= 2.0 ** -11 * abs(want) + 2 * near(size) + 2.0 ** -25).all()


def test_slots_that_are_not_there(device):
    # The query is roped, nothing is appended.
    rng = np.random.default_rng(6)
    paged = Paged(device, rng, [64, 64, 64, 64], 1, 256, 16, F16)
    paged.table[0, 3], paged.table[1, 3] = NONE, paged.pages
    paged.upload()
    requests, positions = [0, 1, 2, 7, NONE], [63, 63, 64, 5, 5]
    query, key, value, gains = inputs(rng, 5, 4, 1, 256)
    turns = fz.rope_turns(1e6, 256)
    got = rope(device, paged, positions, turns, gains, query, key, value, 4, requests)
    for row, p in enumerate(positions):
        want, size = rope_exact(query[row].reshape(4, 256), gains[0], turns, p)
        assert (abs(got[row].reshape(4, 256) - want) <= near(size)).all()
    for now, was in zip(paged.read()[2], paged.pools):
        assert np.array_equal(now, was)


def test_values_out_of_the_format_and_no_numbers(device):
    rng = np.random.default_rng(7)
    paged = {f: Paged(device, rng, [16], 1, 64, 16, f) for f in (F16, BF16)}
    query, key, value, gains = inputs(rng, 1, 1, 1, 64)
    value[0, :6] = [1e6, -1e6, np.inf, np.nan, 65519.9, 1e-7]
    turns = fz.rope_turns(1e4, 64)
    for fmt, p in paged.items():
        rope(device, p, [3], turns, gains, query, key, value, 1)
        got = of_format(p.read()[1][p.page(0, 3), 3].ravel(), fmt)
        want = value[0].astype(np.float64)
        if fmt == F16:
            want = np.clip(want, -65504, 65504)
        assert np.array_equal(of_format(to_format(want, fmt), fmt), got, equal_nan=True)


def test_the_most_rows_of_requests_prompts(device):
    rng = np.random.default_rng(8)
    lengths = [200, 180, 132]
    paged = Paged(device, rng, lengths, 1, 128, 16, BF16)
    requests = np.repeat(np.arange(3), lengths)
    positions = np.concatenate([np.arange(n) for n in lengths])
    order = rng.permutation(512)
    query, key, value, gains = inputs(rng, 512, 2, 1, 128)
    rope(device, paged, positions[order], fz.rope_turns(1e4, 128), gains, query, key, value, 2,
         requests[order])
    values = paged.read()[1]
    for row, i in enumerate(order):
        got = values[paged.page(requests[i], positions[i]), positions[i] % 16]
        assert np.array_equal(got.ravel(), to_format(value[row], BF16))
