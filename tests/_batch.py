"""A batch of requests for the tests: caches in pages, and the three ops over
them with their values in 64 bits."""
import ctypes
import math

import numpy as np
import torch

import frizzle_amd as fz
from frizzle_amd import _lib

NONE = 0xFFFFFFFF
F32, F16, BF16 = 0, 1, 30


def to_format(x, fmt):
    """Float values rounded to a format, as its bits."""
    if fmt == F32:
        return np.ascontiguousarray(x, dtype=np.float32)
    if fmt == F16:
        return np.asarray(x, dtype=np.float32).astype(np.float16).view(np.uint16)
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16)
    return t.view(torch.int16).numpy().view(np.uint16)


def of_format(bits, fmt):
    """A format's bits as float64."""
    if fmt == F32:
        return bits.astype(np.float64)
    if fmt == F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Paged:
    """A pool with every request's pages in no order, on host and device. Slots
    that hold no key are NaN. `interleaved`: a page's keys and values side by
    side in one allocation; `pad` more values lie between pages."""

    def __init__(self, device, rng, lengths, kv_heads, dim, slots, fmt=F16, spare=2, pad=0,
                 interleaved=False, wide=0, scale=1.0):
        self.device, self.fmt, self.kv, self.dim, self.slots = device, fmt, kv_heads, dim, slots
        self.lengths = list(lengths)
        held = [-(-n // slots) for n in self.lengths]
        self.pages = sum(held) + spare
        order = rng.permutation(self.pages).astype(np.uint32)
        self.table = np.full((len(held), max(max(held), 1) + wide), NONE, dtype=np.uint32)
        at = 0
        for i, n in enumerate(held):
            self.table[i, :n] = order[at:at + n]
            at += n
        page = slots * kv_heads * dim
        self.stride = (2 if interleaved else 1) * page + pad
        nan = to_format(np.array([np.nan]), fmt)[0]
        pools = [np.full((self.pages, self.stride), nan, dtype=np.uint16)
                 for _ in range(1 if interleaved else 2)]
        # Views of each page's keys and values as [page][slot][head][dim].
        shape = (self.pages, slots, kv_heads, dim)
        strides = (2 * self.stride, 2 * kv_heads * dim, 2 * dim, 2)
        self.pools = pools
        self.keys = np.lib.stride_tricks.as_strided(pools[0], shape, strides)
        second = pools[0][:, page:] if interleaved else pools[1]
        self.values = np.lib.stride_tricks.as_strided(second, shape, strides)
        for i, n in enumerate(self.lengths):
            for j in range(0, n, slots):
                live, p = min(slots, n - j), self.table[i, j // slots]
                for pool in (self.keys, self.values):
                    x = scale * rng.normal(0, 1, (live, kv_heads, dim))
                    pool[p, :live] = to_format(x, fmt)
        self.offset = 2 * page if interleaved else 0
        self.upload()

    def upload(self):
        self.dev = [self.device.array(p) for p in self.pools]
        self.dev_table = self.device.array(self.table)

    def read(self):
        """The device's keys and values, as [page][slot][head][dim] bits."""
        raw = [d.numpy() for d in self.dev]
        shape, strides = self.keys.shape, self.keys.strides
        second = raw[0][:, self.offset // 2:] if self.offset else raw[1]
        return (np.lib.stride_tricks.as_strided(raw[0], shape, strides).copy(),
                np.lib.stride_tricks.as_strided(second, shape, strides).copy(), raw)

    def c(self, **changed):
        values = self.dev[0].ptr + self.offset if self.offset else self.dev[1].ptr
        p = fz.Pages(self.dev[0].ptr, values, self.fmt, self.kv, self.dim, self.slots, self.pages,
                     self.stride, self.dev_table.ptr, *self.table.shape)
        for k, v in changed.items():
            setattr(p, k, v)
        return p

    def page(self, request, j):
        """The page of a request's key j, or None."""
        if request >= len(self.table) or j // self.slots >= self.table.shape[1]:
            return None
        p = self.table[request, j // self.slots]
        return int(p) if p < self.pages else None

    def rows(self, request, first, end):
        """The keys and values that a row reads, in 64 bits: [key][head][dim]."""
        end = min(end, self.table.shape[1] * self.slots)
        at = [(self.page(request, j), j % self.slots) for j in range(min(first, end), end)]
        at = [x for x in at if x[0] is not None]
        p, s = [x[0] for x in at], [x[1] for x in at]
        return of_format(self.keys[p, s], self.fmt), of_format(self.values[p, s], self.fmt)


def ptr(array):
    return array.ptr if array is not None else None


def attention(device, paged, positions, query, heads, window, scale, requests=None, width=None,
              out=None, out_width=None):
    """The op's outputs, [rows][out_width]; rows start at 7."""
    rows, size = len(positions), heads * paged.dim
    width, out_width = width or size, out_width or size
    q = np.full((rows, width), np.nan, np.float32)
    q[:, :size] = query
    dq, dp = device.array(q), device.array(np.asarray(positions, np.uint32))
    dr = None if requests is None else device.array(np.asarray(requests, np.uint32))
    do = out or device.array(np.full((rows, out_width), 7.0, np.float32))
    _lib.check(fz.load().frz_op_attention_paged(
        device.handle, paged.c(), ptr(dr), dp.ptr, dq.ptr, width, do.ptr, out_width, heads,
        window, scale, rows))
    device.sync()
    return do.numpy()


def attention_exact(paged, positions, query, heads, window, scale, requests=None):
    """(rows' outputs in 64 bits, how far F32 sums may be off them): None for a
    row at no position.

    A score is a sum of D products. The query's parts leave 2^-22 of each
    (three BF16 parts 2^-24), D additions in F32 at most D 2^-24, its scaling
    and the exponent's subtraction a few 2^-24 of the score. An output is then
    off by e^(2 ds) - 1 of the largest value, by 2^-22 for the weights' parts
    and by one 2^-24 an addition of the chain that a key's weight goes through
    (its wave's, at most all keys), and the exponential's and joins' few.
    """
    kv, dim, group = paged.kv, paged.dim, heads // paged.kv
    out, far = [], []
    for row, p in enumerate(positions):
        if p == NONE:
            out.append(None)
            far.append(None)
            continue
        request = row if requests is None else requests[row]
        k, v = paged.rows(request, max(0, int(p) + 1 - window), int(p) + 1)
        q = query[row].astype(np.float64).reshape(kv, group, dim)
        o, f = np.zeros((kv, group, dim)), np.zeros((kv, group, 1))
        if len(k):
            s = np.einsum("hgd,khd->hgk", q, k) * scale
            size = np.einsum("hgd,khd->hgk", abs(q), abs(k)).max(-1) * abs(scale)
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            o = np.einsum("hgk,khd->hgd", w, v)
            ds = size * (2.0 ** -22 + dim * 2.0 ** -24) + abs(s).max(-1) * 2.0 ** -21
            # Weights sum to one, so neither sum passes the largest value.
            off = np.expm1(2 * ds) + 2.0 ** -21 + len(k) * 2.0 ** -24 + 2.0 ** -20
            f = (off * abs(v).max())[..., None]
        out.append(o.reshape(-1))
        far.append(np.broadcast_to(f, o.shape).reshape(-1))
    return out, far


def check_attention(device, paged, positions, query, heads, window, scale, requests=None,
                    near=5e-6, **more):
    """The op against its values in 64 bits: each output within the bound, all of
    them in the mean within `near` (errors of either sign add up like a random
    walk's steps, sqrt(D) 2^-24 and not D 2^-24 of a score)."""
    got = attention(device, paged, positions, query, heads, window, scale, requests, **more)
    want, far = attention_exact(paged, positions, query, heads, window, scale, requests)
    size, off, total = heads * paged.dim, 0.0, 0.0
    for row, (w, f) in enumerate(zip(want, far)):
        if w is None:
            assert (got[row] == 7.0).all(), f"row {row} is none and was written"
            continue
        assert (got[row, size:] == 7.0).all(), f"row {row} was written past its width"
        assert np.isfinite(got[row, :size]).all(), f"row {row}"
        error = abs(got[row, :size] - w)
        assert (error <= f).all(), f"row {row}: {error.max()} of {f[error.argmax()]}"
        off += (error ** 2).sum()
        total += (w ** 2).sum()
    assert off <= (near ** 2) * total, math.sqrt(off / total)
    return got


def rope(device, paged, positions, turns, gains, query, key, value, heads, requests=None,
         epsilon=1e-6, out_width=None, in_place=False, extra=0):
    """One call; the roped queries (rows start at 7), then paged.read() has the
    caches. Query, key and value lie side by side, `extra` floats after them."""
    rows, dim = query.shape[0], paged.dim
    q, k = heads * dim, paged.kv * dim
    width = q + 2 * k + extra
    qkv = np.full((rows, width), np.nan, np.float32)
    qkv[:, :q], qkv[:, q:q + k], qkv[:, q + k:q + 2 * k] = query, key, value
    d = device.array(qkv)
    dt, dq, dk = device.array(turns), device.array(gains[0]), device.array(gains[1])
    dp = device.array(np.asarray(positions, np.uint32))
    dr = None if requests is None else device.array(np.asarray(requests, np.uint32))
    out_width = width if in_place else out_width or q
    do = d if in_place else device.array(np.full((rows, out_width), 7.0, np.float32))
    _lib.check(fz.load().frz_op_rope_paged(
        device.handle, paged.c(), ptr(dr), dp.ptr, dt.ptr, dq.ptr, dk.ptr, d.ptr, d.ptr + 4 * q,
        d.ptr + 4 * (q + k), width, width, do.ptr, out_width, heads, epsilon, rows))
    device.sync()
    return do.numpy()


def rope_exact(x, gain, turns, p, epsilon=1e-6):
    """Heads [n][dim] normed and turned to position p, in 64 bits; the turns'
    product with the position is the model's, in F32."""
    x = x.astype(np.float64)
    dim = x.shape[-1]
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon) * gain.astype(np.float64)
    t = (np.float32(p) * turns).astype(np.float64)
    z = (n[:, :dim // 2] + 1j * n[:, dim // 2:]) * np.exp(2j * np.pi * (t - np.rint(t)))
    return np.concatenate([z.real, z.imag], 1), abs(n).max(-1, keepdims=True)


class Pool:
    """Adapters on host and device; what lies past an adapter's own rank is NaN."""

    def __init__(self, device, rng, count, rank, cols, rows, fmt, ranks=None, scales=None):
        self.count, self.rank, self.cols, self.rows, self.fmt = count, rank, cols, rows, fmt
        self.down = to_format(rng.normal(0, cols ** -0.5, (count, rank, cols)), fmt)
        self.up = to_format(rng.normal(0, rank ** -0.5, (count, rows, rank)), fmt)
        self.ranks = None if ranks is None else np.asarray(ranks, np.uint32)
        self.scales = None if scales is None else np.asarray(scales, np.float32)
        nan = to_format(np.array([np.nan]), fmt)[0]
        for a in range(count):
            self.down[a, self.own(a):] = nan
            self.up[a, :, self.own(a):] = nan
        self.dev = [None if x is None else device.array(x)
                    for x in (self.down, self.up, self.ranks, self.scales)]

    def own(self, a):
        return self.rank if self.ranks is None else min(int(self.ranks[a]), self.rank)

    def c(self, **changed):
        p = fz.Adapters(self.fmt, self.count, self.rank, self.cols, self.rows,
                        *(ptr(d) for d in self.dev))
        for k, v in changed.items():
            setattr(p, k, v)
        return p


def adapters(device, pool, which, x, base, x_width=None, base_width=None, y_width=None,
             in_place=False):
    """The op's outputs, [tokens][y_width]; they start at 7 (in place: at base)."""
    tokens = len(which)
    even = -(-pool.rows // 4) * 4

    def wide(a, width):
        w = np.full((tokens, width), 7.0, np.float32)
        w[:, :a.shape[1]] = a
        return device.array(w)

    x_width, base_width = x_width or pool.cols, base_width or even
    dx, db = wide(x, x_width), wide(base, base_width)
    y_width = base_width if in_place else y_width or even
    dy = db if in_place else device.array(np.full((tokens, y_width), 7.0, np.float32))
    dw = device.array(np.asarray(which, np.uint32))
    _lib.check(fz.load().frz_op_adapters(device.handle, pool.c(), dw.ptr, dx.ptr, x_width, db.ptr,
                                         base_width, dy.ptr, y_width, tokens))
    device.sync()
    return dy.numpy()


def adapters_exact(pool, which, x, base):
    """(y in 64 bits, how far F32 sums may be off it): a product's sum is off by
    at most one 2^-24 an addition of its terms' absolute sum."""
    y = base.astype(np.float64)
    far = 2.0 ** -23 * abs(y)
    which = np.asarray(which)
    for a in sorted(set(which.tolist())):
        r = pool.own(a) if a < pool.count else 0
        if r == 0:
            continue
        rows = np.flatnonzero(which == a)
        d = of_format(pool.down[a, :r], pool.fmt)
        u = of_format(pool.up[a, :, :r], pool.fmt)
        s = 1.0 if pool.scales is None else float(pool.scales[a])
        x64 = x[rows].astype(np.float64)
        y[rows] += s * (x64 @ d.T @ u.T)
        size = abs(s) * (abs(x64) @ abs(d).T @ abs(u).T)
        far[rows] += size * (pool.cols + r + 8) * 2.0 ** -24 + 2.0 ** -23 * abs(y[rows])
    return y, far


def check_adapters(device, pool, which, x, base, near=2e-6, **more):
    got = adapters(device, pool, which, x, base, **more)
    y, far = adapters_exact(pool, which, x, base)
    assert (got[:, pool.rows:] == 7.0).all(), "written past the outputs"
    error = abs(got[:, :pool.rows] - y)
    assert (error <= far).all(), (error / far).max()
    assert np.linalg.norm(error) <= near * np.linalg.norm(y)
    for t, a in enumerate(which):
        if a >= pool.count:  # base, to the bit
            assert np.array_equal(got[t, :pool.rows], base[t]), t
    return got


def fake_device():
    """A handle to refuse arguments by: not one is read that is refused."""
    return ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p)
