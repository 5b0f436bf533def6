"""Caches of 8 bits for the tests: pages of whole numbers and their blocks' scales, the
append as it is defined, and attention over first keys and a window in 64 bits."""
import math

import numpy as np

import frizzle_amd as fz
from _batch import F16, NONE, Paged, of_format, ptr, to_format
from frizzle_amd import _lib

I8 = 24
BLOCK = 16


class Paged8(Paged):
    """A pool of 8 bits with every request's pages in no order, on host and device. What
    no key holds is -128, its scale NaN where no key shares it. `pad` more values, and
    scales, lie between pages."""

    def __init__(self, device, rng, lengths, kv_heads, dim, slots, spare=2, pad=0, wide=0,
                 powers=(-6, -4), most=127):
        self.device, self.fmt, self.kv, self.dim, self.slots = device, I8, kv_heads, dim, slots
        self.lengths = list(lengths)
        held = [-(-n // slots) for n in self.lengths]
        self.pages = sum(held) + spare
        order = rng.permutation(self.pages).astype(np.uint32)
        self.table = np.full((len(held), max(max(held), 1) + wide), NONE, dtype=np.uint32)
        at = 0
        for i, n in enumerate(held):
            self.table[i, :n] = order[at:at + n]
            at += n
        page, blocks = slots * kv_heads * dim, slots // BLOCK * kv_heads
        self.stride, self.scale_stride = page + pad, blocks + pad
        self.pools = [np.full((self.pages, self.stride), -128, np.int8) for _ in range(2)]
        self.scale_pools = [np.full((self.pages, self.scale_stride), np.nan, np.float32)
                            for _ in range(2)]
        for i, n in enumerate(self.lengths):
            for j in range(0, n, BLOCK):
                p, first = self.table[i, j // slots], j % slots
                live = min(BLOCK, n - j)
                for codes, scales in zip(self.codes(), self.scales()):
                    x = np.rint(rng.normal(0, most / 4, (live, kv_heads, dim)))
                    codes[p, first:first + live] = np.clip(x, -most, most)
                    scales[p, first // BLOCK] = 2.0 ** rng.integers(*powers, kv_heads,
                                                                    endpoint=True)
        self.upload()

    def codes(self):
        """Views of keys' and values' numbers, [page][slot][head][dim]."""
        shape = (self.pages, self.slots, self.kv, self.dim)
        strides = (self.stride, self.kv * self.dim, self.dim, 1)
        return [np.lib.stride_tricks.as_strided(p, shape, strides) for p in self.pools]

    def scales(self):
        """Views of their scales, [page][block][head]."""
        shape = (self.pages, self.slots // BLOCK, self.kv)
        strides = (4 * self.scale_stride, 4 * self.kv, 4)
        return [np.lib.stride_tricks.as_strided(p, shape, strides) for p in self.scale_pools]

    def upload(self):
        self.dev = [self.device.array(p) for p in self.pools + self.scale_pools]
        self.dev_table = self.device.array(self.table)

    def download(self):
        """What the device holds: numbers of keys and values, then their scales."""
        return [d.numpy() for d in self.dev]

    def c(self, **changed):
        p = fz.Pages(self.dev[0].ptr, self.dev[1].ptr, I8, self.kv, self.dim, self.slots,
                     self.pages, self.stride, self.dev_table.ptr, *self.table.shape,
                     self.dev[2].ptr, self.dev[3].ptr, self.scale_stride)
        for k, v in changed.items():
            setattr(p, k, v)
        return p

    def held(self, request, positions):
        """The keys and values at these positions, in 64 bits; None for one not there."""
        found = []
        for codes, scales in zip(self.codes(), self.scales()):
            rows = []
            for j in positions:
                p = self.page(request, j)
                # The product of 8 and 24 bits is rounded once, to F32.
                rows.append(None if p is None else (
                    codes[p, j % self.slots].astype(np.float32)
                    * scales[p, j % self.slots // BLOCK][:, None]).astype(np.float64))
            found.append(rows)
        return found

    def rows(self, request, first, end):
        end = min(end, self.table.shape[1] * self.slots)
        return of_found(self.held(request, range(min(first, end), end)), self)


def of_found(found, paged):
    shape = (-1, paged.kv, paged.dim)
    return [np.array([x for x in rows if x is not None], np.float64).reshape(shape)
            for rows in found]


def held(paged, request, positions):
    """The keys and values at these positions in any format, as [key][head][dim]."""
    if isinstance(paged, Paged8):
        return of_found(paged.held(request, positions), paged)
    at = [(paged.page(request, j), j % paged.slots) for j in positions]
    at = [x for x in at if x[0] is not None]
    p, s = [x[0] for x in at], [x[1] for x in at]
    return of_format(paged.keys[p, s], paged.fmt), of_format(paged.values[p, s], paged.fmt)


# ---- the append ------------------------------------------------------------------------


def block_scale(most):
    """The least power of two of which 127 reach `most`, 0 of 0."""
    if most == 0:
        return np.float32(0)
    if math.isinf(most):
        return np.float32(2.0 ** 121)
    m, e = math.frexp(most)
    return np.float32(2.0 ** min(121, max(-126, e - 7 + (m > 127 / 128))))


def append(paged, positions, keys, values, requests=None):
    """The rows' keys and values, as F32 [row][head][dim], into the host's pages."""
    rows = {}  # the last row of each position
    for row, p in enumerate(positions):
        request = row if requests is None else requests[row]
        if p != NONE and paged.page(request, p) is not None:
            rows[request, int(p)] = row
    for request, b in sorted({(r, p // BLOCK) for r, p in rows}):
        page, first = paged.page(request, b * BLOCK), b * BLOCK % paged.slots
        there = {p - b * BLOCK: row for (r, p), row in rows.items()
                 if r == request and p // BLOCK == b}
        for codes, scales, x in zip(paged.codes(), paged.scales(), (keys, values)):
            for h in range(paged.kv):
                block = codes[page, first:first + BLOCK, h]
                before = scales[page, first // BLOCK, h]
                if 0 in there or not 0 < before < np.inf:
                    before = np.float32(0)
                new = np.nan_to_num(x[list(there.values()), h], nan=0.0, posinf=np.inf,
                                    neginf=-np.inf)
                after = max(before, block_scale(float(abs(new).max())))
                ratio = before / after if after > 0 else np.float32(0)
                block[:] = np.rint(block.astype(np.float32) * np.float32(ratio))
                with np.errstate(over="ignore"):
                    y = new / after if after > 0 else 0 * new
                block[list(there)] = np.rint(np.clip(y, -127, 127))
                scales[page, first // BLOCK, h] = after


def read(device, paged, requests, positions, fmt, stride=None, start=7.0):
    """The op's keys and values, [row][stride] bits of `fmt`; rows start at 7."""
    rows, size = len(positions), paged.kv * paged.dim
    stride = stride or size
    out = [device.array(np.broadcast_to(to_format(np.array([start]), fmt), (rows, stride)).copy())
           for _ in range(2)]
    dp = device.array(np.asarray(positions, np.uint32))
    dr = None if requests is None else device.array(np.asarray(requests, np.uint32))
    _lib.check(fz.load().frz_op_read_paged(device.handle, paged.c(), ptr(dr), dp.ptr, fmt,
                                           out[0].ptr, out[1].ptr, stride, rows))
    device.sync()
    return [o.numpy() for o in out]


# ---- attention ---------------------------------------------------------------------------


def attention(device, paged, positions, query, heads, window, scale, requests=None, sinks=0,
              width=None, out_width=None):
    """The op's outputs, [rows][out_width]; rows start at 7."""
    rows, size = len(positions), heads * paged.dim
    width, out_width = width or size, out_width or size
    q = np.full((rows, width), np.nan, np.float32)
    q[:, :size] = query
    dq, dp = device.array(q), device.array(np.asarray(positions, np.uint32))
    dr = None if requests is None else device.array(np.asarray(requests, np.uint32))
    do = device.array(np.full((rows, out_width), 7.0, np.float32))
    _lib.check(fz.load().frz_op_attention_paged_sinks(
        device.handle, paged.c(), ptr(dr), dp.ptr, dq.ptr, width, do.ptr, out_width, heads,
        window, sinks, scale, rows))
    device.sync()
    return do.numpy()


def exact(paged, positions, query, heads, window, scale, requests=None, sinks=0):
    """(rows' outputs in 64 bits, how far F32 sums may be off them): None for a row at no
    position.

    As of 16 bits (_batch.attention_exact): parts of the query leave 2^-22 of a product,
    or whole numbers 2^-30 of the head's largest query for each of a key's values; D
    additions at most D 2^-24, scalings and the exponent a few 2^-24 of the score. Numbers
    of 8 bits are exact in F16, and their scales three more factors of a weight, 2^-24
    each, in what is left of 2^-20.
    """
    kv, dim, group = paged.kv, paged.dim, heads // paged.kv
    whole = isinstance(paged, Paged8)
    out, far = [], []
    for row, p in enumerate(positions):
        if p == NONE:
            out.append(None)
            far.append(None)
            continue
        request = row if requests is None else requests[row]
        end = min(int(p) + 1, paged.table.shape[1] * paged.slots)
        first = min(max(0, int(p) + 1 - window), end)
        at = sorted(set(range(min(sinks, end))) | set(range(first, end)))
        k, v = held(paged, request, at)
        q = query[row].astype(np.float64).reshape(kv, group, dim)
        o, f = np.zeros((kv, group, dim)), np.zeros((kv, group, 1))
        if len(k):
            s = np.einsum("hgd,khd->hgk", q, k) * scale
            size = np.einsum("hgd,khd->hgk", abs(q), abs(k)).max(-1) * abs(scale)
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            o = np.einsum("hgk,khd->hgd", w, v)
            ds = size * ((0 if whole else 2.0 ** -22) + dim * 2.0 ** -24)
            ds += abs(s).max(-1) * 2.0 ** -21
            if whole:
                ds += abs(q).max(-1) * abs(k).sum(-1).max(0)[:, None] * abs(scale) * 2.0 ** -30
            off = np.expm1(2 * ds) + 2.0 ** -21 + len(k) * 2.0 ** -24 + 2.0 ** -20
            f = (off * abs(v).max())[..., None]
        out.append(o.reshape(-1))
        far.append(np.broadcast_to(f, o.shape).reshape(-1))
    return out, far


def check(device, paged, positions, query, heads, window, scale, requests=None, sinks=0,
          near=5e-6, **more):
    """The op against its values in 64 bits: each output within the bound, all of them in
    the mean within `near`, as in _batch.check_attention."""
    got = attention(device, paged, positions, query, heads, window, scale, requests, sinks,
                    **more)
    want, far = exact(paged, positions, query, heads, window, scale, requests, sinks)
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


def any_pool(device, rng, lengths, kv, dim, slots, fmt=F16, wide=0):
    if fmt == I8:
        return Paged8(device, rng, lengths, kv, dim, slots, wide=wide)
    return Paged(device, rng, lengths, kv, dim, slots, fmt, wide=wide)
