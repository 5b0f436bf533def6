"""What the ops over a step of many requests refuse, before any device is asked
for: bad shapes, pointers, strides and sizes. CPU only."""
import pytest

import frizzle_amd as fz
from _batch import BF16, F16, F32, NONE, fake_device
from frizzle_amd import _lib

P = 1 << 20  # an address of the right alignment; nothing is read there


def pages(**changed):
    p = fz.Pages(P, P, F16, 1, 256, 16, 8, 16 * 256, P, 4, 2)
    for k, v in changed.items():
        setattr(p, k, v)
    return p


def attention(cache=None, device=True, sequences=P, positions=P, query=P, q_stride=1024,
              out=2 * P, out_stride=1024, heads=4, window=NONE, scale=0.0625, rows=4):
    return fz.load().frz_op_attention_paged(
        fake_device() if device else None, cache, sequences, positions, query, q_stride, out,
        out_stride, heads, window, scale, rows)


def rope(cache=None, device=True, sequences=P, positions=P, turns=P, query_gain=P, key_gain=P,
         query=P, key=P, value=P, q_stride=1024, kv_stride=256, roped=2 * P, roped_stride=1024,
         heads=4, rows=4):
    return fz.load().frz_op_rope_paged(
        fake_device() if device else None, cache, sequences, positions, turns, query_gain,
        key_gain, query, key, value, q_stride, kv_stride, roped, roped_stride, heads, 1e-6, rows)


def adapters(pool=None, device=True, which=P, x=P, x_stride=64, base=P, base_stride=100, y=2 * P,
             y_stride=100, tokens=4, **changed):
    if pool is None:
        pool = fz.Adapters(F16, 3, 16, 64, 99, P, P, P, P)
    for k, v in changed.items():
        setattr(pool, k, v)
    return fz.load().frz_op_adapters(fake_device() if device else None, pool, which, x, x_stride,
                                     base, base_stride, y, y_stride, tokens)


def refused(status, text):
    assert status == 1  # FRZ_ERR_ARGUMENT
    with pytest.raises(fz.FrzError, match=text):
        _lib.check(status)


CACHES = [
    (dict(keys=None), "null"), (dict(values=None), "null"), (dict(table=None), "null"),
    (dict(keys=P + 8), "16 bytes"), (dict(values=P + 2), "16 bytes"), (dict(table=P + 2), "4 bytes"),
    (dict(format=F32), "format"), (dict(format=8), "format"),
    (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=512), "head_dim"),
    (dict(kv_heads=0), "heads"), (dict(kv_heads=-1), "heads"), (dict(kv_heads=3), "heads"),
    (dict(page_slots=0), "page_slots"), (dict(page_slots=8), "page_slots"),
    (dict(page_slots=24), "page_slots"), (dict(page_slots=NONE - 15), "page_slots"),
    (dict(sequences=0), "sequences"), (dict(pages=0), "pages"), (dict(pages=NONE), "pages"),
    (dict(width=0), "width"), (dict(width=(1 << 20) + 1), "width"), (dict(width=NONE), "width"),
    (dict(page_stride=16 * 256 - 8), "page_stride"), (dict(page_stride=16 * 256 + 4), "page_stride"),
    (dict(page_stride=0), "page_stride"), (dict(page_stride=1 << 60), "page_stride"),
    (dict(page_stride=1 << 40, pages=(1 << 8) + 1), "page_stride"),
]


@pytest.mark.parametrize("changed,text", CACHES)
def test_caches_refused(changed, text):
    refused(attention(pages(**changed)), text)
    refused(rope(pages(**changed)), text)


@pytest.mark.parametrize("more,text", [
    (dict(device=False), "no device"), (dict(positions=None), "null"), (dict(query=None), "null"),
    (dict(out=None), "null"), (dict(query=P + 4), "16 bytes"), (dict(out=P + 8), "16 bytes"),
    (dict(positions=P + 1), "16 bytes"), (dict(sequences=P + 2), "16 bytes"),
    (dict(q_stride=1020), "strides"), (dict(q_stride=1026), "strides"),
    (dict(out_stride=-1024), "strides"), (dict(out_stride=0), "strides"), (dict(out=P), "query"),
    (dict(heads=0), "heads"), (dict(heads=-4), "heads"), (dict(heads=1025), "heads"),
    (dict(window=0), "window"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=4097.0), "scale"),
    (dict(scale=-1e30), "scale"), (dict(rows=0), "rows"), (dict(rows=513), "rows"),
    (dict(rows=NONE), "rows"),
])
def test_attention_refused(more, text):
    refused(attention(pages(), **more), text)


@pytest.mark.parametrize("more,text", [
    (dict(device=False), "no device"), (dict(positions=None), "null"), (dict(turns=None), "null"),
    (dict(query_gain=None), "null"), (dict(key_gain=None), "null"), (dict(query=None), "null"),
    (dict(key=None), "null"), (dict(value=None), "null"), (dict(roped=None), "null"),
    (dict(turns=P + 4), "16 bytes"), (dict(key=P + 4), "16 bytes"), (dict(value=P + 8), "16 bytes"),
    (dict(positions=P + 3), "16 bytes"), (dict(q_stride=1000), "strides"),
    (dict(kv_stride=252), "strides"), (dict(kv_stride=258), "strides"),
    (dict(roped_stride=1023), "strides"), (dict(query=3 * P, roped=3 * P, roped_stride=2048), "in place"),
    (dict(key=3 * P, roped=3 * P), "key or value"), (dict(value=3 * P, roped=3 * P), "key or value"),
    (dict(heads=5000), "heads"), (dict(rows=0), "rows"), (dict(rows=513), "rows"),
])
def test_rope_refused(more, text):
    refused(rope(pages(), **more), text)


def test_null_structures_refused():
    refused(attention(None), "null")
    refused(rope(None), "null")
    refused(fz.load().frz_op_adapters(fake_device(), None, P, P, 64, P, 100, P, 100, 4), "null")


@pytest.mark.parametrize("more,text", [
    (dict(device=False), "no device"), (dict(down=None), "null"), (dict(up=None), "null"),
    (dict(which=None), "null"), (dict(x=None), "null"), (dict(base=None), "null"),
    (dict(y=None), "null"), (dict(format=2), "format"), (dict(format=-1), "format"),
    (dict(count=0), "adapters"), (dict(count=NONE), "adapters"),
    (dict(rank=0), "rank"), (dict(rank=12), "rank"), (dict(rank=136), "rank"),
    (dict(rank=-8), "rank"), (dict(cols=0), "shape"), (dict(cols=60), "shape"),
    (dict(cols=-64), "shape"), (dict(cols=1 << 25), "shape"), (dict(rows=0), "shape"),
    (dict(rows=(1 << 24) + 1), "shape"), (dict(tokens=0), "tokens"), (dict(tokens=513), "tokens"),
    (dict(down=P + 8), "16 bytes"), (dict(up=P + 4), "16 bytes"), (dict(ranks=P + 2), "16 bytes"),
    (dict(scales=P + 1), "16 bytes"), (dict(which=P + 2), "16 bytes"), (dict(x=P + 4), "16 bytes"),
    (dict(base=P + 8), "16 bytes"), (dict(y=P + 12), "16 bytes"), (dict(x_stride=60), "strides"),
    (dict(x_stride=66), "strides"), (dict(base_stride=96), "strides"),
    (dict(y_stride=99), "strides"), (dict(y_stride=-100), "strides"),
    (dict(x=3 * P, y=P, y_stride=104), "another stride"),
    (dict(x=3 * P, y=3 * P), "y is x"),
])
def test_adapters_refused(more, text):
    refused(adapters(**more), text)


def test_formats_of_both():
    # BF16 caches and every format of adapters pass these checks: what is
    # refused here is only the last argument.
    refused(attention(pages(format=BF16), rows=0), "rows")
    for fmt in (F32, F16, BF16):
        refused(adapters(format=fmt, tokens=0), "tokens")
