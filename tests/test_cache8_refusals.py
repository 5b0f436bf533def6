"""What the ops over caches of 8 bits, over first keys and the reads refuse, before any
device is asked for. CPU only."""
import pytest

import frizzle_amd as fz
from _batch import BF16, F16, F32, NONE, fake_device
from frizzle_amd import _lib

I8 = 24
P = 1 << 20  # an address of the right alignment; nothing is read there


def pages(**changed):
    p = fz.Pages(P, P, I8, 2, 256, 32, 8, 32 * 512, P, 4, 2, P, P, 4)
    for k, v in changed.items():
        setattr(p, k, v)
    return p


def attention(cache, sinks=None, window=NONE, rows=4, query=P, out=2 * P, device=True, scale=0.1):
    lib, device = fz.load(), fake_device() if device else None
    if sinks is None:
        return lib.frz_op_attention_paged(device, cache, P, P, query, 1024, out, 1024, 4, window,
                                          scale, rows)
    return lib.frz_op_attention_paged_sinks(device, cache, P, P, query, 1024, out, 1024, 4, window,
                                            sinks, scale, rows)


def rope(cache, rows=4):
    return fz.load().frz_op_rope_paged(fake_device(), cache, P, P, P, P, P, P, P, P, 1024, 512,
                                       2 * P, 1024, 4, 1e-6, rows)


def read(cache, device=True, sequences=P, positions=P, fmt=F16, keys=2 * P, values=3 * P,
         stride=512, rows=4):
    return fz.load().frz_op_read_paged(fake_device() if device else None, cache, sequences,
                                       positions, fmt, keys, values, stride, rows)


def refused(status, text):
    assert status == 1  # FRZ_ERR_ARGUMENT
    with pytest.raises(fz.FrzError, match=text):
        _lib.check(status)


@pytest.mark.parametrize("changed,text", [
    (dict(key_scales=None), "null scales"), (dict(value_scales=None), "null scales"),
    (dict(key_scales=P + 2), "scales not"), (dict(value_scales=P + 1), "scales not"),
    (dict(scale_stride=3), "scale_stride"), (dict(scale_stride=0), "scale_stride"),
    (dict(scale_stride=1 << 60), "scale_stride"), (dict(scale_stride=(1 << 45) + 1), "scale_stride"),
    (dict(page_stride=32 * 512 + 8), "page_stride"), (dict(page_stride=32 * 512 - 16), "page_stride"),
    (dict(page_stride=1 << 60), "page_stride"), (dict(keys=P + 8), "16 bytes"),
    (dict(values=None), "null"), (dict(head_dim=32), "head_dim"), (dict(page_slots=24), "page_slots"),
    (dict(format=8), "format"), (dict(format=25), "format"), (dict(kv_heads=0), "heads"),
    (dict(width=1 << 20), "width"), (dict(sequences=0), "sequences"),
])
def test_caches_refused(changed, text):
    for status in (attention(pages(**changed)), attention(pages(**changed), sinks=4),
                   rope(pages(**changed)), read(pages(**changed))):
        refused(status, text)


def test_caches_of_16_bits_need_no_scales():
    for fmt in (F16, BF16):
        cache = pages(format=fmt, key_scales=None, value_scales=None, scale_stride=0)
        refused(attention(cache, rows=0), "rows")
        refused(rope(cache, rows=0), "rows")
        refused(read(cache, rows=0), "rows")


@pytest.mark.parametrize("more,text", [
    (dict(device=False), "frz_op_attention_paged_sinks: no device"), (dict(window=0), "window"),
    (dict(rows=0), "rows"), (dict(rows=513), "rows"), (dict(query=None), "null"),
    (dict(out=P), "query"), (dict(out=2 * P + 8), "16 bytes"), (dict(scale=float("nan")), "scale"),
])
def test_sinks_refused(more, text):
    refused(attention(pages(), sinks=3, **more), text)


@pytest.mark.parametrize("more,text", [
    (dict(device=False), "no device"), (dict(positions=None), "null"), (dict(keys=None), "null"),
    (dict(values=None), "null"), (dict(fmt=I8), "format"), (dict(fmt=2), "format"),
    (dict(fmt=-1), "format"), (dict(keys=P + 8), "16 bytes"), (dict(values=P + 4), "16 bytes"),
    (dict(positions=P + 2), "16 bytes"), (dict(sequences=P + 1), "16 bytes"),
    (dict(stride=504), "stride"), (dict(stride=516), "stride"), (dict(stride=0), "stride"),
    (dict(stride=1 << 62), "stride"), (dict(stride=1 << 47), "stride"), (dict(rows=0), "rows"),
    (dict(rows=(1 << 23) + 1), "rows"), (dict(rows=NONE), "rows"), (dict(values=2 * P), "each other"),
    (dict(keys=P), "cache"), (dict(values=P), "cache"),
])
def test_reads_refused(more, text):
    refused(read(pages(), **more), text)


def test_null_structures_refused():
    refused(attention(None, sinks=1), "null")
    refused(read(None), "null")


def test_reads_take_every_cache_and_format():
    for cache in (F16, BF16, I8):
        for fmt in (F32, F16, BF16):
            refused(read(pages(format=cache), fmt=fmt, stride=4), "stride")
