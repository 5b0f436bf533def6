"""Caches in 8 bits and a few first tokens that stay visible: a step's operators, as cases.

A cache in pages may hold a byte a value: whole numbers from -127 to 127, times a
scale that 16 tokens of one key-value head share, a power of two as the library writes
it. Beside the products that all requests share, a step over such caches has

  write      queries and keys normed for each head and turned to their request's
             position, keys and values quantised into its pages
             (frz_op_rope_paged), and what the touched blocks then hold read back
             (frz_op_read_paged)
  read       whole requests' keys and values out of their pages, for a product or a
             cache in another type (frz_op_read_paged)
  attention  each row's query over its request's keys (frz_op_attention_paged)
  sinks      the same over a sliding window and the request's first few keys, which
             stay visible; the pages between are gone. Caches of 16 bits as well
             (frz_op_attention_paged_sinks)

Where `own` is false, `run` computes them with elementary torch operations in
32 bits; where it is true it calls the library. Keys read, pages held and blocks
begun follow from the case alone, their order and all values from the seed.
"""
import functools
import math

import numpy as np
import torch

own = False

EPSILON = 1e-6
NONE = 0xFFFFFFFF  # no position, no page
BLOCK = 16         # tokens that share a scale
MOST = 127         # of a value's whole number
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
NUMBERS = {"f32": 0, "f16": 1, "i8": 24, "bf16": 30}  # GGUF's


def listed():
    return [
        # One reply's token of a global layer.
        {"name": "write_reply", "op": "write", "requests": 1, "tokens": 1, "idle": 0,
         "least": 5004, "most": 5004, "heads": 4, "kv": 1, "dim": 256, "slots": 64},
        # A batch of requests' tokens, each into a block of its own.
        {"name": "write_batch", "op": "write", "requests": 61, "tokens": 1, "idle": 3,
         "least": 40, "most": 8192, "heads": 4, "kv": 1, "dim": 256, "slots": 64},
        # Three prompts' rows of a wider model, blocks of 16 tokens at once.
        {"name": "write_prompts", "op": "write", "requests": 3, "tokens": 169, "idle": 2,
         "least": 180, "most": 4001, "heads": 32, "kv": 8, "dim": 128, "slots": 16},
        # A sliding layer's window, for a prompt's next rows.
        {"name": "read_window", "op": "read", "requests": 1, "least": 512, "most": 512, "kv": 1,
         "dim": 256, "slots": 16, "type": "f16"},
        # Two conversations of a wider model that go on in a cache of 16 bits.
        {"name": "read_books", "op": "read", "requests": 2, "least": 30001, "most": 65000,
         "kv": 8, "dim": 128, "slots": 64, "type": "bf16"},
        # One reply late in a conversation: a global layer's token.
        {"name": "attention_reply", "op": "attention", "rows": 1, "idle": 0, "least": 5004,
         "most": 5004, "heads": 4, "kv": 1, "dim": 256, "slots": 64},
        # A full batch of requests, some slots of it empty, over global layers.
        {"name": "attention_batch", "op": "attention", "rows": 64, "idle": 3, "least": 40,
         "most": 8192, "heads": 4, "kv": 1, "dim": 256, "slots": 64},
        # A wider model's heads, from first tokens to documents.
        {"name": "attention_heads", "op": "attention", "rows": 33, "idle": 1, "least": 1,
         "most": 4001, "heads": 16, "kv": 8, "dim": 128, "slots": 32},
        # Few requests over whole books.
        {"name": "attention_long", "op": "attention", "rows": 3, "idle": 0, "least": 98001,
         "most": 131072, "heads": 8, "kv": 4, "dim": 256, "slots": 128},
        # One endless reply, a sliding layer's token.
        {"name": "sinks_reply", "op": "sinks", "rows": 1, "idle": 0, "least": 70001,
         "most": 70001, "window": 512, "sinks": 4, "heads": 4, "kv": 1, "dim": 256, "slots": 16,
         "type": "f16"},
        # A batch of conversations, some shorter than the window, in 8 bits.
        {"name": "sinks_batch", "op": "sinks", "rows": 64, "idle": 3, "least": 100,
         "most": 50000, "window": 1024, "sinks": 5, "heads": 4, "kv": 1, "dim": 256,
         "slots": 64, "type": "i8"},
        # Streams of a wider model over a BF16 cache, a long system prompt kept.
        {"name": "sinks_heads", "op": "sinks", "rows": 29, "idle": 0, "least": 9001,
         "most": 300000, "window": 4000, "sinks": 130, "heads": 16, "kv": 8, "dim": 128,
         "slots": 32, "type": "bf16"},
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    """(query heads, key-value heads, head width)."""
    kv, group = rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 4, 6, 8, 16])
    return kv * group, kv, rng.choice([64, 128, 256, 256])


def draw(rng):
    op = rng.choice(["write", "write", "read", "attention", "attention", "sinks", "sinks"])
    heads, kv, dim = _heads(rng)
    slots = rng.choice([16, 16, 32, 48, 64, 128, 256])
    if op == "write":
        requests = _between(rng, 1, 256)
        tokens = _between(rng, 1, max(1, 512 // requests)) if rng.random() < 0.5 else 1
        most = tokens + _between(rng, 1, max(2, min(8192, 40_000_000 // (requests * kv * dim))))
        return {"op": op, "requests": requests, "tokens": tokens,
                "idle": rng.randint(0, min(requests // 8, 512 - requests * tokens)),
                "least": max(tokens, int(most * rng.uniform(0.01, 1))), "most": most,
                "heads": heads, "kv": kv, "dim": dim, "slots": slots}
    if op == "read":
        requests = rng.randint(1, 9)
        most = _between(rng, 1, max(2, 60_000_000 // (requests * kv * dim)))
        return {"op": op, "requests": requests, "least": max(1, int(most * rng.uniform(0.01, 1))),
                "most": most, "kv": kv, "dim": dim, "slots": slots,
                "type": rng.choice(["f16", "bf16", "f32"])}
    rows = _between(rng, 1, 512)
    # No more keys in all than the largest listed case reads: 3 x 131,072 of 4 x 256 values.
    cap = max(2, min(131072, 300_000_000 // (rows * kv * dim)))
    most = max(_between(rng, 1, cap), _between(rng, 1, cap))
    case = {"op": op, "rows": rows, "idle": rng.randint(0, rows // 8),
            "least": max(1, int(most * rng.uniform(0.01, 1))), "most": most, "heads": heads,
            "kv": kv, "dim": dim, "slots": slots}
    if op == "sinks":
        seen = max(2, min(8192, cap // 2))
        case.update(window=_between(rng, 1, seen), sinks=_between(rng, 1, min(300, seen)),
                    most=_between(rng, most, 1 << 20), type=rng.choice(["f16", "bf16", "i8", "i8"]))
    return case


# ---- what a case's rows are ----------------------------------------------------------


def _steps(case, n):
    """n lengths from least to most."""
    if n == 1:
        return [case["most"]]
    ratio = case["most"] / case["least"]
    return [int(round(case["least"] * ratio ** (i / (n - 1)))) for i in range(n)]


def _lengths(case):
    """Keys of each request, the last of them those of this step."""
    return _steps(case, case["requests"] if "requests" in case else case["rows"] - case["idle"])


def _held(case, length):
    """The keys that a row of the last one's reads, first to last."""
    if case["op"] != "sinks" or length <= case["window"] + case["sinks"]:
        return [(0, length)]
    return [(0, case["sinks"]), (length - case["window"], length)]


def _touched(case):
    """(request, first key, end) of what a step's blocks hold, those of earlier steps too."""
    return [(r, (n - case["tokens"]) // BLOCK * BLOCK, n) for r, n in enumerate(_lengths(case))]


def work(case):
    kv, dim, lengths = case["kv"], case["dim"], _lengths(case)
    if case["op"] == "read":
        keys = sum(lengths) * kv
        scales = sum(-(-n // BLOCK) for n in lengths) * kv
        return {"bytes": float(2 * keys * dim * (1 + TYPES[case["type"]].itemsize) + 8 * scales
                               + 8 * sum(lengths)), "flops": float(2 * keys * dim)}
    if case["op"] == "write":
        rows = len(lengths) * case["tokens"]
        queries, keys = rows * case["heads"] * dim, rows * kv * dim
        seen = sum(end - first for _, first, end in _touched(case)) * kv * dim
        # The step's rows, the touched blocks' earlier codes, and their values as read back.
        return {"bytes": float(4 * 2 * queries + 2 * (4 + 1) * keys + 2 * (seen - keys)
                               + 2 * (1 + 2) * seen), "flops": float(9 * (queries + 2 * keys))}
    queries = len(lengths) * case["heads"] * dim
    keys = sum(b - a for n in lengths for a, b in _held(case, n))
    pages = sum(-(-b // case["slots"]) - a // case["slots"]
                for n in lengths for a, b in _held(case, n))
    each = TYPES[case.get("type", "i8")].itemsize
    scales = 2 * 4 * keys * kv / BLOCK if each == 1 else 0
    return {"bytes": float(2 * keys * kv * dim * each + scales + 4 * 2 * queries + 4 * pages
                           + 8 * case["rows"]), "flops": float(4 * keys * case["heads"] * dim)}


# ---- the states ------------------------------------------------------------------------


def _random(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, kind=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=kind)


def _turns(dim, base=1e6):
    """Each pair's turns a position, rounded once to 32 bits."""
    k = np.arange(dim // 2, dtype=np.float64)
    return torch.from_numpy((base ** (-2 * k / dim) / (2 * math.pi)).astype(np.float32)).cuda()


def _unsigned(array):
    """A 32-bit word each, as torch holds them."""
    return torch.from_numpy(np.asarray(array, dtype=np.uint32).view(np.int32)).cuda()


def _power(of):
    """2 to whole numbers of -126 to 127, by F32's bits."""
    return (of.int() + 127 << 23).view(torch.float32)


def _pool(gen, kind, pages, slots, kv, dim):
    """Values of about 1, and in 8 bits the scales of each block and head."""
    if kind != torch.int8:
        return _normal(gen, pages, slots, kv, dim, kind=kind), None
    codes = torch.empty(pages, slots, kv, dim, dtype=kind, device="cuda")
    for some in codes.split(max(1, (1 << 26) // (slots * kv * dim))):
        some.copy_((_normal(gen, *some.shape) * 24).round_().clamp_(-MOST, MOST))
    return codes, _power(torch.randint(-6, -3, (pages, slots // BLOCK, kv), generator=gen,
                                       device="cuda"))


def _paged(case, seed, rows, kind):
    """The pool, every request's pages in no order, and `rows` of (request, position) with
    the idle ones among them in no order either."""
    rng, gen = np.random.default_rng(seed), _random(seed)
    slots, lengths = case["slots"], _lengths(case)
    held = [sorted({p for a, b in _held(case, n) for p in range(a // slots, -(-b // slots))})
            for n in lengths]
    pages = sum(map(len, held)) + 3
    order = rng.permutation(pages)
    table = np.full((len(held), max(p[-1] for p in held) + 1), NONE, dtype=np.uint32)
    at = 0
    for request, p in enumerate(held):
        table[request, p] = order[at:at + len(p)]
        at += len(p)
    rows = np.asarray(rows + [(0, NONE)] * case.get("idle", 0), dtype=np.uint32)
    if case["op"] != "read":
        rows = rows[rng.permutation(len(rows))]
    keys, key_scales = _pool(gen, kind, pages, slots, case["kv"], case["dim"])
    values, value_scales = _pool(gen, kind, pages, slots, case["kv"], case["dim"])
    return {"table": _unsigned(table), "requests": _unsigned(rows[:, 0]),
            "positions": _unsigned(rows[:, 1]), "keys": keys, "values": values,
            "key_scales": key_scales, "value_scales": value_scales}


def prepare(case, seed):
    s, gen = {"case": case}, _random(seed + 1)
    kv, dim, lengths = case["kv"], case["dim"], _lengths(case)
    if case["op"] == "read":
        rows = [(r, p) for r, n in enumerate(lengths) for p in range(n)]
        s.update(_paged(case, seed, rows, torch.int8))
        s["out"] = torch.empty(2, len(rows), kv, dim, dtype=TYPES[case["type"]], device="cuda")
        return s
    if case["op"] == "write":
        rows = [(r, p) for r, n in enumerate(lengths) for p in range(n - case["tokens"], n)]
        s.update(_paged(case, seed, rows, torch.int8))
        count = len(rows) + case["idle"]
        # One product gives a row's queries, keys and values side by side.
        s.update(qkv=1.5 * _normal(gen, count, (case["heads"] + 2 * kv) * dim),
                 turns=_turns(dim), query_gain=1 + 0.1 * _normal(gen, dim),
                 key_gain=1 + 0.1 * _normal(gen, dim))
        seen = np.asarray([(r, p) for r, a, b in _touched(case) for p in range(a, b)])
        s.update(seen_requests=_unsigned(seen[:, 0]), seen_positions=_unsigned(seen[:, 1]),
                 seen=torch.empty(2, len(seen), kv, dim, dtype=torch.float16, device="cuda"))
    else:
        s.update(_paged(case, seed, [(r, n - 1) for r, n in enumerate(lengths)],
                        TYPES[case.get("type", "i8")]))
        count = case["rows"]
        s["query"] = 1.5 * _normal(gen, count, case["heads"] * dim)
    s["out"] = torch.zeros(count, case["heads"] * dim, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------


def run(s):
    return (_library if own else _plain)[s["case"]["op"]](s)


@functools.lru_cache(None)
def _frizzle():
    import frizzle_amd
    # On torch's stream: the calls read what torch writes there, and torch reads what they write.
    device = frizzle_amd.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    return frizzle_amd, frizzle_amd._lib.check, frizzle_amd.load(), device


def _pages(fz, s):
    case, scales = s["case"], s["key_scales"]
    kind = "i8" if scales is not None else case["type"]
    more = () if scales is None else (scales.data_ptr(), s["value_scales"].data_ptr(),
                                      scales.stride(0))
    return fz.Pages(s["keys"].data_ptr(), s["values"].data_ptr(), NUMBERS[kind],
                    case["kv"], case["dim"], case["slots"], s["keys"].shape[0],
                    s["keys"].stride(0), s["table"].data_ptr(), s["table"].shape[0],
                    s["table"].shape[1], *more)


def _library_read(s, requests, positions, out, kind):
    fz, check, lib, device = _frizzle()
    check(lib.frz_op_read_paged(
        device.handle, _pages(fz, s), requests.data_ptr(), positions.data_ptr(), NUMBERS[kind],
        out[0].data_ptr(), out[1].data_ptr(), out.stride(1), out.shape[1]))
    return {"keys": out[0], "values": out[1]}


def _library_write(s):
    fz, check, lib, device = _frizzle()
    case, qkv = s["case"], s["qkv"]
    width = qkv.shape[1]
    at, q, k = qkv.data_ptr(), case["heads"] * case["dim"], case["kv"] * case["dim"]
    check(lib.frz_op_rope_paged(
        device.handle, _pages(fz, s), s["requests"].data_ptr(), s["positions"].data_ptr(),
        s["turns"].data_ptr(), s["query_gain"].data_ptr(), s["key_gain"].data_ptr(), at,
        at + 4 * q, at + 4 * (q + k), width, width, s["out"].data_ptr(), q, case["heads"],
        EPSILON, qkv.shape[0]))
    return {"query": s["out"],
            **_library_read(s, s["seen_requests"], s["seen_positions"], s["seen"], "f16")}


def _library_attention(s):
    fz, check, lib, device = _frizzle()
    case, width = s["case"], s["query"].shape[1]
    check(lib.frz_op_attention_paged(
        device.handle, _pages(fz, s), s["requests"].data_ptr(), s["positions"].data_ptr(),
        s["query"].data_ptr(), width, s["out"].data_ptr(), width, case["heads"], NONE,
        case["dim"] ** -0.5, case["rows"]))
    return {"out": s["out"]}


def _library_sinks(s):
    fz, check, lib, device = _frizzle()
    case, width = s["case"], s["query"].shape[1]
    check(lib.frz_op_attention_paged_sinks(
        device.handle, _pages(fz, s), s["requests"].data_ptr(), s["positions"].data_ptr(),
        s["query"].data_ptr(), width, s["out"].data_ptr(), width, case["heads"], case["window"],
        case["sinks"], case["dim"] ** -0.5, case["rows"]))
    return {"out": s["out"]}


_library = {"write": _library_write, "attention": _library_attention, "sinks": _library_sinks,
            "read": lambda s: _library_read(s, s["requests"], s["positions"], s["out"],
                                            s["case"]["type"])}


def _plain_norm(x, gain):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON) * gain


def _plain_turn(x, cosine, sine):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cosine - b * sine, a * sine + b * cosine], -1)


def _places(s, requests, positions):
    """The pool's slots, counted through all pages, of these keys."""
    slots = s["case"]["slots"]
    page = s["table"][requests.long(), positions.long() // slots].long()
    return page * slots + positions.long() % slots


def _plain_append(x, codes, scales, at):
    """Rows x [row][head][dim] into their blocks: a scale grows to the least power of two
    by which no number is past MOST, and what a block held goes by it too. A block whose
    first slot is written is begun anew."""
    codes, scales = codes.view(-1, BLOCK, *codes.shape[2:]), scales.view(-1, scales.shape[-1])
    block, slot = at // BLOCK, at % BLOCK
    begun = torch.zeros_like(scales[:, 0]).index_reduce(0, block, (slot == 0).float(), "amax")
    before = torch.where(begun[:, None] > 0, 0.0, scales)
    most, power = torch.frexp(x.abs().amax(-1))
    need = torch.where(most > 0, _power(power - 7 + (most > MOST / 128)), 0.0)
    after = before.index_reduce(0, block, need, "amax")
    # Rows of one block write it alike.
    ratio = torch.where(after > 0, before / after, 0.0)[block]
    codes[block] = (codes[block].float() * ratio[:, None, :, None]).round().to(torch.int8)
    scales[block] = after[block]
    each = after[block][..., None]
    codes[block, slot] = torch.where(each > 0, x / each, 0.0).round().to(torch.int8)


def _plain_values(codes, scales, at, kind):
    x = codes.view(-1, *codes.shape[2:])[at].float()
    return (x * scales.view(-1, scales.shape[-1])[at // BLOCK][..., None]).to(kind)


def _plain_write(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    live = (s["positions"] != -1).nonzero()[:, 0]
    position, request = s["positions"][live], s["requests"][live]
    # A turn count is the 32-bit product of the position and the pair's turns.
    turn = position.float()[:, None] * s["turns"]
    angle = (2 * math.pi * (turn - turn.round()))[:, None]
    cosine, sine = angle.cos(), angle.sin()
    q, k, v = (x.view(len(live), -1, dim) for x in
               s["qkv"][live].split([heads * dim, kv * dim, kv * dim], 1))
    s["out"][live] = _plain_turn(_plain_norm(q, s["query_gain"]), cosine,
                                 sine).view(len(live), -1)
    at = _places(s, request, position)
    _plain_append(_plain_turn(_plain_norm(k, s["key_gain"]), cosine, sine), s["keys"],
                  s["key_scales"], at)
    _plain_append(v, s["values"], s["value_scales"], at)
    seen = _places(s, s["seen_requests"], s["seen_positions"])
    return {"query": s["out"],
            "keys": _plain_values(s["keys"], s["key_scales"], seen, torch.float16),
            "values": _plain_values(s["values"], s["value_scales"], seen, torch.float16)}


def _plain_read(s):
    at, kind = _places(s, s["requests"], s["positions"]), TYPES[s["case"]["type"]]
    return {"keys": _plain_values(s["keys"], s["key_scales"], at, kind),
            "values": _plain_values(s["values"], s["value_scales"], at, kind)}


def _plain_attention(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    live = (s["positions"] != -1).nonzero()[:, 0]
    position, request = s["positions"][live].long()[:, None], s["requests"][live]
    window, first = case.get("window", case["most"]), case.get("sinks", 0)
    # The first keys, and those of the window that are not among them.
    key = torch.arange(first + min(window, case["most"]), device="cuda")
    last = key - first - min(window, case["most"]) + 1 + position
    key = torch.where(key < first, key, last)
    seen = torch.where(torch.arange(key.shape[1], device="cuda") < first, key <= position,
                       key >= first)
    key = torch.where(seen, key, position)
    at = _places(s, request[:, None], key)

    def gather(pool, scales):
        x = pool.view(-1, kv, dim)[at].float()
        if scales is not None:
            x *= scales.view(-1, kv)[at // BLOCK][..., None]
        return x.permute(0, 2, 1, 3)

    q = s["query"][live].view(len(live), kv, heads // kv, dim)
    scores = (q @ gather(s["keys"], s["key_scales"]).transpose(2, 3)) * dim ** -0.5
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    out = (weights @ gather(s["values"], s["value_scales"])) / weights.sum(-1, keepdim=True)
    s["out"][live] = out.reshape(len(live), -1)
    return {"out": s["out"]}


_plain = {"write": _plain_write, "read": _plain_read, "attention": _plain_attention,
          "sinks": _plain_attention}


# ---- the same in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read}.get(case["op"], _exact_attention)(case, s)


def _words(tensor):
    return tensor.cpu().numpy().view(np.uint32)


def _exact_keys(case, s, request, first, end):
    """A request's keys and values [first, end) in 64 bits: [key][head][dim] each."""
    slots, table = case["slots"], _words(s["table"])
    pages = torch.from_numpy(table[request, first // slots:-(-end // slots)].astype(np.int64))
    pages, lead = pages.cuda(), first % slots
    found = []
    for pool, scales in ((s["keys"], s["key_scales"]), (s["values"], s["value_scales"])):
        x = pool[pages].double()
        if scales is not None:
            x = x * scales[pages].double().repeat_interleave(BLOCK, 1)[..., None]
        found.append(x.flatten(0, 1)[lead:lead + end - first])
    return found


def _exact_read(case, s):
    found = [_exact_keys(case, s, r, 0, n) for r, n in enumerate(_lengths(case))]
    return {"keys": torch.cat([k for k, _ in found]), "values": torch.cat([v for _, v in found])}


def _exact_write(case, s):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    half, turns = dim // 2, s["turns"].cpu().numpy()
    query = s["out"].double()
    gains = torch.cat([s["query_gain"].expand(heads, dim), s["key_gain"].expand(kv, dim)])
    new = {}
    for row, (request, p) in enumerate(zip(_words(s["requests"]), _words(s["positions"]))):
        if p == NONE:
            continue
        x = s["qkv"][row].double().view(heads + 2 * kv, dim)
        turned = (np.float32(p) * turns).astype(np.float64)
        angle = torch.from_numpy(2 * math.pi * (turned - np.rint(turned))).cuda()
        rotation = torch.complex(angle.cos(), angle.sin())
        n = x[:heads + kv]
        n = n / ((n ** 2).sum(1, keepdim=True) / dim + EPSILON).sqrt() * gains.double()
        z = torch.complex(n[:, :half], n[:, half:]) * rotation
        n = torch.cat([z.real, z.imag], 1)
        query[row] = n[:heads].reshape(-1)
        new[int(request), int(p)] = (n[heads:], x[heads + kv:])
    table, slots, parts = _words(s["table"]), case["slots"], ([], [])
    for request, first, end in _touched(case):
        for b in range(first, end, BLOCK):
            there = [p for p in range(b, min(b + BLOCK, end)) if (request, p) in new]
            page, slot = int(table[request, b // slots]), b % slots
            for which, (pool, scales) in enumerate((("keys", "key_scales"),
                                                    ("values", "value_scales"))):
                codes = s[pool][page, slot:slot + BLOCK].double()
                before = s[scales][page, slot // BLOCK].double()
                rows = torch.stack([new[request, p][which] for p in there])
                need = torch.exp2((rows.abs().amax((0, 2)) / MOST).log2().ceil())
                after = need if there[0] == b else torch.maximum(before, need)
                held = (codes * (before / after)[:, None]).round()
                held[[p - b for p in there]] = (rows / after[:, None]).round()
                parts[which].append((held * after[:, None])[:min(BLOCK, end - b)])
    return {"query": query, "keys": torch.cat(parts[0]), "values": torch.cat(parts[1])}


def _exact_attention(case, s):
    kv, dim = case["kv"], case["dim"]
    group = case["heads"] // kv
    out = s["out"].double()
    for row, (request, p) in enumerate(zip(_words(s["requests"]), _words(s["positions"]))):
        if p == NONE:
            continue
        found = [_exact_keys(case, s, int(request), a, b) for a, b in _held(case, int(p) + 1)]
        keys, values = (torch.cat([x[i] for x in found]) for i in (0, 1))
        for h in range(kv):
            q = s["query"][row].view(kv, group, dim)[h].double()
            weights = torch.softmax(q @ keys[:, h].T / math.sqrt(dim), 1)
            out[row].view(kv, group, dim)[h] = weights @ values[:, h]
    return {"out": out}
