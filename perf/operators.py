"""A decode step of many requests at once: what differs by request, as cases.

Beside the products that all requests share, a layer's step has three
operators that read each request's own data:

  rope       queries and keys normed for each head and turned to their
             request's position, keys and values put into its pages
             (frz_op_rope_paged)
  attention  each row's query over its request's keys, which lie in pages
             anywhere in one pool (frz_op_attention_paged)
  adapters   each row's low-rank adapter beside a shared projection
             (frz_op_adapters)

Where `own` is false, `run` computes them with elementary torch operations in
32 bits; where it is true it calls the library. Keys read, adapters used and
their ranks follow from the case alone, their order and all values from the
seed.
"""
import functools
import math

import numpy as np
import torch

own = False

EPSILON = 1e-6
NONE = 0xFFFFFFFF  # no position, no page, no adapter
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NUMBERS = {"f32": 0, "f16": 1, "bf16": 30}  # GGUF's


def listed():
    return [
        # One reply late in a conversation: a global layer's token.
        {"name": "attention_reply", "op": "attention", "rows": 1, "idle": 0, "least": 5004,
         "most": 5004, "window": 0, "heads": 4, "kv": 1, "dim": 256, "slots": 64, "type": "f16"},
        # Steered replies to one message, a sliding layer's token each.
        {"name": "attention_window", "op": "attention", "rows": 16, "idle": 0, "least": 150,
         "most": 900, "window": 512, "heads": 4, "kv": 1, "dim": 256, "slots": 16,
         "type": "f16"},
        # A full batch of requests, some slots of it empty, over global layers.
        {"name": "attention_batch", "op": "attention", "rows": 64, "idle": 3, "least": 40,
         "most": 8192, "window": 0, "heads": 4, "kv": 1, "dim": 256, "slots": 64, "type": "f16"},
        # A wider model's heads over a BF16 cache, from first tokens to documents.
        {"name": "attention_heads", "op": "attention", "rows": 33, "idle": 1, "least": 1,
         "most": 4001, "window": 0, "heads": 16, "kv": 8, "dim": 128, "slots": 32,
         "type": "bf16"},
        # Few requests over whole books.
        {"name": "attention_long", "op": "attention", "rows": 3, "idle": 0, "least": 98001,
         "most": 131072, "window": 0, "heads": 8, "kv": 4, "dim": 256, "slots": 128,
         "type": "f16"},
        # One reply's token.
        {"name": "rope_reply", "op": "rope", "rows": 1, "idle": 0, "least": 5004, "most": 5004,
         "heads": 4, "kv": 1, "dim": 256, "slots": 64, "type": "f16"},
        # A batch of requests' tokens.
        {"name": "rope_batch", "op": "rope", "rows": 64, "idle": 3, "least": 40, "most": 8192,
         "heads": 4, "kv": 1, "dim": 256, "slots": 64, "type": "f16"},
        # A step nearly full of rows, of a wider model, over a BF16 cache.
        {"name": "rope_heads", "op": "rope", "rows": 509, "idle": 5, "least": 1, "most": 4001,
         "heads": 32, "kv": 8, "dim": 128, "slots": 16, "type": "bf16"},
        # One reply with an adapter on Q, K and V.
        {"name": "adapters_reply", "op": "adapters", "rows": 1, "requests": 1, "count": 8,
         "rank": 16, "inputs": 1152, "outputs": 1536, "type": "f16"},
        # A batch of replies, most with an adapter of their own, beside the gate.
        {"name": "adapters_batch", "op": "adapters", "rows": 48, "requests": 41, "count": 64,
         "rank": 32, "inputs": 1152, "outputs": 6912, "type": "bf16"},
        # Three prompts' rows beside the down product.
        {"name": "adapters_prompts", "op": "adapters", "rows": 333, "requests": 3, "count": 4,
         "rank": 64, "inputs": 6912, "outputs": 1152, "type": "f16"},
        # A whole step of one prompt, a large adapter in F32.
        {"name": "adapters_block", "op": "adapters", "rows": 512, "requests": 1, "count": 2,
         "rank": 128, "inputs": 1152, "outputs": 6912, "type": "f32"},
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    """(query heads, key-value heads, head width)."""
    kv, group = rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 4, 6, 8, 16])
    return kv * group, kv, rng.choice([64, 128, 256, 256])


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rope", "adapters", "adapters"])
    rows = _between(rng, 1, 512)
    if op == "adapters":
        requests = rng.randint(1, min(rows, 64))
        kind = rng.choice(["f32", "f16", "f16", "bf16"])
        wide, narrow = 8 * _between(rng, 16, 1024), 8 * _between(rng, 16, 256)
        inputs, outputs = rng.choice([(wide, narrow), (narrow, wide)])
        return {"op": op, "rows": rows, "requests": requests,
                "count": requests + rng.randint(0, 8), "rank": 8 * _between(rng, 1, 16),
                "inputs": inputs, "outputs": outputs - rng.randint(0, 7), "type": kind}
    heads, kv, dim = _heads(rng)
    # No more keys in all than the largest listed case reads: 3 x 131,072 of 4 x 256 values.
    cap = max(2, min(131072, 300_000_000 // (rows * kv * dim)))
    most = max(_between(rng, 1, cap), _between(rng, 1, cap))
    case = {"op": op, "rows": rows, "idle": rng.randint(0, rows // 8),
            "least": max(1, int(most * rng.uniform(0.01, 1))), "most": most, "heads": heads,
            "kv": kv, "dim": dim, "slots": rng.choice([16, 16, 32, 48, 64, 128, 256]),
            "type": rng.choice(["f16", "f16", "bf16"])}
    if op == "attention":
        case["window"] = rng.choice([0, 0, 512, rng.randint(1, 1500)])
    return case


# ---- what a case's rows are ----------------------------------------------------------


def _lengths(case):
    """Keys of each working row's request, its own among them, from least to most."""
    n = case["rows"] - case["idle"]
    if n == 1:
        return [case["most"]]
    ratio = case["most"] / case["least"]
    return [int(round(case["least"] * ratio ** (i / (n - 1)))) for i in range(n)]


def _read(case, length):
    return min(length, case["window"] or length)


def _requests(case):
    """(rows, rank) of each request's adapter; the first of several requests has none."""
    n, rows = case["requests"], case["rows"]
    bounds = [i * rows // n for i in range(n + 1)]
    sizes = [b - a for a, b in zip(bounds, bounds[1:])]
    ranks = [case["rank"] - (5 * i) % max(1, case["rank"] // 2) for i in range(n)]
    return [(size, 0 if n > 4 and i == 0 else rank)
            for i, (size, rank) in enumerate(zip(sizes, ranks))]


def work(case):
    rows = case["rows"]
    if case["op"] == "adapters":
        k, n = case["inputs"], case["outputs"]
        each = TYPES[case["type"]].itemsize
        live = [(size, rank) for size, rank in _requests(case) if rank]
        return {"bytes": float(sum(rank * (k + n) * each for _, rank in live)
                               + 4 * (rows * (2 * n + 1) + sum(size for size, _ in live) * k)),
                "flops": float(sum(2 * size * rank * (k + n) for size, rank in live))}
    lengths, dim = _lengths(case), case["dim"]
    queries = len(lengths) * case["heads"] * dim
    if case["op"] == "rope":
        keys = len(lengths) * case["kv"] * dim
        return {"bytes": float(4 * 2 * queries + (4 + 2) * 2 * keys + 12 * rows),
                "flops": float(9 * (queries + keys))}
    keys = sum(_read(case, n) for n in lengths)
    pages = sum(-(-n // case["slots"]) for n in lengths)
    return {"bytes": float(keys * case["kv"] * dim * 4 + 4 * 2 * queries + 4 * pages + 8 * rows),
            "flops": float(4 * keys * case["heads"] * dim)}


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


def _paged(case, seed):
    """The pool, every request's pages in no order, and the rows' requests and positions."""
    rng, gen = np.random.default_rng(seed), _random(seed)
    rows, slots, kind = case["rows"], case["slots"], TYPES[case["type"]]
    lengths = _lengths(case)
    held = [-(-n // slots) for n in lengths]
    pages = sum(held) + 3
    order = rng.permutation(pages)
    table = np.full((rows, max(held)), NONE, dtype=np.uint32)
    at = 0
    for request, n in enumerate(held):
        table[request, :n] = order[at:at + n]
        at += n
    # The batch's rows in no order, the idle ones among them.
    position = np.full(rows, NONE, dtype=np.uint32)
    request = np.arange(rows, dtype=np.uint32)
    position[:len(lengths)] = np.asarray(lengths, dtype=np.uint32) - 1
    shuffled = rng.permutation(rows)
    shape = (pages, slots, case["kv"], case["dim"])
    return {"table": _unsigned(table), "requests": _unsigned(request[shuffled]),
            "positions": _unsigned(position[shuffled]),
            "keys": _normal(gen, *shape, kind=kind), "values": _normal(gen, *shape, kind=kind)}


def prepare(case, seed):
    s, gen = {"case": case}, _random(seed + 1)
    if case["op"] == "adapters":
        rng = np.random.default_rng(seed)
        kind, k, n, rank = TYPES[case["type"]], case["inputs"], case["outputs"], case["rank"]
        ids = rng.permutation(case["count"])
        which, ranks = [], np.full(case["count"], rank, dtype=np.uint32)
        for i, (size, r) in enumerate(_requests(case)):
            which += [int(ids[i]) if r else NONE] * size
            if r:
                ranks[ids[i]] = r
        s.update(which=_unsigned(which), ranks=_unsigned(ranks),
                 scales=0.5 + torch.rand(case["count"], generator=gen, device="cuda"),
                 down=(_normal(gen, case["count"], rank, k) / math.sqrt(k)).to(kind),
                 up=(_normal(gen, case["count"], n, rank) / math.sqrt(rank)).to(kind),
                 x=_normal(gen, case["rows"], k), y=torch.empty(case["rows"], _even(n),
                                                                device="cuda"),
                 base=_normal(gen, case["rows"], _even(n)))
        return s
    rows, heads, kv, dim = case["rows"], case["heads"], case["kv"], case["dim"]
    s.update(_paged(case, seed))
    if case["op"] == "rope":
        # One product gives a row's queries, keys and values side by side.
        s.update(qkv=1.5 * _normal(gen, rows, (heads + 2 * kv) * dim), turns=_turns(dim),
                 query_gain=1 + 0.1 * _normal(gen, dim), key_gain=1 + 0.1 * _normal(gen, dim))
    else:
        s["query"] = 1.5 * _normal(gen, rows, heads * dim)
    s["out"] = torch.zeros(rows, heads * dim, device="cuda")
    return s


def _even(n):
    """Floats a row of outputs takes: whole 16-byte pieces."""
    return -(-n // 4) * 4


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
    case = s["case"]
    return fz.Pages(s["keys"].data_ptr(), s["values"].data_ptr(), NUMBERS[case["type"]],
                    case["kv"], case["dim"], case["slots"], s["keys"].shape[0],
                    s["keys"].stride(0), s["table"].data_ptr(), s["table"].shape[0],
                    s["table"].shape[1])


def _library_rope(s):
    fz, check, lib, device = _frizzle()
    case, qkv = s["case"], s["qkv"]
    width = qkv.shape[1]
    at, q, k = qkv.data_ptr(), case["heads"] * case["dim"], case["kv"] * case["dim"]
    check(lib.frz_op_rope_paged(
        device.handle, _pages(fz, s), s["requests"].data_ptr(), s["positions"].data_ptr(),
        s["turns"].data_ptr(), s["query_gain"].data_ptr(), s["key_gain"].data_ptr(), at,
        at + 4 * q, at + 4 * (q + k), width, width, s["out"].data_ptr(), q, case["heads"],
        EPSILON, case["rows"]))
    return {"query": s["out"], "keys": s["keys"], "values": s["values"]}


def _library_attention(s):
    fz, check, lib, device = _frizzle()
    case, width = s["case"], s["query"].shape[1]
    check(lib.frz_op_attention_paged(
        device.handle, _pages(fz, s), s["requests"].data_ptr(), s["positions"].data_ptr(),
        s["query"].data_ptr(), width, s["out"].data_ptr(), width, case["heads"],
        case["window"] or NONE, case["dim"] ** -0.5, case["rows"]))
    return {"out": s["out"]}


def _library_adapters(s):
    fz, check, lib, device = _frizzle()
    case, y = s["case"], s["y"]
    adapters = fz.Adapters(NUMBERS[case["type"]], case["count"], case["rank"], case["inputs"],
                           case["outputs"], s["down"].data_ptr(), s["up"].data_ptr(),
                           s["ranks"].data_ptr(), s["scales"].data_ptr())
    check(lib.frz_op_adapters(
        device.handle, adapters, s["which"].data_ptr(), s["x"].data_ptr(), case["inputs"],
        s["base"].data_ptr(), s["base"].shape[1], y.data_ptr(), y.shape[1], case["rows"]))
    return {"y": y[:, :case["outputs"]]}


_library = {"rope": _library_rope, "attention": _library_attention,
            "adapters": _library_adapters}


def _plain_norm(x, gain):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON) * gain


def _plain_turn(x, cosine, sine):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cosine - b * sine, a * sine + b * cosine], -1)


def _plain_rope(s):
    case = s["case"]
    rows, heads, kv, dim = case["rows"], case["heads"], case["kv"], case["dim"]
    live = (s["positions"] != -1).nonzero()[:, 0]
    position, request = s["positions"][live].long(), s["requests"][live].long()
    # A turn count is the 32-bit product of the position and the pair's turns.
    turn = position.float()[:, None] * s["turns"]
    angle = (2 * math.pi * (turn - turn.round()))[:, None]
    cosine, sine = angle.cos(), angle.sin()
    q, k, v = (x.view(len(live), -1, dim) for x in
               s["qkv"][live].split([heads * dim, kv * dim, kv * dim], 1))
    s["out"][live] = _plain_turn(_plain_norm(q, s["query_gain"]), cosine,
                                 sine).view(len(live), -1)
    page = s["table"][request, position // case["slots"]].long()
    slot = position % case["slots"]
    kind = s["keys"].dtype
    s["keys"][page, slot] = _plain_turn(_plain_norm(k, s["key_gain"]), cosine, sine).to(kind)
    s["values"][page, slot] = v.to(kind)
    return {"query": s["out"], "keys": s["keys"], "values": s["values"]}


def _plain_attention(s):
    case = s["case"]
    heads, kv, dim, slots = case["heads"], case["kv"], case["dim"], case["slots"]
    live = (s["positions"] != -1).nonzero()[:, 0]
    position, request = s["positions"][live].long(), s["requests"][live].long()
    span = _read(case, case["most"])
    first = (position - span + 1).clamp(min=0)[:, None]
    key = first + torch.arange(span, device="cuda")
    seen = key <= position[:, None]
    key = key.minimum(position[:, None])
    at = s["table"][request[:, None], key // slots].long() * slots + key % slots

    def gather(pool):
        return pool.view(-1, kv, dim)[at].permute(0, 2, 1, 3).float()

    q = s["query"][live].view(len(live), kv, heads // kv, dim)
    scores = (q @ gather(s["keys"]).transpose(2, 3)) * dim ** -0.5
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    out = (weights @ gather(s["values"])) / weights.sum(-1, keepdim=True)
    s["out"][live] = out.reshape(len(live), -1)
    return {"out": s["out"]}


def _plain_adapters(s):
    case, rank = s["case"], s["case"]["rank"]
    # Every adapter beside every row, and each row its own of them.
    ids = torch.arange(case["count"], device="cuda")
    mine = s["which"][:, None] == ids
    held = torch.arange(rank, device="cuda") < s["ranks"][:, None]
    low = s["x"] @ s["down"].float().flatten(0, 1).T
    low = low.view(-1, case["count"], rank) * (mine[:, :, None] & held) * s["scales"][:, None]
    added = low.flatten(1) @ s["up"].float().permute(0, 2, 1).reshape(-1, case["outputs"])
    return {"y": s["base"][:, :case["outputs"]] + added}


_plain = {"rope": _plain_rope, "attention": _plain_attention, "adapters": _plain_adapters}


# ---- the same in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attention": _exact_attention,
            "adapters": _exact_adapters}[case["op"]](case, s)


def _words(tensor):
    return tensor.cpu().numpy().view(np.uint32)


def _exact_rope(case, s):
    heads, kv, dim, slots = case["heads"], case["kv"], case["dim"], case["slots"]
    half, turns, kind = dim // 2, s["turns"].cpu().numpy(), s["keys"].dtype
    query, keys, values = s["out"].double(), s["keys"].double(), s["values"].double()
    gains = torch.cat([s["query_gain"].expand(heads, dim), s["key_gain"].expand(kv, dim)])
    table = _words(s["table"])
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
        page = int(table[request, p // slots])
        keys[page, p % slots] = n[heads:].to(kind).double()
        values[page, p % slots] = x[heads + kv:].to(kind).double()
    return {"query": query, "keys": keys, "values": values}


def _exact_attention(case, s):
    kv, dim, slots = case["kv"], case["dim"], case["slots"]
    group = case["heads"] // kv
    out = s["out"].double()
    table = _words(s["table"])
    for row, (request, p) in enumerate(zip(_words(s["requests"]), _words(s["positions"]))):
        if p == NONE:
            continue
        first = max(0, int(p) + 1 - (case["window"] or int(p) + 1))
        pages = table[request, first // slots:int(p) // slots + 1].astype(np.int64)
        lead = first % slots
        pages = torch.from_numpy(pages).cuda()
        count = int(p) + 1 - first
        for h in range(kv):
            k = s["keys"][pages, :, h].reshape(-1, dim)[lead:lead + count].double()
            v = s["values"][pages, :, h].reshape(-1, dim)[lead:lead + count].double()
            q = s["query"][row].view(kv, group, dim)[h].double()
            weights = torch.softmax(q @ k.T / math.sqrt(dim), 1)
            out[row].view(kv, group, dim)[h] = weights @ v
    return {"out": out}


def _exact_adapters(case, s):
    y = s["base"][:, :case["outputs"]].double()
    which, ranks = _words(s["which"]), _words(s["ranks"])
    for a in sorted(set(which.tolist()) - {NONE}):
        rows, r = torch.from_numpy(np.flatnonzero(which == a)).cuda(), int(ranks[a])
        low = s["x"][rows].double() @ s["down"][a, :r].double().T
        y[rows] += float(s["scales"][a]) * (low @ s["up"][a, :, :r].double().T)
    return {"y": y}
