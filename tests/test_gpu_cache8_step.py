"""A decode step's ops over a cache of 8 bits one after another, as a program calls them:
rope into pages, attention over first keys and a window, keys read back; on torch's
streams, in captured graphs, through two handles at once."""
import threading

import numpy as np
import pytest
import torch

import frizzle_amd as fz
from _batch import F32, rope_exact
from _cache8 import I8, Paged8, exact
from frizzle_amd import _lib

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, SLOTS, WIDTH = 8, 2, 128, 32, 9
OUT, SIZE = HEADS * DIM, KV * DIM
QKV = OUT + 2 * SIZE
WINDOW, SINKS = 40, 5


class Requests:
    """Torch tensors of some requests, a token each a step."""

    def __init__(self, rows, seed, steps=1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rows, pages = rows, rows * WIDTH
        order = torch.randperm(pages, generator=g, device="cuda")
        self.table = order.view(rows, WIDTH).int()
        self.codes = [torch.full((pages, SLOTS, KV, DIM), 99, dtype=torch.int8, device="cuda")
                      for _ in range(2)]
        self.scales = [torch.full((pages, SLOTS // 16, KV), float("nan"), device="cuda")
                       for _ in range(2)]
        self.positions = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.turns = torch.from_numpy(fz.rope_turns(1e4, DIM)).cuda()
        self.gains = [1 + 0.1 * torch.randn(DIM, generator=g, device="cuda") for _ in range(2)]
        self.tokens = torch.randn(steps, rows, QKV, generator=g, device="cuda")
        self.qkv = torch.zeros(rows, QKV, device="cuda")
        self.query = torch.zeros(rows, OUT, device="cuda")
        self.out = torch.zeros(rows, OUT, device="cuda")
        self.read = torch.zeros(2, rows, SIZE, device="cuda")

    def pages(self):
        return fz.Pages(self.codes[0].data_ptr(), self.codes[1].data_ptr(), I8, KV, DIM, SLOTS,
                        self.rows * WIDTH, SLOTS * SIZE, self.table.data_ptr(), self.rows, WIDTH,
                        self.scales[0].data_ptr(), self.scales[1].data_ptr(), SLOTS // 16 * KV)

    def enqueue(self, device):
        lib, h, pages, at = fz.load(), device.handle, self.pages(), self.qkv.data_ptr()
        _lib.check(lib.frz_op_rope_paged(
            h, pages, None, self.positions.data_ptr(), self.turns.data_ptr(),
            self.gains[0].data_ptr(), self.gains[1].data_ptr(), at, at + 4 * OUT,
            at + 4 * (OUT + SIZE), QKV, QKV, self.query.data_ptr(), OUT, HEADS, 1e-6, self.rows))
        _lib.check(lib.frz_op_attention_paged_sinks(
            h, pages, None, self.positions.data_ptr(), self.query.data_ptr(), OUT,
            self.out.data_ptr(), OUT, HEADS, WINDOW, SINKS, DIM ** -0.5, self.rows))
        _lib.check(lib.frz_op_read_paged(h, pages, None, self.positions.data_ptr(), F32,
                                         self.read[0].data_ptr(), self.read[1].data_ptr(), SIZE,
                                         self.rows))

    def set(self, i):
        self.qkv.copy_(self.tokens[i])
        self.positions.fill_(i)

    def outputs(self):
        return [x.clone() for x in (self.query, self.out, self.read, *self.codes, *self.scales)]


class Host(Paged8):
    """The cache as _cache8.exact reads it, from torch's copies."""

    def __init__(self, r, codes, scales):
        self.kv, self.dim, self.slots, self.pages = KV, DIM, SLOTS, r.rows * WIDTH
        self.table = r.table.cpu().numpy().astype(np.uint32)
        self.held_codes = [c.cpu().numpy() for c in codes]
        self.held_scales = [s.cpu().numpy() for s in scales]

    def codes(self):
        return self.held_codes

    def scales(self):
        return self.held_scales


def check(r, i, outputs):
    """A step's outputs: attention and reads over the cache as it is, the cache near the
    keys and values that the step brought."""
    query, out, read, *cache = outputs
    host = Host(r, cache[:2], cache[2:])
    q = query.cpu().numpy()
    want, far = exact(host, [i] * r.rows, q, HEADS, WINDOW, DIM ** -0.5, sinks=SINKS)
    got, back = out.cpu().numpy(), read.cpu().numpy()
    token = r.tokens[i].cpu().numpy()
    for row in range(r.rows):
        assert (abs(got[row] - want[row]) <= far[row]).all(), (i, row)
        keys, values = (x[0] for x in host.held(row, [i]))
        assert np.array_equal(back[0, row], keys.reshape(-1).astype(np.float32))
        assert np.array_equal(back[1, row], values.reshape(-1).astype(np.float32))
        turned, size = rope_exact(token[row, OUT:OUT + SIZE].reshape(KV, DIM),
                                  r.gains[1].cpu().numpy(), r.turns.cpu().numpy(), i)
        page, slot = host.page(row, i), i % SLOTS
        ks, vs = (s[page, slot // 16][:, None] for s in host.scales())
        assert (abs(keys - turned) <= 0.5 * ks + 2.0 ** -18 * size.max()).all()
        assert (abs(values - token[row, OUT + SIZE:].reshape(KV, DIM)) <= 0.5 * vs).all()


@pytest.fixture(params=["default", "own"])
def stream(request):
    yield torch.cuda.default_stream() if request.param == "default" else torch.cuda.Stream()
    torch.cuda.synchronize()


def test_replies_grow_in_order_with_torch(stream):
    steps = 100  # past the window, over several pages
    device = fz.Device(0, stream=stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            r = Requests(3, 1, steps)
            kept = {}
            for i in range(steps):
                r.set(i)
                r.enqueue(device)
                if i in (0, 1, 15, 16, 31, 44, 45, 46, 64, 99):
                    kept[i] = r.outputs()
                r.qkv.fill_(float("nan"))
            device.sync()
        for i, outputs in kept.items():
            check(r, i, outputs)
    finally:
        torch.cuda.synchronize()
        device.close()


def test_a_graph_replayed_beside_eager_steps():
    # Every replay against the same step run eagerly from the same cache; a second graph
    # of the handle's, over other requests, shares the workspace in between.
    steps, stream = 60, torch.cuda.Stream()
    device = fz.Device(0, stream=stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            a, b, eager = Requests(3, 1, steps), Requests(5, 2, steps), Requests(3, 1, steps)
            graphs = []
            for r in (a, b):
                r.set(0)
                r.enqueue(device)
                stream.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    r.enqueue(device)
                graphs.append(g)
            got, want = [], []
            for i in range(steps):
                a.set(i)
                b.set(i)
                graphs[0].replay()
                graphs[1].replay()
                eager.set(i)
                eager.enqueue(device)
                got.append(a.outputs())
                want.append(eager.outputs())
                if i % 7 == 0:
                    stream.synchronize()
            stream.synchronize()
        for i, (g, w) in enumerate(zip(got, want)):
            for x, y in zip(g, w):
                assert torch.equal(torch.nan_to_num(x.float()), torch.nan_to_num(y.float())), i
        check(a, steps - 1, got[-1])
        check(b, steps - 1, b.outputs())
        del graphs
    finally:
        torch.cuda.synchronize()
        device.close()


def test_two_handles_at_once():
    steps = 50
    sets = [Requests(3 + i, 4 + i, steps) for i in range(2)]
    torch.cuda.synchronize()
    devices = [fz.Device(0) for _ in sets]
    failed = []

    def work(r, device):
        try:
            for i in range(steps):
                device_set(r, device, i)
                r.enqueue(device)
            device.sync()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    def device_set(r, device, i):
        # Through the handle, whose stream is ordered with no other.
        lib = fz.load()
        _lib.check(lib.frz_copy(device.handle, r.qkv.data_ptr(), r.tokens[i].data_ptr(),
                                4 * r.rows * QKV))
        at = np.full(r.rows, i, np.uint32)
        _lib.check(lib.frz_write(device.handle, r.positions.data_ptr(), at.ctypes.data, at.nbytes))

    try:
        threads = [threading.Thread(target=work, args=x) for x in zip(sets, devices)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failed
        for r in sets:
            check(r, steps - 1, r.outputs())
    finally:
        torch.cuda.synchronize()
        for d in devices:
            d.close()


def test_no_position_leaves_everything_as_it_is():
    device = fz.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    try:
        r = Requests(4, 9)
        r.positions.fill_(-1)
        before = r.outputs()
        r.enqueue(device)
        for x, y in zip(before, r.outputs()):
            assert torch.equal(torch.nan_to_num(x.float()), torch.nan_to_num(y.float()))
    finally:
        torch.cuda.synchronize()
        device.close()
