"""Decode steps over long caches, whose rows attention cuts into parts and joins from the
handle's workspace: in captured graphs that share it, on torch's streams and through two
handles at once."""
import threading

import numpy as np
import pytest
import torch

import frizzle_amd as fz
from _batch import BF16, F16, NONE
from _cache8 import I8, Paged8, exact
from frizzle_amd import _lib

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, SLOTS, WIDTH = 8, 2, 128, 32, 512
OUT, SIZE = HEADS * DIM, KV * DIM
QKV = OUT + 2 * SIZE
STEPS = 24
SEEN = pytest.mark.parametrize("window,sinks", [(NONE, 0), (3000, 70)])
TYPES = {I8: torch.int8, F16: torch.float16, BF16: torch.bfloat16}


class Requests:
    """Torch tensors of requests that hold some keys and get a token each a step."""

    def __init__(self, lengths, seed, fmt, window, sinks):
        # A row of these is cut whatever it holds: past 36 blocks, and 8,192 values a head.
        assert (min(window, WIDTH * SLOTS) // 32) * DIM > 8192
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths, self.rows, self.fmt = lengths, len(lengths), fmt
        self.window, self.sinks = window, sinks
        held = [-(-(n + STEPS) // SLOTS) for n in lengths]
        self.count = sum(held)
        order = torch.randperm(self.count, generator=g, device="cuda").int()
        self.table = torch.full((self.rows, WIDTH), -1, dtype=torch.int32, device="cuda")
        at = 0
        for row, n in enumerate(held):
            self.table[row, :n] = order[at:at + n]
            at += n
        shape = (self.count, SLOTS, KV, DIM)
        self.pools = [(torch.randn(shape, generator=g, device="cuda") * (30 if fmt == I8 else 1))
                      .clamp(-127, 127).round_(decimals=0 if fmt == I8 else 3).to(TYPES[fmt])
                      for _ in range(2)]
        self.scales = [torch.exp2(torch.randint(-6, -3, (self.count, SLOTS // 16, KV),
                                                generator=g, device="cuda").float())
                       for _ in range(2)]
        self.start = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.positions = self.start.clone()
        self.turns = torch.from_numpy(fz.rope_turns(1e4, DIM)).cuda()
        self.gains = [1 + 0.1 * torch.randn(DIM, generator=g, device="cuda") for _ in range(2)]
        self.tokens = torch.randn(STEPS, self.rows, QKV, generator=g, device="cuda")
        self.qkv = torch.zeros(self.rows, QKV, device="cuda")
        self.query = torch.zeros(self.rows, OUT, device="cuda")
        self.out = torch.zeros(self.rows, OUT, device="cuda")

    def enqueue(self, device):
        lib, h, at = fz.load(), device.handle, self.qkv.data_ptr()
        pages = fz.Pages(self.pools[0].data_ptr(), self.pools[1].data_ptr(), self.fmt, KV, DIM,
                         SLOTS, self.count, SLOTS * SIZE, self.table.data_ptr(), self.rows, WIDTH,
                         self.scales[0].data_ptr(), self.scales[1].data_ptr(), SLOTS // 16 * KV)
        _lib.check(lib.frz_op_rope_paged(
            h, pages, None, self.positions.data_ptr(), self.turns.data_ptr(),
            self.gains[0].data_ptr(), self.gains[1].data_ptr(), at, at + 4 * OUT,
            at + 4 * (OUT + SIZE), QKV, QKV, self.query.data_ptr(), OUT, HEADS, 1e-6, self.rows))
        _lib.check(lib.frz_op_attention_paged_sinks(
            h, pages, None, self.positions.data_ptr(), self.query.data_ptr(), OUT,
            self.out.data_ptr(), OUT, HEADS, self.window, self.sinks, DIM ** -0.5, self.rows))

    def set(self, i):
        self.qkv.copy_(self.tokens[i])
        torch.add(self.start, i, out=self.positions)

    def outputs(self):
        return self.query.clone(), self.out.clone()

    def check(self, i):
        """The step's attention over the cache of 8 bits as it is."""
        if self.fmt != I8:
            return
        want, far = exact(Host(self), [n + i for n in self.lengths], self.query.cpu().numpy(),
                          HEADS, self.window, DIM ** -0.5, sinks=self.sinks)
        got = self.out.cpu().numpy()
        for row in range(self.rows):
            assert (abs(got[row] - want[row]) <= far[row]).all(), (i, row)


class Host(Paged8):
    """The cache as _cache8.exact reads it, from torch's copies."""

    def __init__(self, r):
        self.kv, self.dim, self.slots, self.pages = KV, DIM, SLOTS, r.count
        self.table = r.table.cpu().numpy().view(np.uint32)
        self.parts = [[x.cpu().numpy() for x in p] for p in (r.pools, r.scales)]

    def codes(self):
        return self.parts[0]

    def scales(self):
        return self.parts[1]


def same(a, b):
    return all(torch.equal(x.view(torch.int32), y.view(torch.int32)) for x, y in zip(a, b))


# Rows of many parts, of a few and of one; the second set's joins are others and more.
FIRST, SECOND = [5000, 40, 900], [70, 3100, 9000, 12, 2000, 333, 4096]


@SEEN
@pytest.mark.parametrize("fmt", [I8, F16, BF16])
def test_graphs_that_share_the_workspace(fmt, window, sinks):
    # Each replay against the same step run eagerly from the same cache through a handle
    # of its own, whose workspace is another.
    stream = torch.cuda.Stream()
    devices = [fz.Device(0, stream=stream.cuda_stream) for _ in range(2)]
    try:
        with torch.cuda.stream(stream):
            sets = [[Requests(n, seed, fmt, window, sinks) for _ in range(2)]
                    for seed, n in enumerate((FIRST, SECOND))]
            graphs = []
            for replayed, eager in sets:
                for r, device in ((replayed, devices[0]), (eager, devices[1])):
                    r.set(0)
                    r.enqueue(device)
                stream.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    replayed.enqueue(devices[0])
                graphs.append(g)
            got, want = [], []
            for i in range(STEPS):
                for r in sum(sets, []):
                    r.set(i)
                # In turn the one or the other first, so that each finds both in the workspace.
                for k in ((0, 1), (1, 0), (0, 0, 1), (1, 1, 0))[i % 4]:
                    graphs[k].replay()
                for _, eager in sets:
                    eager.enqueue(devices[1])
                got.append([r.outputs() for r, _ in sets])
                want.append([r.outputs() for _, r in sets])
                if i % 5 == 0:
                    stream.synchronize()
            stream.synchronize()
        for i in range(STEPS):
            assert all(same(g, w) for g, w in zip(got[i], want[i])), i
        for replayed, _ in sets:
            replayed.check(STEPS - 1)
        del graphs
    finally:
        torch.cuda.synchronize()
        for d in devices:
            d.close()


@SEEN
@pytest.mark.parametrize("own", [False, True])
def test_steps_in_order_with_torch(own, window, sinks):
    stream = torch.cuda.Stream() if own else torch.cuda.default_stream()
    device = fz.Device(0, stream=stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            sets = [Requests(n, 5 + i, I8, window, sinks) for i, n in enumerate((FIRST, SECOND))]
            for i in range(STEPS):
                for r in sets:
                    r.set(i)
                    r.enqueue(device)
                    r.qkv.fill_(float("nan"))
                if i in (0, 9, STEPS - 1):
                    stream.synchronize()
                    for r in sets:
                        r.check(i)
    finally:
        torch.cuda.synchronize()
        device.close()


@SEEN
def test_two_handles_at_once(window, sinks):
    sets = [Requests(n, 8 + i, I8, window, sinks) for i, n in enumerate((FIRST, SECOND))]
    torch.cuda.synchronize()
    devices = [fz.Device(0) for _ in sets]
    failed = []

    def work(r, device):
        # Through the handle, whose stream is ordered with no other.
        lib = fz.load()
        try:
            for i in range(STEPS):
                _lib.check(lib.frz_copy(device.handle, r.qkv.data_ptr(), r.tokens[i].data_ptr(),
                                        4 * r.rows * QKV))
                at = np.array(r.lengths, np.uint32) + i
                _lib.check(lib.frz_write(device.handle, r.positions.data_ptr(), at.ctypes.data,
                                         at.nbytes))
                r.enqueue(device)
            device.sync()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    try:
        threads = [threading.Thread(target=work, args=x) for x in zip(sets, devices)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failed
        for r in sets:
            r.check(STEPS - 1)
    finally:
        torch.cuda.synchronize()
        for d in devices:
            d.close()
