"""The ops over a step of many requests on a stream of the caller's
(frz_open_on): in order with torch's work there, with no wait of the host
between, and in a captured graph."""
import numpy as np
import pytest
import torch

import frizzle_amd as fz
import test_gpu_batch_adapters as layer
from _batch import F16, NONE, adapters_exact, attention_exact, rope_exact
from frizzle_amd import _lib

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, SLOTS, ROWS, PAGES = 4, 1, 256, 16, 5, 7
HIDDEN, RANK, COUNT = 64, 16, 3
OUT = HEADS * DIM
QKV = (HEADS + 2 * KV) * DIM


@pytest.fixture(params=["default", "own"])
def stream(request):
    yield torch.cuda.default_stream() if request.param == "default" else torch.cuda.Stream()
    torch.cuda.synchronize()


class Step:
    """Torch tensors of one step: adapters beside Q/K/V, rope into pages,
    attention."""

    def __init__(self):
        self.table = torch.tensor([[3, 1], [6, -1], [0, 2], [5, -1], [4, -1]], dtype=torch.int32,
                                  device="cuda")
        self.positions = torch.tensor([20, 9, 31, -1, 0], dtype=torch.int32, device="cuda")
        self.which = torch.tensor([2, 0, -1, 1, 1], dtype=torch.int32, device="cuda")
        self.turns = torch.from_numpy(fz.rope_turns(1e4, DIM)).cuda()
        self.gain = torch.ones(DIM, device="cuda")
        self.down = (torch.randn(COUNT, RANK, HIDDEN, device="cuda") / 8).half()
        self.up = (torch.randn(COUNT, QKV, RANK, device="cuda") / 4).half()
        self.keys = torch.randn(PAGES, SLOTS, KV, DIM, device="cuda").half()
        self.values = torch.randn(PAGES, SLOTS, KV, DIM, device="cuda").half()
        self.x = torch.zeros(ROWS, HIDDEN, device="cuda")
        self.base = torch.zeros(ROWS, QKV, device="cuda")
        self.qkv = torch.zeros(ROWS, QKV, device="cuda")
        self.out = torch.zeros(ROWS, OUT, device="cuda")

    def enqueue(self, device):
        lib, h = fz.load(), device.handle
        pool = fz.Adapters(F16, COUNT, RANK, HIDDEN, QKV, self.down.data_ptr(),
                           self.up.data_ptr(), None, None)
        pages = fz.Pages(self.keys.data_ptr(), self.values.data_ptr(), F16, KV, DIM, SLOTS, PAGES,
                         SLOTS * KV * DIM, self.table.data_ptr(), ROWS, 2)
        _lib.check(lib.frz_op_adapters(h, pool, self.which.data_ptr(), self.x.data_ptr(), HIDDEN,
                                       self.base.data_ptr(), QKV, self.qkv.data_ptr(), QKV, ROWS))
        q = self.qkv.data_ptr()
        _lib.check(lib.frz_op_rope_paged(
            h, pages, None, self.positions.data_ptr(), self.turns.data_ptr(),
            self.gain.data_ptr(), self.gain.data_ptr(), q, q + 4 * OUT, q + 4 * (OUT + KV * DIM),
            QKV, QKV, q, QKV, HEADS, 1e-6, ROWS))
        _lib.check(lib.frz_op_attention_paged(
            h, pages, None, self.positions.data_ptr(), q, QKV, self.out.data_ptr(), OUT, HEADS,
            NONE, 1 / 16, ROWS))


class Values:
    """What attention_exact reads of a batch, from torch's copies."""

    def __init__(self, step, keys, values):
        self.kv, self.dim = KV, DIM
        self.table = step.table.cpu().numpy()
        self.keys, self.values = keys.double().cpu().numpy(), values.double().cpu().numpy()

    def rows(self, request, first, end):
        at = [(self.table[request, j // SLOTS], j % SLOTS) for j in range(first, end)]
        p, s = [a[0] for a in at], [a[1] for a in at]
        return self.keys[p, s], self.values[p, s]


class Host:
    fmt = F16
    count, rank = COUNT, RANK
    scales = None

    def __init__(self, step):
        self.down = step.down.cpu().numpy().view(np.uint16)
        self.up = step.up.cpu().numpy().view(np.uint16)

    def own(self, a):
        return RANK

    cols, rows = HIDDEN, QKV


def check(step, x, base, qkv, out, keys, values):
    which = [w if w >= 0 else NONE for w in step.which.tolist()]
    full, _ = adapters_exact(Host(step), which, x.cpu().numpy(), base.cpu().numpy())
    positions = [p if p >= 0 else NONE for p in step.positions.tolist()]
    got, turns, one = qkv.cpu().numpy(), step.turns.cpu().numpy(), np.ones(DIM, np.float32)
    for r, p in enumerate(positions):
        if p == NONE:
            continue
        want, size = rope_exact(full[r, :OUT].reshape(HEADS, DIM), one, turns, p)
        assert abs(got[r, :OUT].reshape(HEADS, DIM) - want).max() <= 4e-6 * size.max(), r
    want, far = attention_exact(Values(step, keys, values), positions, got[:, :OUT], HEADS, NONE,
                                1 / 16)
    o = out.cpu().numpy()
    for r, p in enumerate(positions):
        if p == NONE:
            assert (o[r] == 0).all()
        else:
            assert (abs(o[r] - want[r]) <= far[r]).all(), r


def test_in_order_with_torch(stream):
    """Inputs that torch has yet to write when the ops are called, outputs that
    torch copies at once and inputs that it then overwrites: three steps, and
    nothing waits until their end."""
    device = fz.Device(0, stream=stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            torch.manual_seed(3)
            step, slow = Step(), torch.randn(4096, 4096, device="cuda")
            kept = []
            for i in range(3):
                for _ in range(8):  # milliseconds of work ahead of the inputs
                    slow = slow @ slow
                    slow = slow / slow.norm()
                x, base = torch.randn(ROWS, HIDDEN, device="cuda"), torch.randn(ROWS, QKV,
                                                                               device="cuda")
                step.x.copy_(x)
                step.base.copy_(base)
                step.enqueue(device)
                kept.append((x, base, step.qkv.clone(), step.out.clone(), step.keys.clone(),
                             step.values.clone()))
                step.x.fill_(7.0)
                step.base.fill_(7.0)
                step.qkv.fill_(7.0)
            device.sync()
        for k in kept:
            check(step, *k)
    finally:
        device.close()


def test_in_a_captured_graph():
    stream = torch.cuda.Stream()
    device = fz.Device(0, stream=stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            torch.manual_seed(4)
            step = Step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        # The handle's first calls are the captured ones.
        with torch.cuda.graph(graph, stream=stream):
            step.enqueue(device)
        for i in range(4):
            with torch.cuda.stream(stream):
                x, base = torch.randn(ROWS, HIDDEN, device="cuda"), torch.randn(ROWS, QKV,
                                                                               device="cuda")
                step.x.copy_(x)
                step.base.copy_(base)
                step.out.zero_()
                graph.replay()
                kept = (x, base, step.qkv.clone(), step.out.clone(), step.keys.clone(),
                        step.values.clone())
            stream.synchronize()
            check(step, *kept)
            with torch.cuda.stream(stream):  # an eager call between replays
                step.enqueue(device)
            torch.cuda.synchronize()
    finally:
        device.close()


def test_single_kernels_beside_them_on_the_default_stream():
    # Products, which wait for their stream, between the ops, which do not.
    device = fz.Device(0, stream=0)
    try:
        layer.test_a_batch_of_requests_steps_through_a_layer(device)
    finally:
        device.close()


def test_two_handles_on_one_stream():
    # Each with a workspace of its own, their calls in the stream's order.
    stream = torch.cuda.Stream()
    devices = [fz.Device(0, stream=stream.cuda_stream) for _ in range(2)]
    try:
        with torch.cuda.stream(stream):
            torch.manual_seed(5)
            steps, kept = [Step(), Step()], []
            for i in range(6):
                step = steps[i % 2]
                x, base = torch.randn(ROWS, HIDDEN, device="cuda"), torch.randn(ROWS, QKV,
                                                                               device="cuda")
                step.x.copy_(x)
                step.base.copy_(base)
                step.enqueue(devices[i % 2])
                kept.append((step, x, base, step.qkv.clone(), step.out.clone(),
                             step.keys.clone(), step.values.clone()))
        torch.cuda.synchronize()
        for k in kept:
            check(*k)
    finally:
        for d in devices:
            d.close()


def test_the_stream_outlives_the_handle_and_holds_no_model():
    stream = torch.cuda.Stream()
    device = fz.Device(0, stream=stream.cuda_stream)
    cfg = fz.gemma3_1b_config(layers=2, vocab=2048, window=64, pattern=2, context=1024,
                              local_slots=640)
    with pytest.raises(fz.FrzError, match="caller's stream"):
        fz.Model(device, cfg)
    a = device.array(np.arange(40, dtype=np.float32))
    assert np.array_equal(a.numpy(), np.arange(40))
    a.free()
    device.close()
    with torch.cuda.stream(stream):
        assert float(torch.ones(3, device="cuda").sum()) == 3.0
