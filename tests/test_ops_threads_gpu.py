"""Calls from several host threads at once, each on its own stream and of its own size, straight
at the C entries (ctypes lets the other threads run meanwhile)."""
import ctypes
import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from gafime_b200 import _native
    return _native.load()


class Call:
    """One prepared call of the library, its buffers and its stream."""

    def __init__(self, lib, n, d, c, gradients, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.x = torch.randn((n, d), generator=g, device="cuda")
        self.w = torch.randn((c, d), generator=g, device="cuda") * 0.1
        self.labels = torch.randint(0, c, (n,), generator=g, device="cuda")
        self.loss = torch.empty(n, device="cuda")
        self.dw = torch.empty((c, d), device="cuda")
        want = 8 | 2 if gradients else 0
        size = ctypes.c_size_t(0)
        table = (0, self.x.data_ptr(), d, 1, self.w.data_ptr(), d, 1)
        assert lib.gafime_xent_workspace(*table, n, d, c, want, ctypes.byref(size)) == 0
        self.ws = torch.empty(max(size.value, 256), dtype=torch.uint8, device="cuda")
        self.stream = torch.cuda.Stream()
        head = table + (None, self.labels.data_ptr(), n, d, c)
        tail = (self.ws.data_ptr(), size.value, self.stream.cuda_stream)
        if gradients:
            self.fn = lib.gafime_xent_gradient
            self.args = head + (None, 0, 1.0, 0, self.loss.data_ptr(), None, None, 0, 0, self.dw.data_ptr(), None) + tail
        else:
            self.fn = lib.gafime_xent_forward
            self.args = head + (self.loss.data_ptr(), None) + tail

    def __call__(self):
        return self.fn(*self.args)


# few classes, a few rows, the products: the same kernel with little and with much shared memory
@pytest.mark.parametrize("shapes", [((64, 72, 3), (64, 2000, 3)), ((4, 200, 64), (4, 3000, 64)),
                                    ((300, 60, 40), (300, 900, 40))])
@pytest.mark.parametrize("gradients", [False, True])
def test_tables_of_different_width(lib, shapes, gradients):
    calls = [Call(lib, *s, gradients, i) for i, s in enumerate(shapes * 2)]
    torch.cuda.synchronize()
    wanted = []
    for call in calls:
        assert call() == 0
        torch.cuda.synchronize()
        wanted.append((call.loss.clone(), call.dw.clone()))
    codes, start = [], threading.Barrier(len(calls))

    def work(call):
        start.wait()
        bad = 0
        for _ in range(4000):
            bad += call() != 0
        codes.append(bad)

    threads = [threading.Thread(target=work, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [0] * len(calls)
    for call, (loss, dw) in zip(calls, wanted):
        assert torch.equal(call.loss, loss)
        if gradients:
            assert torch.equal(call.dw, dw)
