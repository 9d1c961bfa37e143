"""Which device a call's workspace is sized for, on a stand-in for the library and for torch.cuda."""
import pytest

torch = pytest.importorskip("torch")


def test_the_workspace_is_sized_on_the_tensors_device(monkeypatch):
    """The plan follows from the device's SM count: the query runs with the tensors' device current,
    whichever device the caller has."""
    from gafime_b200 import _native, ops
    current, asked = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    class Lib:
        def gafime_xent_workspace(self, *args):
            asked.append(current[0])
            args[-1]._obj.value = 512
            return 0

        def gafime_grad_norm_workspace(self, count, out):
            out._obj.value = 256
            return 0

    monkeypatch.setattr(_native, "load", lambda require_gpu=True: Lib())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    ops._workspace_bytes.cache_clear()
    try:
        assert ops._workspace_bytes(1, 0, 0, 40, 1, 0, 40, 1, 10, 40, 3, 0) == 512
        assert ops._workspace_bytes(0, 0, 0, 40, 1, 0, 40, 1, 10, 40, 3, 0) == 512
    finally:
        ops._workspace_bytes.cache_clear()
    assert asked == [1, 0] and current == [0]
