"""CPU checks of how the wrappers of the trainable block pieces make their
calls: what they refuse before a pointer leaves them, and what a wait leaves
alone.  The library, the contexts and torch's device are stood in for, so no
GPU is needed."""
import contextlib
import threading

import pytest
import torch
import vestra_kernels as vk


class FakeContext:
    """A context that follows one of the streams of `work`, as Context follows a cudaStream_t."""

    handle = 1

    def __init__(self, device, work, current):
        self.device, self.work, self.current, self.stream, self.started = device, work, current, 7, threading.Event()

    def set_stream(self, stream):
        self.stream = stream

    def synchronize(self):
        self.current.device = self.device  # as vk_synchronize does
        self.started.set()
        if self.stream in self.work:
            assert self.work[self.stream].wait(20)


@pytest.fixture
def fake(monkeypatch):
    """Two devices whose default-context calls go to stand-ins; `device` is the calling thread's current one."""
    work, current = {7: threading.Event()}, threading.local()

    @contextlib.contextmanager
    def device(i):
        before = getattr(current, "device", 0)
        current.device = i
        yield
        current.device = before

    class External:
        def __init__(self, stream, device=None):
            self.stream = stream

        def synchronize(self):
            contexts[0].started.set()
            if self.stream in work:
                assert work[self.stream].wait(20)

    class Lib:
        def __getattr__(self, name):
            return lambda *a: vk.VK_OK

    contexts = {d: FakeContext(d, work, current) for d in (0, 1)}
    monkeypatch.setattr(vk, "_on_stream", {d: [c, 7] for d, c in contexts.items()})
    monkeypatch.setattr(vk, "lib", lambda: Lib())
    monkeypatch.setattr(vk, "_torch_stream", lambda d: 8)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: getattr(current, "device", 0))
    monkeypatch.setattr(torch.cuda, "ExternalStream", External)
    return work, contexts


def test_synchronize_leaves_other_threads_calls_alone(fake):
    """While one thread waits for its work, another's call on another stream goes through."""
    work, contexts = fake
    waiting = threading.Thread(target=vk.synchronize, args=(0,))
    waiting.start()
    assert contexts[0].started.wait(20)
    called = threading.Thread(target=vk._launch, args=("vk_rope_axes", 0, None))
    called.start()
    called.join(5)
    through = not called.is_alive()
    work[7].set()
    waiting.join()
    called.join()
    assert through


def test_synchronize_waits_for_a_call_made_during_another_wait(fake):
    """A call that another thread made while one waited is the last one for the next wait."""
    work, contexts = fake
    first = threading.Thread(target=vk.synchronize, args=(0,))
    first.start()
    assert contexts[0].started.wait(20)
    vk._launch("vk_rope_axes", 0, None)  # goes to stream 8
    work[7].set()
    first.join()
    work[8] = threading.Event()
    second = threading.Thread(target=vk.synchronize, args=(0,))
    second.start()
    second.join(0.5)
    assert second.is_alive()
    work[8].set()
    second.join(20)
    assert not second.is_alive()


def test_synchronize_leaves_the_current_device(fake):
    work, _ = fake
    work[7].set()
    vk.synchronize(1)
    assert torch.cuda.current_device() == 0


class OnGpu:
    """What the wrappers ask of a CUDA tensor, with an address of its own."""

    is_cuda = True

    def __init__(self, *shape, dtype=torch.float32, address=1 << 20, device=0, strides=None):
        self.shape, self.dtype, self.address, self.device = torch.Size(shape), dtype, address, torch.device("cuda", device)
        self.strides = strides or torch.empty(shape, device="meta").stride()

    def get_device(self):
        return self.device.index

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def element_size(self):
        return self.dtype.itemsize

    def stride(self):
        return self.strides

    def is_contiguous(self):
        return self.strides == torch.empty(self.shape, device="meta").stride()

    def data_ptr(self):
        return self.address


@pytest.fixture
def launched(monkeypatch):
    """The calls that would have reached the library."""
    calls = []
    monkeypatch.setattr(vk, "_launch", lambda name, device, ctx, *args: calls.append((name, device, args)))
    return calls


def norm_backward(workspace):
    x, vec, stats = OnGpu(2, 3, 8), OnGpu(8), OnGpu(2, 3, 2)
    vk.residual_norm_backward(x, x, x, x, stats, vec, x, x, vec, vec, workspace=workspace)


@pytest.mark.parametrize("workspace,error", [
    (torch.empty(1 << 16, dtype=torch.uint8), TypeError),  # in host memory: its address means nothing on the GPU
    (OnGpu(1 << 16, dtype=torch.uint8, device=1), TypeError),
    (OnGpu(64, 1024, dtype=torch.uint8, strides=(4096, 1)), ValueError),  # more bytes than lie together
])
def test_norm_workspace_is_on_the_device(launched, workspace, error):
    with pytest.raises(error, match="workspace"):
        norm_backward(workspace)
    assert not launched


def test_norm_workspace_of_any_type(launched):
    norm_backward(OnGpu(1 << 16, dtype=torch.uint8))
    norm_backward(OnGpu(64, 256))
    assert [c[2][-2:] for c in launched] == [(1 << 20, 1 << 16), (1 << 20, 1 << 16)]


def test_norm_workspace_of_matrices_at_odd_addresses(launched):
    """bf16 matrices may start at any even address; the vectors, which only have to be there, are aligned f32."""
    x = OnGpu(2, 3, 8, dtype=torch.bfloat16, address=(1 << 20) + 2)
    vk.residual_norm_workspace(x, x, scale=x, gate=x, post_gamma=x)
    shape = launched[0][2][0]._obj
    for name in ("gamma", "beta", "scale", "gate", "post_gamma", "post_beta"):
        assert getattr(shape, name) and getattr(shape, name) % 4 == 0, name
