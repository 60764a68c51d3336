"""CPU: where the products with 4-bit weights take their workspace from.  The kernels and the tensors' devices are
stood in for; sizes and plans are the library's."""
import weakref

import pytest
import torch

from iitj_llm_coopt_amd import _lib, fused
from iitj_llm_coopt_amd.mxfp4 import MXFP4Weight
from test_wrapper_devices import OnGpu


class Gpu:
    """The current device, which devices' streams are under capture, and what was allocated and launched."""

    def __init__(self):
        self.current, self.capturing, self.cached, self.own, self.launches = 0, set(), [], [], []


class Tensor(OnGpu):
    gpu = None

    def new_empty(self, *shape, dtype=None):
        t = OnGpu.on(torch.zeros(*shape, dtype=dtype or self.dtype), self.index).as_subclass(Tensor)
        t.index = self.index
        if t.dtype == torch.uint8:
            self.gpu.own.append(t.numel())
        return t


def on(t, index):
    t = OnGpu.on(t, index).as_subclass(Tensor)
    t.index = index
    return t


@pytest.fixture
def gpu(monkeypatch):
    state = Gpu()
    entry, empty = _lib.entry, torch.empty

    def call_on(index, fn, *args):
        was, state.current = state.current, index
        try:
            return fn(*args)
        finally:
            state.current = was

    def product(*args):
        state.launches.append(args[-2])   # workspace bytes
        return _lib.COOPT_OK

    def cached(*size, device=None, **kw):
        t = empty(*size, **kw)
        state.cached.append((weakref.ref(t), t.numel()))
        return t

    names = ("coopt_mxfp4_linear", "coopt_mxfp4_linear_partials")
    monkeypatch.setattr(_lib, "entry", lambda name: product if name in names else entry(name))
    monkeypatch.setattr(_lib, "call_on", call_on)
    for name in ("stream_handle", "raw_stream"):
        monkeypatch.setattr(_lib, name, lambda device=None: 0)
    monkeypatch.setattr(torch, "empty", cached)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.current in state.capturing)
    monkeypatch.setattr(fused._WS4, "_bufs", {})
    monkeypatch.setattr(Tensor, "gpu", state)
    return state


def weight(N, K, index, activations="mxfp4"):
    size = _lib.load().coopt_mxfp4_packed_bytes(N, K)
    u8 = lambda *s: on(torch.zeros(s, dtype=torch.uint8), index)
    return MXFP4Weight(u8(N, K // 2), u8(N, K // 32), u8(size), activations)


def rows(M, K, index):
    return on(torch.zeros(M, K, dtype=torch.bfloat16), index)


@pytest.mark.parametrize("current", [0, 1])
def test_a_capture_on_the_tensors_gpu_gets_a_workspace_of_its_own(gpu, current):
    """Also where another GPU is the current one; and a capture there leaves other GPUs' products alone."""
    w, x = weight(64, 512, 1), rows(80, 512, 1)
    gpu.current, gpu.capturing = current, {1}
    fused.linear(x, w)
    assert len(gpu.launches) == 1 and gpu.own == gpu.launches and not gpu.cached
    gpu.capturing = {0}
    fused.linear(x, w)
    assert len(gpu.launches) == 2 and len(gpu.own) == 1 and len(gpu.cached) == 1


def test_outgrown_workspaces_are_freed(gpu):
    """Rows that grow 16 at a time, as prompts do: one workspace is alive, at most an eighth larger than the largest
    need, and few were allocated."""
    w = weight(64, 14336, 0)
    for M in range(80, 4096, 16):
        fused.linear(rows(M, 14336, 0), w)
    alive = [n for ref, n in gpu.cached if ref() is not None]
    need = w.plan(4080)[0]
    assert len(alive) == 1 and need <= alive[0] <= need * 9 // 8
    assert len(gpu.cached) <= 8 * 5   # eight sizes a doubling of the need, which grows 20-fold
    assert not gpu.own
