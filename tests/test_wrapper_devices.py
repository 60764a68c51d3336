"""CPU: the wrappers of the cache writes launch with their tensors' GPU as the current device, and take
tensors of one GPU only.  The library and the tensors' devices are stood in for."""
import types

import pytest
import torch

import iitj_llm_coopt_amd as M
from iitj_llm_coopt_amd import _lib


class OnGpu(torch.Tensor):
    """A CPU tensor that says it lies on a GPU."""

    @staticmethod
    def on(t, index):
        t = t.as_subclass(OnGpu)
        t.index = index
        return t

    @property
    def device(self):
        return torch.device("cuda", self.index)

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return self.index

    def contiguous(self):
        return self

    def new_empty(self, shape, dtype=None):
        return OnGpu.on(torch.empty(shape, dtype=dtype or self.dtype), self.index)


@pytest.fixture
def launched(monkeypatch):
    """(current device of each launch); GPU 0 is the current one outside of call_on."""
    calls, current = [], [0]

    def call_on(index, fn, *args):
        was, current[0] = current[0], index
        try:
            return fn(*args)
        finally:
            current[0] = was

    def fn(*args):
        calls.append(current[0])
        return _lib.COOPT_OK

    lib = types.SimpleNamespace(coopt_kv_write=fn, coopt_qkv_epilogue=fn, coopt_dequantize=fn)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "entry", lambda name: getattr(lib, name))
    monkeypatch.setattr(_lib, "call_on", call_on)
    for name in ("stream_handle", "raw_stream"):
        monkeypatch.setattr(_lib, name, lambda device=None: 0)
    monkeypatch.setattr(torch, "empty", lambda *a, _empty=torch.empty, device=None, **kw: _empty(*a, **kw))
    return calls


def tensors(index, kv="int4"):
    t = dict(zip(("kc", "vc", "ks", "vs"), M.allocate_kv_cache(2, 16, 2, 64, kv, device="cpu")))
    t.update(k=torch.zeros(3, 2, 64, dtype=torch.bfloat16), slots=torch.zeros(3, dtype=torch.int64),
             qkv=torch.zeros(3, 8 * 64, dtype=torch.bfloat16), pos=torch.zeros(3, dtype=torch.int64),
             tab=torch.zeros(4, 32, dtype=torch.bfloat16))
    return {n: x if x is None else OnGpu.on(x, index) for n, x in t.items()}


def write(t, kv="int4"):
    M.reshape_and_cache_flash(t["k"], t["k"], t["kc"], t["vc"], t["slots"], kv, t["ks"], t["vs"])


def rope(t, kv="int4"):
    M.qkv_rope_and_cache(t["qkv"], t["pos"], t["tab"], t["tab"], t["kc"], t["vc"], t["slots"], 4, 2, 64, kv,
                         t["ks"], t["vs"])


def read(t):
    M.dequantize(t["kc"], t["ks"], 4)


@pytest.mark.parametrize("call", [write, rope, read])
def test_launches_on_the_tensors_gpu(launched, call):
    call(tensors(1))
    assert launched == [1]


@pytest.mark.parametrize("kv", ["auto", "int8"])
def test_other_caches_launch_there_too(launched, kv):
    write(tensors(1, kv), kv)
    rope(tensors(1, kv), kv)
    assert launched == [1, 1]


@pytest.mark.parametrize("call,names", [(write, ("kc", "vc", "slots", "ks", "vs")), (read, ("ks",)),
                                        (rope, ("kc", "vc", "slots", "ks", "vs", "pos"))])
def test_tensors_of_two_gpus_are_refused(launched, call, names):
    for name in names:
        t = tensors(0)
        t[name] = OnGpu.on(t[name], 1)
        with pytest.raises(ValueError, match="one device"):
            call(t)
    assert not launched
