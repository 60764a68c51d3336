"""CPU: attention calls of several threads do not run between the launches of one that shares their
stream's workspace.  The library's functions are stood in for by ones that note when they overlap."""
import threading
import time
import types

import pytest
import torch

from iitj_llm_coopt_amd import _lib, attention


@pytest.fixture
def launches(monkeypatch):
    """Lets the wrappers take CPU tensors; the list holds the entry points that ran beside another."""
    overlaps, running = [], []

    def launch(name):
        def fn(*args):
            running.append(name)
            time.sleep(0.002)        # a call's launches, the interpreter free for other threads
            if len(running) > 1:
                overlaps.append(tuple(running))
            running.remove(name)
            return _lib.COOPT_OK
        return fn

    names = ("coopt_verify_attention_rows", "coopt_verify_attention_qkv", "coopt_window_attention")
    lib = types.SimpleNamespace(**{n: launch(n) for n in names}, coopt_verify_attention_qkv_supported=lambda *a: 1,
                                coopt_verify_attention_workspace=lambda *a: 512,
                                coopt_window_attention_workspace=lambda *a: 1024)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "entry", lambda name: getattr(lib, name))
    monkeypatch.setattr(_lib, "call_on", lambda index, fn, *args: fn(*args))
    for name in ("require_cuda", "require_one_device"):
        monkeypatch.setattr(_lib, name, lambda *t: None)
    for name in ("stream_handle", "raw_stream"):
        monkeypatch.setattr(_lib, name, lambda device=None: 0)
    monkeypatch.setattr(attention, "_workspace_bytes", lambda *sizes: 512)
    monkeypatch.setattr(attention, "_window_workspace_bytes", lambda *sizes: 1024)
    monkeypatch.setattr(attention, "_WS", _lib.WorkspaceCache())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return overlaps


def calls():
    kc = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    codes, s = torch.zeros(4, 16, 2, 32, dtype=torch.uint8), torch.zeros(4, 16, 2, dtype=torch.float16)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    cu, lens = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([40], dtype=torch.int32)
    table, one = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    tab = torch.zeros(64, 32, dtype=torch.bfloat16)
    meta = (cu, lens, table, 1, 40)
    return {
        "plain": lambda **kw: attention.paged_attention(q, kc, kc, *meta, **kw),
        "window": lambda **kw: attention.paged_attention(q, kc, kc, *meta, window=8, **kw),
        "int4": lambda **kw: attention.paged_attention(q, codes, codes, *meta, k_scale=s, v_scale=s, **kw),
        "fused": lambda **kw: attention.paged_attention_qkv(torch.zeros(1, 8 * 64, dtype=torch.bfloat16), one, tab, tab,
                                                            one, kc, kc, *meta, 4, **kw),
    }


@pytest.mark.parametrize("kinds", [("window", "plain"), ("int4", "plain"), ("window", "fused"), ("plain", "plain"),
                                   ("plain", "int4", "fused", "window")])
def test_calls_with_the_shared_workspace_take_turns(launches, kinds):
    todo = calls()
    start = threading.Barrier(len(kinds))
    failed = []

    def work(kind):
        try:
            start.wait()
            for _ in range(20):
                todo[kind]()
        except Exception as e:  # noqa: BLE001 -- shown by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in kinds]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert not launches, (len(launches), launches[0])


def test_calls_with_workspaces_of_their_own_do_not_wait(launches):
    todo = calls()
    ws = torch.empty(4096, dtype=torch.uint8)
    with attention._WS_LOCK:
        for kind in todo:
            todo[kind](workspace=ws)


def test_a_call_that_fails_leaves_the_lock_free(launches, monkeypatch):
    def fail(*args):
        raise RuntimeError("no launch")
    for name in ("coopt_verify_attention_rows", "coopt_verify_attention_qkv", "coopt_window_attention"):
        monkeypatch.setattr(_lib.load(), name, fail)
    for kind, call in calls().items():
        with pytest.raises(RuntimeError, match="no launch"):
            call()
        assert not attention._WS_LOCK.locked(), kind
