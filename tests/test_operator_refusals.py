"""CPU: what the window / 4-bit attention, the q / k norm and the 4-bit writes refuse, before any
launch, and the sizes of their workspaces."""
import pytest
import torch

import iitj_llm_coopt_amd as M
from iitj_llm_coopt_amd import _lib
from iitj_llm_coopt_amd.attention import window_workspace_bytes


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(rc):
    assert rc == _lib.COOPT_EINVAL, rc
    return _lib.last_error()


def attention(lib, **kw):
    a = dict(kv=_lib.DT_I4, q=16, qts=4096, qhs=128, k=16, v=16, cbs=8192, cts=512, chs=64, ks=16, vs=16, B=2, Hq=32,
             Hkv=8, D=128, bs=16, nb=64, mq=5, mk=100, bt=16, win=0, sinks=0, scale=0.088, out=16, ws=16, wsb=1 << 30)
    a.update(kw)
    return lib.coopt_window_attention(a["kv"], a["q"], a["qts"], a["qhs"], a["k"], a["v"], a["cbs"], a["cts"],
                                      a["chs"], a["ks"], a["vs"], 128, 8, 1, 16, a["bt"], 16, 16, a["B"], a["Hq"],
                                      a["Hkv"], a["D"], a["bs"], a["nb"], a["mq"], a["mk"], 0, a["win"], a["sinks"],
                                      a["scale"], a["out"], 4096, 128, a["ws"], a["wsb"], None)


def test_window_attention_refuses(lib):
    for kw, what in ((dict(kv=_lib.DT_F16), "kv_dtype"), (dict(D=96), "head_dim"), (dict(Hq=30), "multiple of Hkv"),
                     (dict(Hq=130, Hkv=2), "<= 64"), (dict(bs=24), "power of two"), (dict(bs=8), "power of two"),
                     (dict(bt=3), "narrower"), (dict(win=-1), "negative"), (dict(win=5, sinks=-1), "negative"),
                     (dict(sinks=4), "needs a window"), (dict(mq=0), "positive"), (dict(mk=0), "positive"),
                     (dict(k=None), "null"), (dict(q=8), "aligned"), (dict(qts=4097), "aligned"),
                     (dict(k=8), "aligned"), (dict(cts=520), "aligned"), (dict(ks=None), "k_scale"),
                     (dict(kv=_lib.DT_I8, vs=None), "k_scale"), (dict(ks=17), "k_scale"), (dict(nb=0), "num_blocks"),
                     (dict(B=70000, wsb=1 << 40), "65535"), (dict(B=-1), "Hq"), (dict(scale=-1.0), "softmax_scale"), (dict(scale=float("nan")), "softmax_scale"),
                     (dict(scale=float("inf")), "softmax_scale"), (dict(mk=1 << 30), "out of range"),
                     (dict(mq=1 << 29), "out of range")):
        assert what in refused(attention(lib, **kw)), (kw, _lib.last_error())
    assert attention(lib, B=0) == _lib.COOPT_OK
    assert attention(lib, wsb=8) == _lib.COOPT_EWORKSPACE
    assert attention(lib, ws=None) == _lib.COOPT_EWORKSPACE


def test_window_workspace_sizes(lib):
    size = lib.coopt_window_attention_workspace
    assert size(1, 32, 8, 128, 1, 8192, 0, 0) > 0
    # refused shapes have none
    for bad in ((0, 32, 8, 128, 1, 100, 0, 0), (1, 30, 8, 128, 1, 100, 0, 0), (1, 32, 8, 96, 1, 100, 0, 0),
                (1, 32, 8, 128, 1, 100, -1, 0), (1, 32, 8, 128, 1, 100, 5, -1)):
        assert size(*bad) == 0, bad
    # a window keeps it small, and the wrapper takes any window and first tokens past the context
    a = window_workspace_bytes(1, 32, 8, 128, 1, 16000, 1024, 4)
    assert 0 < a <= window_workspace_bytes(1, 32, 8, 128, 1, 16000)
    assert window_workspace_bytes(1, 32, 8, 128, 1, 16000, 2 ** 50, 2 ** 40) > 0
    for bad, kind in ((dict(window=0), ValueError), (dict(sink_tokens=1), ValueError),
                      (dict(window=4, sink_tokens=-1), ValueError), (dict(window=1.5), TypeError)):
        with pytest.raises(kind):
            window_workspace_bytes(1, 32, 8, 128, 1, 16000, **bad)


def epilogue(lib, **kw):
    a = dict(kv=_lib.DT_BF16, qkv=16, ts=6144, part=None, ks=0, slice=0, qw=16, kw=16, eps=1e-5, cos=16, tab=64, mp=4,
             k=16, v=16, cts=1024, sk=None, sv=None, T=2, Hq=32, Hkv=8, D=128, nb=4)
    a.update(kw)
    return lib.coopt_qkv_norm_epilogue(a["kv"], a["qkv"], a["ts"], a["part"], a["ks"], a["slice"], a["qw"], a["kw"],
                                       a["eps"], 16, a["cos"], 16, a["tab"], a["mp"], 16, 4096, 128, a["k"], a["v"],
                                       16384, a["cts"], 128, a["sk"], a["sv"], 128, 8, 1, 16, a["T"], a["Hq"],
                                       a["Hkv"], a["D"], 16, a["nb"], None)


def test_norm_epilogue_refuses(lib):
    for kw, what in ((dict(kv=0), "cache_dtype"), (dict(D=96), "D must be"), (dict(T=-1), "bad sizes"),
                     (dict(mp=0), "bad sizes"), (dict(nb=0), "bad sizes"), (dict(eps=-1e-9), "eps"),
                     (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(qkv=None), "exactly one"),
                     (dict(part=16), "exactly one"), (dict(qw=None), "null"), (dict(kw=8), "16-byte aligned"),
                     (dict(ts=6136), "qkv rows"), (dict(ts=6145), "qkv rows"), (dict(cos=8), "cos/sin"),
                     (dict(tab=56), "cos/sin"), (dict(k=8), "bf16 cache rows"), (dict(cts=1028), "bf16 cache rows"),
                     (dict(kv=_lib.DT_I8), "needs k_scale"), (dict(kv=_lib.DT_I4), "needs k_scale"),
                     (dict(kv=_lib.DT_I4, sk=16, sv=16, k=18), "INT4 cache rows"),
                     (dict(kv=_lib.DT_I8, sk=16, sv=16, k=20), "INT8 cache rows"),
                     (dict(kv=_lib.DT_I4, sk=17, sv=16), "2-byte"), (dict(T=1 << 23), "too many rows"),
                     (dict(qkv=None, part=16, ks=17, slice=1 << 20), "1 to 16"),
                     (dict(qkv=None, part=16, ks=2, slice=6144), "partials")):
        assert what in refused(epilogue(lib, **kw)), (kw, _lib.last_error())
    assert epilogue(lib, T=0) == _lib.COOPT_OK


def test_int4_kv_write_refuses(lib):
    def call(k=16, cts=512, ks=16):
        return lib.coopt_kv_write(_lib.DT_I4, 16, 16, 1024, 128, 1024, 128, k, 16, 8192, cts, 64, ks, 16, 128, 8, 1,
                                  16, 1, 8, 128, 16, 4, None)
    assert "INT4 cache rows" in refused(call(k=18))
    assert "INT4 cache rows" in refused(call(cts=514))
    assert "needs k_scale" in refused(call(ks=None))


def test_wrappers_refuse_cpu_tensors_and_odd_heads():
    z = torch.zeros(2, 8 * 64, dtype=torch.bfloat16)
    w, t, i = torch.ones(64, dtype=torch.bfloat16), torch.ones(4, 32, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    kc, vc, ks, vs = M.allocate_kv_cache(2, 16, 2, 64, "int4", device="cpu")
    assert kc.shape == (2, 16, 2, 32) and kc.dtype == torch.uint8 and ks.shape == (2, 16, 2)
    with pytest.raises(_lib.CooptError, match="no CPU fallback"):
        M.qkv_norm_rope_and_cache(z, w, w, 1e-5, i, t, t, kc, vc, i, 4, 2, 64, "int4", ks, vs)
    with pytest.raises(ValueError, match="even head_dim"):
        M.allocate_kv_cache(2, 16, 2, 33, "int4", device="cpu")
    with pytest.raises(ValueError, match="'int4'"):
        M.allocate_kv_cache(2, 16, 2, 64, "int2", device="cpu")


def test_the_fused_call_leaves_int4_caches_to_the_two_calls():
    assert not M.qkv_attention_supported("int4", 1, 32, 8, 128, 1, 100)
