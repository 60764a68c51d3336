"""CPU: what the microscaled 4-bit codec and products and the residual norm refuse, before any launch, and
the sizes of their buffers."""
import pytest
import torch

import iitj_llm_coopt_amd as M
from iitj_llm_coopt_amd import _lib, fused


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(rc, code=_lib.COOPT_EINVAL):
    assert rc == code, rc
    return _lib.last_error()


def test_codec_refuses(lib):
    q, d = lib.coopt_mxfp4_quantize, lib.coopt_mxfp4_dequantize
    for args, what in (((_lib.DT_I8, 16, 1, 32, 16, 16), "in_dtype"), ((_lib.DT_BF16, 16, 1, 48, 16, 16), "multiple of 32"),
                       ((_lib.DT_BF16, 16, -1, 32, 16, 16), "multiple of 32"), ((_lib.DT_BF16, 16, 1, -32, 16, 16), "multiple of 32"),
                       ((_lib.DT_BF16, None, 1, 32, 16, 16), "null"), ((_lib.DT_BF16, 8, 1, 32, 16, 16), "aligned"),
                       ((_lib.DT_BF16, 16, 1, 32, 18, 16), "aligned"), ((_lib.DT_BF16, 16, 1 << 38, 32, 16, 16), "too large"),
                       ((_lib.DT_BF16, 16, 1 << 28, 128, 16, 16), "too large")):
        assert what in refused(q(*args, None)), args
    for args, what in (((16, 16, 1, 32, _lib.DT_I8, 16), "out_dtype"), ((16, 16, 1, 33, _lib.DT_F32, 16), "multiple of 32"),
                       ((16, None, 1, 32, _lib.DT_F32, 16), "null"), ((18, 16, 1, 32, _lib.DT_F32, 16), "aligned"),
                       ((16, 16, 1, 32, _lib.DT_F32, 8), "aligned")):
        assert what in refused(d(*args, None)), args
    assert q(_lib.DT_BF16, None, 0, 32, None, None, None) == _lib.COOPT_OK
    assert d(None, None, 4, 0, _lib.DT_BF16, None, None) == _lib.COOPT_OK


def test_pack_refuses(lib):
    pack = lib.coopt_mxfp4_pack_weight
    for args, what in (((16, 16, 16, 40, 16), "multiple of 32"), ((16, 16, -1, 32, 16), "multiple of 32"),
                       ((None, 16, 16, 32, 16), "null"), ((8, 16, 16, 32, 16), "aligned"), ((16, 16, 16, 32, 8), "aligned")):
        assert what in refused(pack(*args, None)), args
    size = lib.coopt_mxfp4_packed_bytes
    assert size(0, 32) == size(16, 0) == size(16, 33) == size(-1, 32) == 0
    assert size(16, 128) == 2 * (4096 + 256) and size(33, 544) == 4 * 2 * (4096 + 256)


def product(lib, partials=False, **kw):
    a = dict(x=16, ldx=256, w=16, M=8, N=64, K=256, act4=0, y=16, ldy=64, ws=16, wsb=1 << 30)
    a.update(kw)
    if partials:
        return lib.coopt_mxfp4_linear_partials(a["x"], a["ldx"], a["w"], a["M"], a["N"], a["K"], a["act4"], a["ws"],
                                               a["wsb"], None)
    return lib.coopt_mxfp4_linear(a["x"], a["ldx"], a["w"], a["M"], a["N"], a["K"], a["act4"], a["y"], a["ldy"],
                                  a["ws"], a["wsb"], None)


@pytest.mark.parametrize("partials", [False, True])
def test_products_refuse(lib, partials):
    for kw, what in ((dict(K=200), "multiple of 32"), (dict(K=0), "multiple of 32"), (dict(M=-1), "negative"),
                     (dict(N=-4), "negative"), (dict(M=(1 << 19) + 1), "2^19"), (dict(N=(1 << 24) + 16), "2^24"),
                     (dict(x=None), "null"), (dict(w=None), "null"), (dict(x=8), "aligned"), (dict(w=8), "aligned"),
                     (dict(K=(1 << 22) + 32), "2^22"), (dict(ldx=(1 << 22) + 8), "row stride of x"),
                     (dict(ldx=255), "row stride of x"), (dict(ldx=260), "row stride of x")):
        assert what in refused(product(lib, partials, **kw)), kw
    if partials:
        assert "multiple of 32" in refused(product(lib, True, N=80))
        refused(product(lib, True, wsb=8), _lib.COOPT_EWORKSPACE)
    else:
        assert "null" in refused(product(lib, y=None)) and "row stride of y" in refused(product(lib, ldy=63))
    assert "workspace" in refused(product(lib, partials, M=20, act4=1, wsb=8), _lib.COOPT_EWORKSPACE)
    assert "workspace" in refused(product(lib, partials, M=20, act4=1, ws=8), _lib.COOPT_EWORKSPACE)
    assert product(lib, partials, M=0) == product(lib, partials, N=0) == _lib.COOPT_OK


def test_product_workspaces(lib):
    import ctypes
    ws, split = lib.coopt_mxfp4_linear_workspace, lib.coopt_mxfp4_linear_split
    for M, N, K in ((17, 4096, 4096), (32, 2048, 8192), (77, 4096, 14336), (160, 6144, 4096), (2000, 4096, 14336)):
        for act4 in (0, 1):
            ks, rows = ctypes.c_int(), ctypes.c_int()
            assert split(M, N, K, act4, ctypes.byref(ks), ctypes.byref(rows)) == _lib.COOPT_OK
            assert 1 <= ks.value <= 16 and rows.value >= M
            part, rows16 = 4 * ks.value * rows.value * N, -(-M // 16) * 16
            room = 9 * 16 if M > 64 else 0   # what the last block of rows reads past them
            packed = act4 * (rows16 + room) * -(-K // 512) * (256 + 16)
            assert ws(M, N, K, act4, 1) == part + packed
            # whole slices, if any, where no consumer adds them
            rest = ws(M, N, K, act4, 0) - packed
            assert rest >= 0 and rest % (4 * rows.value * N) == 0 and rest // (4 * rows.value * N) in (0, *range(2, 17))
    for bad in ((0, 16, 32), (4, 0, 32), (4, 16, 48), (-1, 16, 32)):
        assert ws(*bad, 0, 1) == 0
    assert "null" in refused(split(1, 16, 32, 0, None, None))


def norm(lib, **kw):
    a = dict(x=16, part=None, ks=0, slice=0, res=16, ro=16, post=16, gate=16, gs=0, w=16, out=16, rows=2, H=64, eps=1e-5)
    a.update(kw)
    return lib.coopt_residual_norm(a["x"], a["part"], a["ks"], a["slice"], a["res"], a["ro"], a["post"], a["gate"], a["gs"],
                                   a["w"], a["out"], a["rows"], a["H"], a["eps"], 1.0, 1.0, None)


def test_residual_norm_refuses(lib):
    for kw, what in ((dict(H=60), "multiple of 8"), (dict(H=0), "multiple of 8"), (dict(H=16392), "multiple of 8"),
                     (dict(rows=-1), "multiple of 8"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                     (dict(eps=float("inf")), "eps"), (dict(x=None), "exactly one"), (dict(part=16), "exactly one"),
                     (dict(x=None, part=16, ks=17, slice=128), "partial"), (dict(x=None, part=16, ks=0, slice=128), "partial"),
                     (dict(x=None, part=16, ks=2, slice=64), "partial"), (dict(res=None), "null"), (dict(ro=None), "null"),
                     (dict(w=None), "null"), (dict(out=None), "null"), (dict(gs=32), "gate rows"), (dict(gs=68), "gate rows"),
                     (dict(x=8), "aligned"), (dict(gate=24), "aligned"), (dict(post=8), "aligned"), (dict(out=8), "aligned")):
        assert what in refused(norm(lib, **kw)), kw
    assert norm(lib, rows=0) == _lib.COOPT_OK


def test_wrappers_refuse():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    with pytest.raises(_lib.CooptError, match="no CPU fallback"):
        M.quantize_mxfp4(bf(2, 32))
    with pytest.raises(_lib.CooptError, match="no CPU fallback"):
        M.dequantize_mxfp4(u8(2, 16), u8(2, 1))
    with pytest.raises(_lib.CooptError, match="no CPU fallback"):
        M.pack_mxfp4_weight(u8(2, 16), u8(2, 1))
    with pytest.raises(ValueError, match="activations"):
        M.pack_mxfp4_weight(u8(2, 16), u8(2, 1), "int8")
    with pytest.raises(ValueError, match="must be .N, K."):
        M.quantize_mxfp4_weight(bf(32))
    w = M.MXFP4Weight(u8(16, 16), u8(16, 1), u8(8704))
    with pytest.raises(_lib.CooptError, match="no CPU fallback"):
        fused.linear(bf(2, 32), w)
    with pytest.raises(_lib.CooptError, match="no CPU fallback"):
        fused.residual_norm(bf(2, 64), bf(2, 64), bf(64), 1e-5)
