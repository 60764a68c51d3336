"""GPU: the KV write into 4-bit caches, and the q / k head norms with rotation and cache write.

4-bit codes and scales equal the codec's (oracle.codec, IEEE fp32) bit for bit.  The norm against
float64: |got - ref| <= 2^-8 |ref| (the one rounding to bf16) + 2^-20 (|y1| + |y2|), y the two
normed elements a rotation combines: the sum of D <= 256 squares in fp32 (D / 8 + 8 additions in
the longest chain, 2^-24 each, halved by the root), rsqrt, four products and one addition of
2^-24 each come to less than 2^-20.
"""
import numpy as np
import pytest
import torch

import iitj_llm_coopt_amd as M
from iitj_llm_coopt_amd import _lib, fused
from oracle import codec as OC

pytestmark = pytest.mark.gpu


def cache(dev, nb, bs, Hkv, D, kv, layout):
    """Caches of a kind, full of a value no write leaves, and their scales."""
    def one(last, dt, fill):
        if layout == "head":
            return torch.full((nb, Hkv, bs, last), fill, dtype=dt, device=dev).transpose(1, 2)
        if layout == "token":
            return torch.full((nb, bs, Hkv, last), fill, dtype=dt, device=dev)
        return torch.full((nb, bs + 2, Hkv + 1, last + 32), fill, dtype=dt, device=dev)[:, 1:bs + 1, 1:, :last]
    kind = {"auto": (D, torch.bfloat16, 9.0), "int8": (D, torch.int8, 99), "int4": (D // 2, torch.uint8, 3)}[kv]
    sc = [None, None] if kv == "auto" else [one(1, torch.float16, 5.0).squeeze(-1) for _ in range(2)]
    return one(*kind), one(*kind), *sc


@pytest.mark.parametrize("layout", ["head", "token", "padded"])
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 16), (8, 24), (16, 16), (256, 64), (512, 16), (32, 10)])
def test_int4_write_is_the_codecs(dev, layout, D, bs):
    nb, Hkv, T = 9, 3, 61
    gen = torch.Generator(device=dev).manual_seed(D + bs)
    x = torch.randn(2, T, Hkv + 1, D, generator=gen, device=dev)
    x = torch.where(torch.rand(x.shape, generator=gen, device=dev) < 0.02, 20 * x, x).to(torch.bfloat16)
    x[:, 3] = 0
    x[:, 4] = x[:, 4].abs().amax(-1, keepdim=True) * torch.randint(-14, 15, x[:, 4].shape, generator=gen, device=dev) / 14
    k, v = x[0][:, :Hkv], x[1][:, 1:]
    slots = torch.randperm(nb * bs, generator=gen, device=dev)[:T]
    slots[5], slots[11], slots[60] = -1, nb * bs, -2 ** 40
    kc, vc, ks, vs = cache(dev, nb, bs, Hkv, D, "int4", layout)
    M.reshape_and_cache_flash(k, v, kc, vc, slots, "int4", ks, vs)
    ok = ((slots >= 0) & (slots < nb * bs)).cpu().numpy()
    s = slots.cpu().numpy()[ok]
    for src, c, sc in ((k, kc, ks), (v, vc, vs)):
        q, scale = OC.quantize(src.float().cpu().numpy(), 4)
        want = np.full(c.shape, 3, np.uint8)
        wants = np.full(sc.shape, 5.0, np.float16)
        want[s // bs, s % bs], wants[s // bs, s % bs] = q[ok], scale[ok]
        assert np.array_equal(c.cpu().numpy(), want) and np.array_equal(sc.cpu().numpy(), wants)
        got = M.quantize(src.contiguous(), 4)
        assert np.array_equal(got[0].cpu().numpy(), q) and np.array_equal(got[1].cpu().numpy(), scale)


def test_int4_write_of_extreme_values_is_quantize(dev):
    """Infinities, subnormals and the type's largest values: the bytes of quantize(x, 4).  A vector
    with a NaN has a NaN for its scale."""
    gen = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(40, 2, 128, generator=gen, device=dev)
    for i, v in enumerate((float("inf"), float("-inf"), float("nan"), 1e-40, 3.3e38, -3.3e38, 1e-38, 0.0)):
        x[4 * i:4 * i + 2, 0, 7 * i] = v
        x[4 * i + 2, 1] = v
    x = x.to(torch.bfloat16)
    kc, vc, ks, vs = M.allocate_kv_cache(3, 16, 2, 128, "int4", device=dev)
    M.reshape_and_cache_flash(x, x.flip(0).contiguous(), kc, vc, torch.arange(40, device=dev), "int4", ks, vs)
    for src, c, s in ((x, kc, ks), (x.flip(0).contiguous(), vc, vs)):
        q, sc = M.quantize(src, 4)
        t = torch.arange(40, device=dev)
        c, s, nan = c[t // 16, t % 16], s[t // 16, t % 16], src.isnan().any(-1)
        assert torch.equal(c[~nan], q[~nan]) and torch.equal(s[~nan], sc[~nan])
        assert nan.sum() == 3 and s[nan].isnan().all()
        assert M.dequantize(c, s, 4)[nan].isnan().all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_int4_rope_and_cache_is_rope_then_write(dev, D):
    Hq, Hkv, T, nb = 6, 3, 37, 4
    gen = torch.Generator(device=dev).manual_seed(D)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen, device=dev).to(torch.bfloat16)
    cos, sin = (torch.randn(50, D, generator=gen, device=dev).to(torch.bfloat16) for _ in range(2))
    pos = torch.randint(0, 50, (T,), generator=gen, device=dev)
    slots = torch.randperm(nb * 16, generator=gen, device=dev)[:T]
    slots[7] = -1
    one, two = (M.allocate_kv_cache(nb, 16, Hkv, D, "int4", device=dev) for _ in range(2))
    q = M.qkv_rope_and_cache(qkv, pos, cos, sin, one[0], one[1], slots, Hq, Hkv, D, "int4", one[2], one[3])
    x = qkv.clone().view(T, Hq + 2 * Hkv, D)
    fused.rope_(x[:, :Hq], x[:, Hq:Hq + Hkv], pos, cos, sin)
    M.reshape_and_cache_flash(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], two[0], two[1], slots, "int4", two[2], two[3])
    assert torch.equal(q, x[:, :Hq])
    for a, b in zip(one, two):
        assert torch.equal(a, b)


def norm_reference(x, w, cos, sin, eps):
    """float64 (z, |y1| + |y2|) of head vectors x [T, H, D]."""
    D = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    a, b = y[..., : D // 2], y[..., D // 2:]
    c, s = cos[:, None, : D // 2], sin[:, None, : D // 2]
    mag = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([mag, mag], -1)


@pytest.mark.parametrize("kv,layout", [("auto", "head"), ("auto", "padded"), ("int8", "head"), ("int8", "token"),
                                       ("int4", "head"), ("int4", "padded")])
@pytest.mark.parametrize("D,Hq,Hkv,T", [(128, 32, 8, 1), (64, 32, 8, 77), (256, 3, 1, 5), (128, 7, 1, 130),
                                        (64, 5, 3, 1), (128, 4, 4, 600)])
def test_norm_rotation_and_write(dev, kv, layout, D, Hq, Hkv, T):
    bs, eps, rows = 16, 1e-6, 90
    nb = -(-T // bs) + 1
    gen = torch.Generator(device=dev).manual_seed(T + D)
    mag = torch.exp(3 * torch.randn(T, Hq + 2 * Hkv, 1, generator=gen, device=dev))
    x = (torch.randn(T, Hq + 2 * Hkv, D, generator=gen, device=dev) * mag).to(torch.bfloat16)
    x[0, 0] = 0                                   # a head of zeros normed stays zero
    wide = torch.zeros(T, (Hq + 2 * Hkv) * D + 8, dtype=torch.bfloat16, device=dev)
    wide[:, : (Hq + 2 * Hkv) * D] = x.reshape(T, -1)
    qkv = wide[:, : (Hq + 2 * Hkv) * D]           # rows further apart than they are wide
    qw, kw = ((1 + torch.randn(D, generator=gen, device=dev)).to(torch.bfloat16) for _ in range(2))
    ang = torch.rand(rows, D, generator=gen, device=dev, dtype=torch.float64) * 6.3
    cos, sin = ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)
    pos = torch.randint(0, rows, (T,), generator=gen, device=dev)
    slots = torch.randperm(nb * bs, generator=gen, device=dev)[:T]
    if T > 3:
        slots[1], slots[3], pos[2] = -1, nb * bs + 3, rows + 1000   # padding, off the pool; the last table row
    kc, vc, ks, vs = cache(dev, nb, bs, Hkv, D, kv, layout)
    qo = torch.empty(T, Hq + 2, D, dtype=torch.bfloat16, device=dev)[:, 1:Hq + 1]
    q = M.qkv_norm_rope_and_cache(qkv, qw, kw, eps, pos, cos, sin, kc, vc, slots, Hq, Hkv, D, kv, ks, vs, q_out=qo)
    assert q.data_ptr() == qo.data_ptr()
    xd = x.double().cpu().numpy()
    p = pos.clamp(max=rows - 1).cpu().numpy()
    c, s = cos.double().cpu().numpy()[p], sin.double().cpu().numpy()[p]

    def near(got, ref, m):
        d = np.abs(got.double().cpu().numpy() - ref)
        assert (d <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * m).all(), float(d.max())

    near(q, *norm_reference(xd[:, :Hq], qw.double().cpu().numpy(), c, s, eps))
    # what a bf16 cache gets
    plain = M.allocate_kv_cache(nb, bs, Hkv, D, "auto", device=dev)
    q2 = M.qkv_norm_rope_and_cache(qkv, qw, kw, eps, pos, cos, sin, plain[0], plain[1], slots, Hq, Hkv, D)
    assert torch.equal(q, q2)
    ok = (slots >= 0) & (slots < nb * bs)
    blk, off = slots[ok] // bs, slots[ok] % bs
    kref, kmag = norm_reference(xd[:, Hq:Hq + Hkv], kw.double().cpu().numpy(), c, s, eps)
    okn = ok.cpu().numpy()
    near(plain[0][blk, off], kref[okn], kmag[okn])
    assert torch.equal(plain[1][blk, off], x[:, Hq + Hkv:][ok])
    # and this cache, every place of it
    k = torch.zeros(T, Hkv, D, dtype=torch.bfloat16, device=dev)
    k[ok] = plain[0][blk, off]
    kc2, vc2, ks2, vs2 = cache(dev, nb, bs, Hkv, D, kv, layout)
    M.reshape_and_cache_flash(k, x[:, Hq + Hkv:].contiguous(), kc2, vc2, slots, kv, ks2, vs2)
    for a, b in ((kc, kc2), (vc, vc2), (ks, ks2), (vs, vs2)):
        assert a is None or torch.equal(a, b)


def test_norm_of_a_projections_partials(dev):
    """The projection's split-K partials, reduced and rounded to bf16 first."""
    D, Hq, Hkv, T, K = 128, 8, 4, 5, 1024
    gen = torch.Generator(device=dev).manual_seed(4)
    w = (torch.randn((Hq + 2 * Hkv) * D, K, generator=gen, device=dev) * 0.05).to(torch.bfloat16)
    h = torch.randn(T, K, generator=gen, device=dev).to(torch.bfloat16)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=gen, device=dev)).to(torch.bfloat16) for _ in range(2))
    cos, sin = (torch.randn(40, D // 2, generator=gen, device=dev).to(torch.bfloat16) for _ in range(2))
    pos, slots = torch.arange(T, device=dev), torch.arange(T, device=dev)
    got = []
    for defer in (True, False):
        caches = M.allocate_kv_cache(2, 16, Hkv, D, "auto", device=dev)
        part = fused.linear(h, w, defer_reduce=True)
        qkv = part if defer else part.reduce()
        q = M.qkv_norm_rope_and_cache(qkv, qw, kw, 1e-5, pos, cos, sin, caches[0], caches[1], slots, Hq, Hkv, D)
        got.append((q, caches[0], caches[1]))
        assert isinstance(part, fused.LinearPartials) and part.ks > 1
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_norm_in_a_graph_on_another_stream(dev):
    D, Hq, Hkv, T = 128, 8, 2, 9
    gen = torch.Generator(device=dev).manual_seed(6)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen, device=dev).to(torch.bfloat16)
    qw = kw = torch.ones(D, dtype=torch.bfloat16, device=dev)
    cos, sin = (torch.randn(40, D // 2, generator=gen, device=dev).to(torch.bfloat16) for _ in range(2))
    pos, slots = torch.arange(T, device=dev), torch.arange(T, device=dev)
    a, b = (M.allocate_kv_cache(1, 16, Hkv, D, "int4", device=dev) for _ in range(2))
    q = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=dev)

    def call(c, **kw_):
        return M.qkv_norm_rope_and_cache(qkv, qw, kw, 1e-5, pos, cos, sin, c[0], c[1], slots, Hq, Hkv, D,
                                         "int4", c[2], c[3], **kw_)
    call(a)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(a, q_out=q)
    side = torch.cuda.Stream()
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=gen, device=dev))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = call(b)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, eager)
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_a_step_through_all_of_them(dev):
    """Norm and rotation into a 4-bit cache, then windowed attention over it, token after token:
    what each step attends over is what the earlier ones wrote."""
    from tests.test_gpu_window_attention import OC_values, closed_form
    D, Hq, Hkv, bs, window, sinks = 128, 8, 2, 16, 40, 4
    gen = torch.Generator(device=dev).manual_seed(7)
    table = torch.randperm(9, generator=gen, device=dev)[:8].to(torch.int32)[None]
    caches = M.allocate_kv_cache(9, bs, Hkv, D, "int4", device=dev)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=gen, device=dev)).to(torch.bfloat16) for _ in range(2))
    inv = 10000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
    ang = torch.outer(torch.arange(128, device=dev, dtype=torch.float64), inv)
    cos, sin = ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)
    done = 0
    for n in (70, 1, 1, 5, 1, 30, 1):         # a prompt, tokens, a verify step, a chunk
        x = torch.randn(n, (Hq + 2 * Hkv) * D, generator=gen, device=dev).to(torch.bfloat16)
        pos = torch.arange(done, done + n, device=dev)
        slots = table[0, pos // bs].long() * bs + pos % bs
        q = M.qkv_norm_rope_and_cache(x, qw, kw, 1e-6, pos, cos, sin, caches[0], caches[1], slots, Hq, Hkv, D,
                                      "int4", caches[2], caches[3])
        done += n
        out = M.flash_attn_varlen_func(
            q=q, k=caches[0], v=caches[1], cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device=dev),
            max_seqlen_q=n, seqused_k=torch.tensor([done], dtype=torch.int32, device=dev), max_seqlen_k=done,
            softmax_scale=D ** -0.5, causal=True, block_table=table, k_scale=caches[2], v_scale=caches[3],
            window=window, sink_tokens=sinks)
        t = torch.arange(done, device=dev)
        blk, off = table[0, t // bs].long(), t % bs
        K, V = (OC_values(caches[i][blk, off].cpu().numpy(), caches[2 + i][blk, off].cpu().numpy(), "int4")
                for i in range(2))
        ref, tol = closed_form(q.double().cpu().numpy(), K, V, D ** -0.5, window, sinks, "int4",
                               caches[2][blk, off].double().cpu().numpy(), caches[3][blk, off].double().cpu().numpy())
        assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all(), n
        # the values of the new tokens are within half a step of a 4-bit code of what came in
        new = x.view(n, Hq + 2 * Hkv, D)[:, Hq + Hkv:].double().cpu().numpy()
        step = caches[3][blk, off].double().cpu().numpy()[done - n:, :, None]
        assert (np.abs(V[done - n:] - new) <= step * (0.5 + 8 * 2.0 ** -11)).all()


def test_refusals(dev):
    D, Hq, Hkv = 128, 4, 2
    qkv = torch.zeros(2, 8 * D, dtype=torch.bfloat16, device=dev)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    cos = torch.ones(4, D // 2, dtype=torch.bfloat16, device=dev)
    ids = torch.zeros(2, dtype=torch.int64, device=dev)
    c4, c16 = M.allocate_kv_cache(2, 16, Hkv, D, "int4", device=dev), M.allocate_kv_cache(2, 16, Hkv, D, device=dev)

    def call(**kw):
        a = dict(qkv=qkv, q_weight=w, k_weight=w, eps=1e-5, positions=ids, cos=cos, sin=cos, k_cache=c4[0],
                 v_cache=c4[1], slot_mapping=ids, num_heads=Hq, num_kv_heads=Hkv, head_dim=D,
                 kv_cache_dtype="int4", k_scale=c4[2], v_scale=c4[3])
        return M.qkv_norm_rope_and_cache(**{**a, **kw})

    call()
    for kw, what in ((dict(q_weight=w.float()), "q_weight must be bf16"), (dict(k_weight=w[:64]), "k_weight must be"),
                     (dict(qkv=qkv[:, :-8]), "qkv must be"), (dict(k_cache=c16[0], v_cache=c16[1]), "cache heads/dim"),
                     (dict(k_scale=None), "need k_scale"), (dict(k_scale=c4[2].float()), "scale caches must be"),
                     (dict(kv_cache_dtype="fp8", k_cache=c16[0], v_cache=c16[1]), "must be 'auto'"), (dict(kv_cache_dtype="auto"), "cache heads/dim"),
                     (dict(positions=ids.int()), "positions"), (dict(slot_mapping=ids[:1]), "slot_mapping"),
                     (dict(cos=cos.float(), sin=cos.float()), "cos/sin"),
                     (dict(q_out=torch.empty(2, Hq, D, device=dev)), "q_out must be")):
        with pytest.raises(ValueError, match=what):
            call(**kw)
    with pytest.raises(_lib.CooptError, match="eps"):
        call(eps=-1.0)
    with pytest.raises(_lib.CooptError, match="aligned"):
        call(qkv=torch.zeros(2 * 8 * D + 8, dtype=torch.bfloat16, device=dev)[1:-7].view(2, -1))
    with pytest.raises(ValueError, match="need k_scale"):
        M.reshape_and_cache_flash(qkv.view(2, 8, D)[:, :2], qkv.view(2, 8, D)[:, :2], c4[0], c4[1], ids, "int4")
    with pytest.raises(ValueError, match="uint8"):
        M.reshape_and_cache_flash(qkv.view(2, 8, D)[:, :2], qkv.view(2, 8, D)[:, :2], c4[0].view(torch.int8),
                                  c4[1].view(torch.int8), ids, "int4", c4[2], c4[3])
    # a 4-bit cache is not swapped
    with pytest.raises(ValueError, match="bf16 or int8"):
        M.swap_out_blocks(c4[0], ids, 4, c4[2])
