"""GPU: the speculative step of models with a sliding window, first tokens that stay visible and
head norms, over bf16, INT8 and 4-bit caches.

Every layer's calls are held against float64 as they run: the rotated, normed queries against the
closed form on the qkv rows, the attention against the closed form on what the cache then holds, at
the tolerances of the operators' own tests.  Then the step around them: an identical draft is
accepted, and graph replays equal eager steps.
"""
import numpy as np
import pytest
import torch

from iitj_llm_coopt_amd import fused
from iitj_llm_coopt_amd.spec_engine import HipOps, LlamaShape, PagedKV, RandomLlama, SpecDecoder
from test_gpu_qk_norm_int4 import norm_reference
from test_gpu_window_attention import closed_form

pytestmark = pytest.mark.gpu

SHAPE = dict(hidden=256, ffn=512, layers=2, heads=4, kv_heads=2, head_dim=64, vocab=1000)
WINDOWED = LlamaShape(**SHAPE, window=16, sink_tokens=2, qk_norm=True)
DRAFT = LlamaShape(hidden=128, ffn=256, layers=1, heads=4, kv_heads=2, head_dim=64, vocab=1000,
                   tie_embeddings=True, window=8, sink_tokens=1)


def cached(kv, layer, b, L):
    """float64 (K, V, s_k, s_v) of the first L tokens of sequence b, as attention defines them."""
    kc, vc, ks, vs = kv.layers[layer]
    pages = kv.block_table[b].long()
    t = torch.arange(L, device=kc.device)
    blk, off = pages[t // kv.block_size], t % kv.block_size
    scales = [None if s is None else s[blk, off].double().cpu().numpy() for s in (ks, vs)]
    vals = []
    for c, s in ((kc, scales[0]), (vc, scales[1])):
        x = c[blk, off]
        if kv.kv_dtype == "auto":
            vals.append(x.double().cpu().numpy())
        elif kv.kv_dtype == "int8":       # the kernel's keys and values are rounded to bf16
            y = torch.from_numpy(x.double().cpu().numpy() * s[..., None])
            vals.append(y.to(torch.bfloat16).double().numpy())
        else:
            n = x.cpu().numpy()
            codes = np.stack([n & 15, n >> 4], -1).reshape(*n.shape[:-1], -1).astype(np.float64) - 8
            vals.append(codes * s[..., None])
    return *vals, *scales


class CheckedOps(HipOps):
    """HipOps whose head norms and attention are compared with float64 at each call."""

    def __init__(self, device, shapes):
        super().__init__(device)
        self.shapes, self.calls = shapes, {"norm": 0, "attend": 0}

    def qkv_norm_epilogue(self, kv, layer, qkv, qw, kw, eps, pos, cos, sin, slots, H, Hkv, D):
        q = super().qkv_norm_epilogue(kv, layer, qkv, qw, kw, eps, pos, cos, sin, slots, H, Hkv, D)
        x = qkv.reduce() if isinstance(qkv, fused.LinearPartials) else qkv
        x = x.double().cpu().numpy().reshape(-1, H + 2 * Hkv, D)[:, :H]
        p = pos.reshape(-1).cpu().numpy()
        c, s = cos.double().cpu().numpy()[p], sin.double().cpu().numpy()[p]
        ref, mag = norm_reference(x, qw.double().cpu().numpy(), c, s, eps)
        assert (np.abs(q.double().cpu().numpy() - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * mag).all()
        self.calls["norm"] += 1
        return q

    def attend(self, kv, layer, q, meta, scale, window=None, sink_tokens=0):
        out = super().attend(kv, layer, q, meta, scale, window, sink_tokens)
        cu, lens = meta[0].tolist(), meta[1].tolist()
        for b, L in enumerate(lens):
            K, V, s_k, s_v = cached(kv, layer, b, L)
            rows = slice(cu[b], cu[b + 1])
            ref, tol = closed_form(q[rows].double().cpu().numpy(), K, V, scale, window, sink_tokens,
                                   kv.kv_dtype, s_k, s_v)
            assert (np.abs(out[rows].double().cpu().numpy() - ref) <= tol).all(), (layer, b, L)
        assert (window, sink_tokens) in self.shapes
        self.calls["attend"] += 1
        return out


def make(dev, kv, T=0.0, same=False, ops=None, P=37, steps=8, seed=0):
    t = RandomLlama(WINDOWED, dev, seed=seed + 1, std=0.2)
    for L in t.layers:
        L["q_norm"].copy_(torch.linspace(0.5, 1.5, 64))
        L["k_norm"].copy_(torch.linspace(1.5, 0.5, 64))
    d = t if same else RandomLlama(DRAFT, dev, seed=seed + 2, std=0.2)
    dec = SpecDecoder(t, d, 3, 3, P, steps, ops=ops, target_kv=kv, draft_kv=kv if same else "int4",
                      temperature=T, seed=seed, batch_buckets=(3,))
    g = torch.Generator(device=dev).manual_seed(seed + 3)
    prompts = torch.randint(0, WINDOWED.vocab, (3, P), generator=g, device=dev)
    dec.prefill(prompts, torch.rand(3, generator=g, device=dev))
    return dec


@pytest.mark.parametrize("kv", ["auto", "int8", "int4"])
def test_every_call_of_a_step_is_the_closed_form(dev, kv):
    """Prompts longer than both windows, then steps: prompt rows, catch-up, proposals, verify."""
    ops = CheckedOps(dev, {(16, 2), (8, 1)})
    dec = make(dev, kv, ops=ops)
    for _ in range(2):
        dec.step()
    # layers: target 2, draft 1; prompts, then per step a verify, a catch-up and 2 proposals
    assert ops.calls == {"norm": 2 * 3, "attend": 2 * 3 + 1 + 2 * 3}


@pytest.mark.parametrize("kv", ["auto", "int8", "int4"])
def test_graph_replays_match_eager_steps(dev, kv):
    a, b = (make(dev, kv, seed=5) for _ in range(2))
    a.step()
    b.step()
    b.capture()
    for i in range(4):
        b.replay()
        a.step()
        torch.cuda.synchronize(dev)
        _ = torch.randn(1000, device=dev).sum().item()  # unrelated eager work between replays
        assert torch.equal(a.n, b.n) and torch.equal(a.hist, b.hist), i


def test_sizes(dev):
    assert WINDOWED.params() - LlamaShape(**SHAPE).params() == 2 * 2 * 64
    kv = PagedKV(WINDOWED, 2, 64, "int4", dev)
    assert kv.nbytes() == 2 * 2 * kv.num_blocks * 16 * 2 * (32 + 2)
    t = RandomLlama(WINDOWED, dev)
    assert all(torch.equal(t.to(dev).layers[1][k], t.layers[1][k]) for k in ("q_norm", "k_norm"))
