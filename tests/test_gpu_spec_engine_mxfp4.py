"""GPU: the speculative step of models with 4-bit weights, 4-bit activations, norms, gates and scales on their
branches.

Every projection and residual norm is held against float64 as it runs, at the tolerances of the operators'
own tests; then the step around them: graph replays equal eager steps, and a copy of the model in bf16 on the
CPU holds the same weights.
"""
import numpy as np
import pytest
import torch

from iitj_llm_coopt_amd import fused
from iitj_llm_coopt_amd.mxfp4 import MXFP4Weight
from iitj_llm_coopt_amd.spec_engine import HipOps, LlamaShape, RandomLlama, SpecDecoder
from test_gpu_mxfp4 import quantized
from test_gpu_residual_norm import check, reference

pytestmark = pytest.mark.gpu

SIZES = dict(hidden=256, ffn=512, heads=4, kv_heads=2, head_dim=64, vocab=1000)
TARGET = LlamaShape(**SIZES, layers=2, post_norm=True, branch_gate=True, branch_scale=0.5, residual_scale=1.25)
DRAFT = LlamaShape(hidden=128, ffn=1024, heads=4, kv_heads=2, head_dim=64, vocab=1000, layers=1, tie_embeddings=True,
                   post_norm=True)
WHOLE = ("qkv", "o", "gate_up", "down", "lm_head")


class CheckedOps(HipOps):
    def __init__(self, device):
        super().__init__(device)
        self.calls = {"linear": 0, "norm": 0}

    def linear(self, x, w, out=None, defer_reduce=False):
        y = super().linear(x, w, out=out, defer_reduce=defer_reduce)
        assert isinstance(w, MXFP4Weight)
        got = (y.reduce() if isinstance(y, fused.LinearPartials) else y).double().cpu().numpy().reshape(-1, w.shape[0])
        xd, wd = x.double().cpu().numpy().reshape(-1, w.shape[1]), w.dequantize().double().cpu().numpy()
        if w.activations == "mxfp4":
            xd = quantized(xd)
        ref, mag = xd @ wd.T, np.abs(xd) @ np.abs(wd).T
        assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + (w.shape[1] / 32 + 160) * 2.0 ** -22 * mag).all()
        self.calls["linear"] += 1
        return y

    def linear_silu(self, x, w):
        y = super().linear_silu(x, w)
        gu = self.linear(x, w)
        assert torch.equal(y, fused.silu_and_mul(gu))
        return y

    def residual_norm(self, x, residual, w, eps, post_weight, gate, branch_scale, residual_scale):
        full = x.reduce() if isinstance(x, fused.LinearPartials) else x
        ref = reference(full, residual, w, eps, post_weight, gate, branch_scale, residual_scale)
        out = super().residual_norm(x, residual, w, eps, post_weight, gate, branch_scale, residual_scale)
        check(out, residual, ref)
        self.calls["norm"] += 1
        return out


def make(dev, activations, ops=None, B=3, P=37, steps=8, seed=0):
    t = RandomLlama(TARGET, dev, seed=seed + 1, std=0.2, packed=WHOLE, weights="mxfp4", activations=activations)
    d = RandomLlama(DRAFT, dev, seed=seed + 2, std=0.2, packed=WHOLE, weights="mxfp4", activations=activations)
    for model in (t, d):
        for i, L in enumerate(model.layers):
            for k in L:
                if k.endswith(("_post", "_gate")):
                    L[k].copy_(torch.linspace(0.5 + 0.1 * i, 1.5, model.s.hidden))
    dec = SpecDecoder(t, d, B, 3, P, steps, ops=ops, temperature=0.0, seed=seed, batch_buckets=(B,))
    g = torch.Generator(device=dev).manual_seed(seed + 3)
    dec.prefill(torch.randint(0, 1000, (B, P), generator=g, device=dev), torch.rand(B, generator=g, device=dev))
    return dec


@pytest.mark.parametrize("activations", ["bf16", "mxfp4"])
@pytest.mark.parametrize("B", [3, 24])
def test_every_call_of_a_step_is_the_definition(dev, activations, B):
    """Prompts, then steps: prompt rows, catch-up, proposals, verify."""
    ops = CheckedOps(dev)
    dec = make(dev, activations, ops=ops, B=B)
    for _ in range(2):
        dec.step()
    # a forward: four projections a layer (in a step gate_up twice here is one), the logits; two sums a layer
    forwards = {"t": 1 + 2, "d": 1 + 2 * 3}
    assert ops.calls["norm"] == 2 * 2 * forwards["t"] + 2 * forwards["d"]
    assert ops.calls["linear"] == (4 * 2 + 1) * forwards["t"] + (4 + 1) * forwards["d"]


@pytest.mark.parametrize("activations", ["bf16", "mxfp4"])
def test_graph_replays_match_eager_steps(dev, activations):
    a, b = (make(dev, activations, seed=5) for _ in range(2))
    a.step()
    b.step()
    b.capture()
    for i in range(4):
        b.replay()
        a.step()
        torch.cuda.synchronize(dev)
        _ = torch.randn(1000, device=dev).sum().item()  # unrelated eager work between replays
        assert torch.equal(a.n, b.n) and torch.equal(a.hist, b.hist), i


def test_copies_hold_the_same_weights(dev):
    m = RandomLlama(TARGET, dev, packed=WHOLE, weights="mxfp4", activations="mxfp4")
    on_cpu, again = m.to("cpu"), m.to(dev)
    for L, C, G in zip(m.layers, on_cpu.layers, again.layers):
        for k, w in L.items():
            if isinstance(w, MXFP4Weight):
                assert torch.equal(w.dequantize().cpu(), C[k]) and torch.equal(w.codes, G[k].codes)
                assert torch.equal(w.scales, G[k].scales) and G[k].activations == "mxfp4"
            else:
                assert torch.equal(w.cpu(), C[k]) and torch.equal(w, G[k])
    assert torch.equal(m.lm_head.dequantize().cpu(), on_cpu.lm_head)
    tied = RandomLlama(DRAFT, dev, packed=WHOLE, weights="mxfp4")
    assert torch.equal(tied.lm_head.dequantize().cpu(), tied.to("cpu").lm_head)


def test_sizes_and_refusals(dev):
    plain = LlamaShape(**SIZES, layers=2)
    assert TARGET.params() - plain.params() == 2 * 4 * 256 and not plain.scaled_branches and TARGET.scaled_branches
    with pytest.raises(ValueError, match="need 4-bit weights"):
        RandomLlama(plain, dev, activations="mxfp4")
    with pytest.raises(ValueError, match="must be"):
        RandomLlama(plain, dev, weights="int4")
    with pytest.raises(ValueError, match="need a GPU"):
        RandomLlama(plain, "cpu", weights="mxfp4")
