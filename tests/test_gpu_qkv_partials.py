"""GPU: the epilogues of a qkv projection from its split-K partial sums, at the rows of a draft and a
verify step and into every cache type: bit for bit what they make of the reduced projection."""
import pytest
import torch

import iitj_llm_coopt_amd as M
from iitj_llm_coopt_amd import fused

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 32, 160])
@pytest.mark.parametrize("kv", ["auto", "int8", "int4"])
@pytest.mark.parametrize("D,Hq,Hkv,K", [(128, 32, 8, 4096), (64, 32, 8, 2048)])
@pytest.mark.parametrize("norm", [False, True])
def test_epilogues_of_partial_sums(dev, norm, D, Hq, Hkv, K, kv, T):
    gen = torch.Generator(device=dev).manual_seed(T)
    w = (torch.randn((Hq + 2 * Hkv) * D, K, generator=gen, device=dev) * 0.05).to(torch.bfloat16)
    h = torch.randn(T, K, generator=gen, device=dev).to(torch.bfloat16)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=gen, device=dev)).to(torch.bfloat16) for _ in range(2))
    cos, sin = (torch.randn(400, D // 2, generator=gen, device=dev).to(torch.bfloat16) for _ in range(2))
    pos = torch.randint(0, 400, (T,), generator=gen, device=dev)
    slots = torch.randperm(16 * 12, generator=gen, device=dev)[:T].contiguous()
    slots[T // 2] = -1
    part = fused.linear(h, w, defer_reduce=True)
    assert isinstance(part, fused.LinearPartials) and part.ks > 1
    got = []
    for qkv in (part, part.reduce()):
        kc, vc, ks, vs = M.allocate_kv_cache(12, 16, Hkv, D, kv, device=dev)
        if norm:
            q = M.qkv_norm_rope_and_cache(qkv, qw, kw, 1e-5, pos, cos, sin, kc, vc, slots, Hq, Hkv, D, kv, ks, vs)
        else:
            q = M.qkv_rope_and_cache(qkv, pos, cos, sin, kc, vc, slots, Hq, Hkv, D, kv, ks, vs)
        got.append([t for t in (q, kc, vc, ks, vs) if t is not None])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    fresh = M.allocate_kv_cache(12, 16, Hkv, D, kv, device=dev)[0]
    assert torch.equal(got[0][1], fresh) == (T == 1)      # its one row is padding: no entry is written
    assert got[0][0].isfinite().all()
