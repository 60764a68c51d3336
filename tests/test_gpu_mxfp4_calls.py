"""GPU: calls around the products with 4-bit weights that the operators' own tests do not make."""
import pytest
import torch

from iitj_llm_coopt_amd import fused
from test_gpu_mxfp4 import make_weight, small_numbers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("activations", ["bf16", "mxfp4"])
def test_rows_that_grow_keep_one_workspace(dev, activations):
    """On a stream of its own: what stays allocated is the last workspace, and a workspace that is outgrown while its
    product still runs changes nothing."""
    w, _ = make_weight(dev, 64, 8192, 3, activations, integers=True)
    x = small_numbers(dev, (2064, 8192), 3)
    sizes = range(80, 2065, 32)
    assert any(w.plan(m)[0] for m in sizes)
    want = fused.linear(x, w)
    torch.cuda.synchronize(dev)
    side = torch.cuda.Stream(device=dev)
    with torch.cuda.stream(side):
        before = torch.cuda.memory_allocated(dev)
        out = [fused.linear(x[:m], w) for m in sizes]
        after = torch.cuda.memory_allocated(dev) - sum(-(-o.nbytes // 512) * 512 for o in out)
    side.synchronize()
    assert after - before <= max(w.plan(m)[0] for m in sizes) * 9 // 8 + 512
    for m, o in zip(sizes, out):
        assert torch.equal(o, want[:m])
