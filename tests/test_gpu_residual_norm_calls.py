"""GPU: calls of the residual norm that its documentation allows and its other tests do not make."""
import numpy as np
import pytest
import torch

from iitj_llm_coopt_amd import fused
from test_gpu_residual_norm import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["token", "channel"])
@pytest.mark.parametrize("off", [1, 3, 8])
def test_gates_at_any_offset(dev, kind, off):
    """A gate cut from a wider tensor, or from within a vector, where its rows start off a 16-byte border."""
    T, H = 5, 264
    x, residual, weight, pw, gv = inputs(dev, T, H, kind, True)
    new = torch.empty_like(residual)
    want = fused.residual_norm(x, residual, weight, 1e-5, pw, gv, residual_out=new)
    if kind == "token":
        gates = [torch.zeros(T, 400, dtype=torch.bfloat16, device=dev)[:, off:off + H],
                 torch.zeros(T * H + 8, dtype=torch.bfloat16, device=dev)[off:off + T * H].view(T, H)]
    else:
        gates = [torch.zeros(H + 8, dtype=torch.bfloat16, device=dev)[off:off + H]]
    for gate in gates:
        gate.copy_(gv)
        other = torch.empty_like(residual)
        got = fused.residual_norm(x, residual, weight, 1e-5, pw, gate, residual_out=other)
        assert torch.equal(got, want) and torch.equal(other, new)
