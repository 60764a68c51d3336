"""CPU: weights and partial sums of derived classes are taken as what they are."""
import pytest
import torch

from iitj_llm_coopt_amd import _lib, fused
from iitj_llm_coopt_amd.mxfp4 import MXFP4Weight


class Weight(MXFP4Weight):
    pass


class Partials(fused.LinearPartials):
    pass


def test_derived_classes():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    w = Weight(u8(16, 16), u8(16, 1), u8(8704))
    for call in (lambda: fused.linear(bf(2, 32), w), lambda: fused.linear_silu(bf(2, 32), w)):
        with pytest.raises(_lib.CooptError, match="no CPU fallback"):
            call()
    part = Partials(u8(4 * 16 * 64), 1, 2, 16, 64, torch.Size((2, 64)), torch.device("cpu"))
    with pytest.raises(_lib.CooptError, match="no CPU fallback"):
        fused.residual_norm(part, bf(2, 64), bf(64), 1e-5)
