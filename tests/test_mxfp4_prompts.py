"""CPU: prompts of more rows than a product with 4-bit weights takes.  The product is stood in for."""
import pytest
import torch

from iitj_llm_coopt_amd import _lib, spec_engine
from iitj_llm_coopt_amd.mxfp4 import MAX_ROWS, MXFP4Weight


class Ops:
    def __init__(self):
        self.rows = []

    def linear(self, x, w, out=None, defer_reduce=False):
        assert x.shape[0] <= MAX_ROWS and not defer_reduce
        self.rows.append(x.shape[0])
        y = x[:, :1].expand(-1, w.shape[0]) + torch.arange(w.shape[0], dtype=x.dtype)
        return y if out is None else out.copy_(y)


@pytest.mark.parametrize("rows,calls", [(5, [5]), (MAX_ROWS, [MAX_ROWS]), (MAX_ROWS + 3, [MAX_ROWS, 3]),
                                        (2 * MAX_ROWS + 1, [MAX_ROWS, MAX_ROWS, 1])])
def test_prompt_rows_go_in_several_products(rows, calls):
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    w = MXFP4Weight(u8(4, 16), u8(4, 1), u8(_lib.load().coopt_mxfp4_packed_bytes(4, 32)))
    dec = object.__new__(spec_engine.SpecDecoder)
    dec.ops = Ops()
    x = (torch.arange(rows) % 100).to(torch.bfloat16)[:, None].expand(rows, 32)
    y = dec._prompt_linear(x, w)
    assert dec.ops.rows == calls and y.shape == (rows, 4)
    assert torch.equal(y, x[:, :4] + torch.arange(4, dtype=torch.bfloat16))
