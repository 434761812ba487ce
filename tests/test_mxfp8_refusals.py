"""CPU: tensors of any rank are refused by the MXFP8 row operators in the same words."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("shape", [(), (64,), (2, 2, 64)])
def test_rows_are_two_dimensional(shape):
    from vllm_qdq_plugin.qdq import mxfp8_rows, rmsnorm_mxfp8, silu_mul_mxfp8
    x, w = torch.zeros(shape, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    for call in (lambda: mxfp8_rows(x), lambda: silu_mul_mxfp8(x), lambda: rmsnorm_mxfp8(x, w)):
        with pytest.raises(AssertionError, match=f"2D tensors, but got {len(shape)}D"):
            call()
