"""GPU: the MXFP8 operators where values are very large, very small or not finite."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _gate_exact(x):
    g, u = x.double().chunk(2, 1)
    return g / (1 + torch.exp(-g)) * u


def _gate_rel(g):
    """Worst relative error of the gate in fp32: exp(-|g| / 2), whose rounded argument and constant cost |g| 2^-24 together
    and ex2 2 ulp, counts twice; the sum, the reciprocal and four products are half an ulp or one each: below this."""
    return g.abs() * 2.0 ** -23 + 2.0 ** -20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gate_codes_are_those_of_the_exact_product(cuda_device, dtype):
    """No code differs where the worst case of the rounding errors cannot change it, and where it can, no more than twice
    as many as with the formula in plain fp32 (expf and a division, as many roundings), and 8 for chance at small counts."""
    from vllm_qdq_plugin.qdq import mxfp8_quantize, silu_mul_mxfp8
    m, k = 2048, 14336
    plain_differ = differ = 0
    for seed in range(2):
        gen = torch.Generator(device=cuda_device).manual_seed(seed)
        x = (torch.randn(m, 2 * k, generator=gen, device=cuda_device) * 2).to(dtype)
        codes = silu_mul_mxfp8(x).codes
        y, rel = _gate_exact(x), _gate_rel(x.double()[:, :k])
        lo, hi = (mxfp8_quantize((y * (1 + s * rel)).to(dtype))[0] for s in (-1, 1))
        want = mxfp8_quantize(y.to(dtype))[0]
        assert not ((codes != want) & (lo == hi)).any()
        g, u = x.float().chunk(2, 1)
        plain = mxfp8_quantize((g / (1 + torch.exp(-g)) * u).to(dtype))[0]
        plain_differ, differ = plain_differ + int((plain != want).sum()), differ + int((codes != want).sum())
    assert differ <= 2 * plain_differ + 8, (differ, plain_differ)


@pytest.mark.parametrize("gate", [-80.0, -88.0, -96.0, -103.0, -110.0, -130.0, -160.0, 88.0])
def test_gate_of_far_gates_and_large_factors(cuda_device, gate):
    """silu(g) alone falls below what fp32 holds, times u it is an ordinary number (bf16 reaches 3e38)."""
    from vllm_qdq_plugin.qdq import silu_mul_mxfp8
    checked = 0
    for up in (1.0, -1e30, 3e38):
        x = torch.full((1, 64), gate, dtype=torch.bfloat16, device=cuda_device)
        x[0, 32:] = up
        want = _gate_exact(x)
        if 2.0 ** -108 < float(want[0, 0].abs()) < torch.finfo(torch.bfloat16).max:  # the range of bf16 and of normal codes
            got = silu_mul_mxfp8(x).dequantize().double()
            # half a bf16 step, then E4M3 of a group of equal values: half a step (2^-4), or saturation at 448 of up to
            # 512 (2^-3)
            assert ((got - want).abs() <= (2.0 ** -8 + 2.0 ** -3) * want.abs()).all(), (up, got[0, 0], want[0, 0])
            checked += 1
    assert checked
