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


@pytest.mark.parametrize("k", [64, 544, 2880, 8192, 32800])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
def test_rmsnorm_over_the_range_of_bf16(cuda_device, k, eps):
    """Rows whose squares fp32 does not hold, next to ordinary ones: the norm is that of 64 bits."""
    from vllm_qdq_plugin.qdq import mxfp8_quantize, rmsnorm_mxfp8
    dev = cuda_device
    exponents = [126, 100, 70, 63, 58, 40, 0, -40, -50, -62, -70, -100, -125, -131]
    gen = torch.Generator(device=dev).manual_seed(k)
    x = torch.rand(len(exponents), k, generator=gen, device=dev).double() + 0.5
    x = x * torch.exp2(torch.tensor(exponents, device=dev).double())[:, None]
    x[:, 1::2] *= -1
    x[:, 5] *= 2.0 ** -40  # one small value among the others
    x = x.to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(k, generator=gen, device=dev)).to(torch.bfloat16)
    rows, _, y = rmsnorm_mxfp8(x, w, eps=eps, norm_out=True)
    d = x.double()
    want = d / (d.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
    # half a bf16 step and the fp32 path (sums, rsqrtf, products: 2^-17), absolutely half a step of the smallest numbers
    bound = (2.0 ** -8 + 2.0 ** -17) * want.abs() + 2.0 ** -134
    assert x.isfinite().all() and ((y.double() - want).abs() <= bound).all()
    codes, scales = mxfp8_quantize(y)
    assert torch.equal(rows.codes, codes) and torch.equal(rows.scales, scales)


def test_rmsnorm_of_infinite_rows(cuda_device):
    """An infinity makes its own row what the formula gives: 0 where h is finite, NaN where it is not."""
    from vllm_qdq_plugin.qdq import rmsnorm_mxfp8
    x = torch.ones(3, 96, dtype=torch.bfloat16, device=cuda_device)
    x[1, 7] = float("inf")
    y = rmsnorm_mxfp8(x, x[0], norm_out=True)[2]
    assert y[1, 7].isnan() and not y[1, torch.arange(96, device=cuda_device) != 7].any()
    assert torch.equal(y[0], y[2]) and (y[0] == 1).all()
