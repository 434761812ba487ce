"""GPU: the MXFP8 operators where values are very large, very small or not finite."""

from __future__ import annotations

import pytest
import torch

from mxfp8_cases import activation, check_moe, check_product, random_weight, routing, values

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


def _far_groups(m, k, dev):
    """bf16 groups with maxima of 2^20 to 2^127 (scale exponents to both sides of 143), values up to 2^200 below them and
    zeros of both signs among them."""
    gen = torch.Generator(device=dev).manual_seed(m + k)
    exponent = torch.randint(20, 127, (m, k // 32), generator=gen, device=dev).double().repeat_interleave(32, 1)
    below = torch.randint(0, 200, (m, k), generator=gen, device=dev).double()
    below[torch.rand(m, k, generator=gen, device=dev) < 0.6] = 0
    x = (torch.randn(m, k, generator=gen, device=dev).double() * torch.exp2(exponent - below)).to(torch.bfloat16)
    x[torch.rand(m, k, generator=gen, device=dev) < 0.1] = -0.0
    x[torch.rand(m, k, generator=gen, device=dev) < 0.1] = 0.0
    assert x.isfinite().all()
    return x


def test_rows_of_large_values(cuda_device):
    from vllm_qdq_plugin.qdq import mxfp8_qdq, mxfp8_quantize, mxfp8_rows
    x = _far_groups(300, 544, cuda_device)
    rows = mxfp8_rows(x)
    codes, scales = mxfp8_quantize(x)
    assert int(scales.min()) < 143 < int(scales.max())
    assert torch.equal(rows.codes, codes) and torch.equal(rows.scales, scales)
    assert torch.equal(rows.dequantize(), mxfp8_qdq(x))


@pytest.mark.parametrize("m", [2, 50, 300])
def test_products_of_large_16_bit_rows(cuda_device, m):
    """Quantised inside the product of few rows, by the pass before it, and by the experts' layout pass."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    dev, k, n, e = cuda_device, 288, 200, 3
    x = _far_groups(m, k, dev) * 2.0 ** -60  # the sums stay in bf16's range; groups keep exponents beyond 143 - 60
    big = _far_groups(m, k, dev)
    codes, scales = random_weight(e, n, k, seed=1, dev=dev)
    w, wm = prepare_mxfp8_weight(codes[0], scales[0]), prepare_mxfp8_moe_weight(codes, scales)
    ids, sid, eid, ntp, tw = routing(m, e, 2, 16, 1, dev)
    rows = mxfp8_rows(x)
    a = values(rows.codes, rows.scales)
    check_product(mxfp8_linear(x, w), a, values(codes[0], scales[0]), what=f"m={m}")
    check_moe(mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, 16, 2, True), a, codes, scales, ids, f"experts m={m}", tw)
    # the codes inside are those of mxfp8_rows, whatever the exponent: the same product of both
    rows = mxfp8_rows(big)
    assert int(rows.scales.max()) > 143
    same = lambda a, b: torch.equal(a.nan_to_num(1, 2, 3), b.nan_to_num(1, 2, 3))  # noqa: E731
    assert same(mxfp8_linear(big, w), mxfp8_linear(rows, w))
    assert same(mxfp8_moe_linear(big, wm, sid, eid, ntp, tw, 16, 2, True), mxfp8_moe_linear(rows, wm, sid, eid, ntp, tw, 16, 2, True))


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("m", [3, 70, 300])
def test_products_of_rows_that_are_not_finite(cuda_device, m, bad):
    """The rule of mxfp8_qdq: a NaN makes its row's outputs NaN; an infinity gives its group the scale 2^-127, in which
    the infinity saturates to 448 2^-127 and the finite values beside it to as little.  Other rows are as they were."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_qdq, mxfp8_rows
    dev, n, k, e = cuda_device, 160, 416, 2
    x = activation(m, k, torch.bfloat16, 9, dev)
    x[m // 2, 37] = bad
    codes, scales = random_weight(e, n, k, seed=4, dev=dev)
    w, wm = prepare_mxfp8_weight(codes[0], scales[0]), prepare_mxfp8_moe_weight(codes, scales)
    ids, sid, eid, ntp, tw = routing(m, e, 1, 16, 1, dev)
    q = mxfp8_qdq(x).double()
    clean = torch.arange(m, device=dev) != m // 2
    for a in (x, mxfp8_rows(x)):
        out, grouped = mxfp8_linear(a, w), mxfp8_moe_linear(a, wm, sid, eid, ntp, tw, 16, 1, False)
        if bad != bad:
            assert out[m // 2].isnan().all() and grouped[m // 2].isnan().all()
        else:
            assert q.isfinite().all() and q[m // 2, 32:64].abs().max() <= 448 * 2.0 ** -127
            check_product(out[~clean], q[~clean], values(codes[0], scales[0]), what=f"m={m}")
        check_product(out[clean], q[clean], values(codes[0], scales[0]), what=f"m={m}")
        rest = clean.nonzero()[:, 0]
        check_moe(grouped[rest], q[rest], codes, scales, ids[rest.cpu().numpy()], f"experts m={m}")


@pytest.mark.parametrize("m,n,k", [(1, 50257, 64), (64, 20000, 96), (1, 64, 131072), (3, 130, 262144), (70, 128, 65536),
                                   (100000, 8, 32)])
def test_linear_of_extreme_shapes(cuda_device, m, n, k):
    """More W tiles than SMs for one token, K beyond what a CTA keeps, many rows of a narrow weight."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    x = activation(m, k, torch.bfloat16, m + n, cuda_device)
    codes, scales = random_weight(n, k, seed=n, dev=cuda_device)
    w = prepare_mxfp8_weight(codes, scales)
    rows = mxfp8_rows(x)
    a, exact_w = values(rows.codes, rows.scales), values(codes, scales)
    for given in (x, rows):
        check_product(mxfp8_linear(given, w), a, exact_w, what=f"{m}x{n}x{k}")


@pytest.mark.parametrize("m,e,n,k", [(3, 1, 64, 131072), (40, 2, 40000, 32), (500, 1, 64, 32), (9, 500, 32, 64)])
def test_experts_of_extreme_shapes(cuda_device, m, e, n, k):
    """One expert, many, wide and long ones; num_tokens_post_padded beyond the sorted slots counts as all of them."""
    from vllm_qdq_plugin.gemm import mxfp8_moe_linear, prepare_mxfp8_moe_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    x = activation(m, k, torch.bfloat16, m + n, cuda_device)
    codes, scales = random_weight(e, n, k, seed=n, dev=cuda_device)
    w = prepare_mxfp8_moe_weight(codes, scales)
    ids, sid, eid, ntp, tw = routing(m, e, 1, 16, 3, cuda_device)
    live = int(ntp)
    rows = mxfp8_rows(x)
    a = values(rows.codes, rows.scales)
    for given in (x, rows):
        out = mxfp8_moe_linear(given, w, sid[:live].contiguous(), eid, ntp * 1000, tw, 16, 1, True)
        check_moe(out, a, codes, scales, ids, f"m={m} e={e}", tw)


@pytest.mark.parametrize("m,k", [(3, 20480), (1300, 2880), (5, 1024), (7, 512), (2, 65536)])
def test_rmsnorm_of_far_rows_between_others(cuda_device, m, k):
    """Every form of the kernel, the sum taken from the residual's: far rows as in 64 bits, the others to the bit as in a
    call without far ones."""
    from vllm_qdq_plugin.qdq import mxfp8_quantize, rmsnorm_mxfp8
    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(k)
    x, r = (torch.randn(m, k, generator=gen, device=dev).to(torch.bfloat16) for _ in range(2))
    w = (1 + 0.1 * torch.randn(k, generator=gen, device=dev)).to(torch.bfloat16)
    near = rmsnorm_mxfp8(x, w, r, 0.0, norm_out=True)
    far = torch.arange(m, device=dev) % 2 == 1
    scale = torch.where(torch.arange(m, device=dev) % 4 == 1, 2.0 ** 100, 2.0 ** -90)[:, None]
    x2, r2 = (torch.where(far[:, None], t.double() * scale, t.double()).to(torch.bfloat16) for t in (x, r))
    rows, h, y = rmsnorm_mxfp8(x2, w, r2, 0.0, norm_out=True)
    assert torch.equal(h, (x2.float() + r2.float()).to(torch.bfloat16))
    assert torch.equal(y[~far], near[2][~far]) and torch.equal(rows.codes[~far], near[0].codes[~far])
    d = h.double()
    want = d / d.square().mean(1, keepdim=True).sqrt() * w.double()
    assert ((y.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -17) * want.abs() + 2.0 ** -134).all()
    codes, scales = mxfp8_quantize(y)
    assert torch.equal(rows.codes, codes) and torch.equal(rows.scales, scales)
    again = rmsnorm_mxfp8(x2, w, r2, 0.0)[0]
    assert torch.equal(again.codes, codes) and torch.equal(again.scales, scales)
