"""GPU: MXFP8 rows, RMSNorm with residual and the gated activation, against 64-bit plain forms.

Codes are compared exactly: with mxfp8_quantize (itself bit-exact with the
reference) of the 16-bit tensor they are made from.  That tensor is the norm's
16-bit output where it is returned; for the gate, whose 16-bit value is not,
every group is compared whose 64-bit values all lie clear of a rounding border.
"""

from __future__ import annotations

import pytest
import torch

from mxfp8_cases import half_step

pytestmark = pytest.mark.gpu

# fp32 path of the norm: a sum of squares (fma chains of at most 64 terms, then trees: 2^-17 at the worst, halved
# by the square root), rsqrtf (2 ulp) and three products: below 2^-17 of the value.
NORM_REL = 2.0 ** -17


def gate_rel(g):
    """fp32 path of the gate: exp(-|g|) = 2^(|g| log2 e), whose rounded argument and constant cost |g| 2^-24 each;
    ex2 and the division 2 ulp each, the sum and two products half an ulp: below 2^-20."""
    return g.abs() * 2.0 ** -23 + 2.0 ** -20



def _quantize(y):
    from vllm_qdq_plugin.qdq import mxfp8_quantize
    return mxfp8_quantize(y)


def _same_rows(rows, y):
    codes, scales = _quantize(y)
    assert torch.equal(rows.codes, codes) and torch.equal(rows.scales, scales)


def _wide(m, k, dtype, seed, dev):
    """Values over many binades, zeros, subnormals and large ones among them."""
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(m, k, generator=g, device=dev)
    x = x * torch.exp2(torch.randint(-14, 8, (m, k), generator=g, device=dev).float())
    x[torch.rand(m, k, generator=g, device=dev) < 0.05] = 0.0
    x = x.to(dtype)
    x[:, : min(k, 32)] = 0          # a group of zeros
    if m > 1:
        x[1, -32:] = torch.finfo(dtype).smallest_normal / 4   # a group of subnormals
        x[1, -1] = -0.0
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 4096), (3, 96), (17, 544), (129, 1056), (1000, 2880)])
def test_rows_are_the_codes_of_mxfp8_quantize(cuda_device, m, k, dtype):
    from vllm_qdq_plugin.qdq import mxfp8_qdq, mxfp8_rows
    x = _wide(m, k, dtype, m + k, cuda_device)
    rows = mxfp8_rows(x)
    _same_rows(rows, x)
    assert rows.dtype == dtype and rows.shape == x.shape
    if dtype == torch.bfloat16:  # every bf16 scale is a bf16 value: the decode is exact
        assert torch.equal(rows.dequantize().float(), mxfp8_qdq(x).float())


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_rows_hold_infinities_and_nan_within_their_group(cuda_device, bad):
    from vllm_qdq_plugin.qdq import mxfp8_rows, rmsnorm_mxfp8
    x = _wide(5, 256, torch.bfloat16, 3, cuda_device)
    clean = mxfp8_rows(x)
    y = x.clone()
    y[2, 70] = bad
    rows = mxfp8_rows(y)
    _same_rows(rows, y)
    keep = torch.ones_like(x, dtype=torch.bool)
    keep[2, 64:96] = False
    assert torch.equal(rows.codes[keep], clean.codes[keep])
    # through the norm it reaches its own row alone
    w = torch.ones(256, dtype=torch.bfloat16, device=cuda_device)
    a, b = rmsnorm_mxfp8(x, w)[0], rmsnorm_mxfp8(y, w)[0]
    others = torch.arange(5, device=cuda_device) != 2
    assert torch.equal(a.codes[others], b.codes[others]) and torch.equal(a.scales[others], b.scales[others])


def test_rows_from_codes_and_strided_inputs(cuda_device):
    from vllm_qdq_plugin.qdq import Mxfp8Rows, mxfp8_quantize, mxfp8_rows, rmsnorm_mxfp8, silu_mul_mxfp8
    x = _wide(37, 288, torch.bfloat16, 5, cuda_device)
    want = mxfp8_rows(x)
    rows = Mxfp8Rows.from_codes(*mxfp8_quantize(x))
    assert torch.equal(rows.codes, want.codes) and torch.equal(rows.scales, want.scales)
    w = torch.randn(288, device=cuda_device).to(torch.bfloat16)
    for view in (torch.cat([x, x], 1)[:, :288],                       # padded rows, 16-byte aligned
                 torch.nn.functional.pad(x, (8, 8))[:, 8:296],        # 16-byte aligned, off the 32-byte grid
                 torch.nn.functional.pad(x, (1, 2))[:, 1:289],        # rows off the 16-byte grid
                 x.t().contiguous().t(),                              # strided along K
                 torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(37, 288)):  # base off the grid
        assert torch.equal(view, x)
        got = mxfp8_rows(view)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        a, b = rmsnorm_mxfp8(view, w, view)[:2], rmsnorm_mxfp8(x, w, x)[:2]
        assert torch.equal(a[0].codes, b[0].codes) and torch.equal(a[1], b[1])
    wide = torch.cat([x, x.flip(0), x], 1)[:, : 2 * 288]
    assert torch.equal(silu_mul_mxfp8(wide).codes, silu_mul_mxfp8(wide.contiguous()).codes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 4096), (9, 256), (8, 288), (33, 512), (7, 544), (20, 1024), (5, 1056),
                                 (300, 2880), (2, 8192), (3, 8224), (2, 32768), (2, 32800), (1, 65536)])
@pytest.mark.parametrize("with_residual", [True, False])
def test_rmsnorm_against_64_bits(cuda_device, m, k, dtype, with_residual):
    from vllm_qdq_plugin.qdq import rmsnorm_mxfp8
    g = torch.Generator(device=cuda_device).manual_seed(m * 7 + k)
    x = torch.randn(m, k, generator=g, device=cuda_device).to(dtype)
    w = torch.randn(k, generator=g, device=cuda_device).to(dtype)
    r = (torch.randn(m, k, generator=g, device=cuda_device) * 3).to(dtype) if with_residual else None
    rows, h, y = rmsnorm_mxfp8(x, w, r, 1e-5, norm_out=True)
    if with_residual:
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
    else:
        assert h is None
    d = (h if with_residual else x).double()
    want = d * torch.rsqrt(d.square().mean(1, keepdim=True) + 1e-5) * w.double()
    bound = (half_step(dtype) + NORM_REL) * want.abs() + torch.finfo(dtype).tiny * half_step(dtype)
    assert ((y.double() - want).abs() <= bound).all()
    _same_rows(rows, y)
    again = rmsnorm_mxfp8(x, w, r, 1e-5)
    assert again[2] is None and torch.equal(again[0].codes, rows.codes) and torch.equal(again[0].scales, rows.scales)


def test_rmsnorm_of_zero_rows_and_zero_eps(cuda_device):
    from vllm_qdq_plugin.qdq import rmsnorm_mxfp8
    x = torch.zeros(3, 64, dtype=torch.bfloat16, device=cuda_device)
    w = torch.ones(64, dtype=torch.bfloat16, device=cuda_device)
    rows, _, y = rmsnorm_mxfp8(x, w, eps=1e-6, norm_out=True)
    assert not y.any() and not rows.codes.any()
    x[1] = 2.0
    _, _, y = rmsnorm_mxfp8(x, w, eps=0.0, norm_out=True)
    assert torch.equal(y[1], torch.ones_like(y[1])) and y[0].isnan().all()  # 0 / 0, as the formula has it


def _gate_exact(x):
    g, u = x.double().chunk(2, 1)
    return g * torch.sigmoid(g) * u


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 2880), (33, 96), (256, 2880), (100, 14336)])
def test_gate_against_64_bits(cuda_device, m, k, dtype):
    from vllm_qdq_plugin.qdq import silu_mul_mxfp8
    g = torch.Generator(device=cuda_device).manual_seed(m + k)
    x = (torch.randn(m, 2 * k, generator=g, device=cuda_device) * 4).to(dtype)
    x[0, :8] = torch.tensor([0.0, -0.0, 30.0, -30.0, 80.0, -80.0, 1e-3, -1e-3], device=cuda_device).to(dtype)
    rows = silu_mul_mxfp8(x)
    y = _gate_exact(x)
    y16 = y.to(dtype)
    # a value within gate_rel of a border between two 16-bit values may round to either (a zero is exact)
    rel = gate_rel(x.double()[:, :k])
    lo, hi = (y * (1 - rel)).to(dtype), (y * (1 + rel)).to(dtype)
    clear = ((lo == hi) & ((y.abs() > torch.finfo(dtype).tiny) | (y == 0))).view(m, k // 32, 32).all(2)
    codes, scales = _quantize(y16)
    assert clear.float().mean() > 0.3 or m * k < 1024
    assert torch.equal(rows.scales[clear], scales[clear])
    assert torch.equal(rows.codes.view(m, k // 32, 32)[clear], codes.view(m, k // 32, 32)[clear])
    # the others: one 16-bit step moves a value by 2 half steps, and its code by one E4M3 step (2^-3) at the most;
    # saturation at 448 of a maximum below 512 costs 2^-3, a subnormal code 2^-9 of the scale
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    assert ((rows.dequantize().double() - y).abs() <= 2.0 ** -2 * y.abs() + 2.0 ** -8 * scale).all()


def test_gate_of_extreme_gates(cuda_device):
    """exp does not overflow: silu(-100) is a tiny number, silu(100) is 100."""
    from vllm_qdq_plugin.qdq import silu_mul_mxfp8
    x = torch.ones(1, 64, dtype=torch.bfloat16, device=cuda_device)
    x[0, :32] = 100.0
    assert (silu_mul_mxfp8(x).dequantize() == 96.0).logical_or(silu_mul_mxfp8(x).dequantize() == 104.0).all()
    x[0, :32] = -88.0
    got, want = silu_mul_mxfp8(x).dequantize().double(), _gate_exact(x)
    assert ((got - want).abs() <= 2.0 ** -3 * want.abs()).all() and (want != 0).all()
    x[0, 0] = float("nan")
    assert silu_mul_mxfp8(x).dequantize()[0, 0].isnan()


def test_empty_rows(cuda_device):
    from vllm_qdq_plugin.qdq import mxfp8_rows, rmsnorm_mxfp8, silu_mul_mxfp8
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=cuda_device)
    w = torch.ones(64, dtype=torch.bfloat16, device=cuda_device)
    assert mxfp8_rows(x).shape == (0, 64) and silu_mul_mxfp8(x).shape == (0, 32)
    rows, h, y = rmsnorm_mxfp8(x, w, x, norm_out=True)
    assert rows.shape == h.shape == y.shape == (0, 64)


def test_rows_on_another_stream_and_in_a_graph(cuda_device):
    from vllm_qdq_plugin.qdq import rmsnorm_mxfp8, silu_mul_mxfp8
    x = _wide(64, 1024, torch.bfloat16, 1, cuda_device)
    w = torch.randn(512, device=cuda_device).to(torch.bfloat16)
    h = x[:, :512].contiguous()
    want, gate = rmsnorm_mxfp8(h, w, h)[0], silu_mul_mxfp8(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rmsnorm_mxfp8(h, w, h)[0]
    side.synchronize()
    assert torch.equal(got.codes, want.codes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = rmsnorm_mxfp8(h, w, h)[0], silu_mul_mxfp8(x)
    for fill in (0, 255):
        for t in (a.codes, a.scales, b.codes, b.scales):
            t.fill_(fill)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.codes, want.codes) and torch.equal(a.scales, want.scales)
        assert torch.equal(b.codes, gate.codes) and torch.equal(b.scales, gate.scales)
    h.mul_(2)  # the graph reads its inputs anew
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a.codes, rmsnorm_mxfp8(h, w, h)[0].codes)
