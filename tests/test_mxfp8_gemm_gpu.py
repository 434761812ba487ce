"""GPU: the dense and grouped MXFP8 products against float64 products of the same codes.

Every product of two E4M3 values with E8M0 scales is exact in fp32, so the
tolerance is half a step of the output type plus the fp32 accumulation bound
of the FP4 GEMM tests (2^-16 of sum |a_k w_k|).
"""

from __future__ import annotations

import pytest
import torch

from mxfp8_cases import activation, check_moe, check_product, random_weight, routing, values

pytestmark = pytest.mark.gpu


def _ok():
    from vllm_qdq_plugin import _native
    assert _native.device_status() == 0


def _rows_values(rows):
    return values(rows.codes, rows.scales)


@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (1, 1, 32), (1, 4096, 4096), (2, 300, 96), (16, 512, 1024),
                                   (17, 129, 544), (33, 640, 512), (64, 1024, 2080), (5, 300, 4128), (65, 200, 288), (100, 1001, 2880),
                                   (128, 256, 256), (129, 257, 352), (192, 384, 512), (193, 384, 512),
                                   (333, 768, 2048), (1000, 136, 160), (257, 2050, 4128),
                                   (1500, 2560, 544), (2100, 1281, 288), (700, 5002, 320), (4111, 640, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_against_64_bits(cuda_device, m, n, k, dtype):
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    a = activation(m, k, dtype, m + n + k, cuda_device)
    codes, scales = random_weight(n, k, seed=n, dev=cuda_device)
    w = prepare_mxfp8_weight(codes, scales)
    bias = torch.randn(n, device=cuda_device).to(dtype)
    rows = mxfp8_rows(a)
    exact_a, exact_w = _rows_values(rows), values(codes, scales)
    for x in (a, rows):
        out = mxfp8_linear(x, w)
        assert out.dtype == dtype and out.shape == (m, n)
        check_product(out, exact_a, exact_w, what=f"linear {m}x{n}x{k}")
        check_product(mxfp8_linear(x, w, bias), exact_a, exact_w, bias, f"linear {m}x{n}x{k} + bias")
    _ok()


def test_linear_takes_strided_rows_and_its_weights_bias(cuda_device):
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import Mxfp8Rows, mxfp8_rows
    m, n, k = 40, 200, 320
    a = activation(m, k, torch.bfloat16, 1, cuda_device)
    codes, scales = random_weight(n, k, seed=2, dev=cuda_device)
    bias = torch.randn(n, device=cuda_device)
    w = prepare_mxfp8_weight(codes.view(torch.float8_e4m3fn), scales, bias)
    want = mxfp8_linear(a, w)
    rows = mxfp8_rows(a)
    check_product(want, _rows_values(rows), values(codes, scales), bias.to(torch.bfloat16))
    wide = torch.cat([a, a], 1)[:, :k]
    assert torch.equal(mxfp8_linear(wide, w), want)
    assert torch.equal(mxfp8_linear(torch.nn.functional.pad(a, (3, 0))[:, 3:], w), want)
    held = torch.full((m, k + 64), 0x7F, dtype=torch.uint8, device=cuda_device)  # NaN codes behind every row
    held[:, :k] = rows.codes
    stored = torch.full((m, 48), 0xFF, dtype=torch.uint8, device=cuda_device)  # and NaN scales
    stored[:, : k // 32] = rows.scales
    view = Mxfp8Rows(held[:, :k], stored[:, : k // 32], torch.bfloat16)
    assert torch.equal(mxfp8_linear(view, w), want)
    wpad = torch.full((n, k + 16), 0x7F, dtype=torch.uint8, device=cuda_device)
    wpad[:, :k] = codes
    assert torch.equal(mxfp8_linear(a, prepare_mxfp8_weight(wpad[:, :k], scales, bias)), want)
    _ok()


@pytest.mark.parametrize("m", [3, 70, 300])
def test_linear_keeps_nan_and_infinite_rows_apart(cuda_device, m):
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    n, k = 160, 416
    a = activation(m, k, torch.bfloat16, 9, cuda_device)
    w = prepare_mxfp8_weight(*random_weight(n, k, seed=4, dev=cuda_device))
    want = mxfp8_linear(a, w)
    b = a.clone()
    b[m // 2, 5] = float("nan")
    got = mxfp8_linear(b, w)
    others = torch.arange(m, device=cuda_device) != m // 2
    assert torch.equal(got[others], want[others]) and got[m // 2].isnan().all()


def test_linear_empty(cuda_device):
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    w = prepare_mxfp8_weight(*random_weight(96, 64, seed=4, dev=cuda_device))
    a = torch.empty(0, 64, dtype=torch.bfloat16, device=cuda_device)
    assert mxfp8_linear(a, w).shape == (0, 96) and mxfp8_linear(mxfp8_rows(a), w).shape == (0, 96)


@pytest.mark.parametrize("m,e,top_k,bs,n,k,mul", [(1, 4, 1, 16, 128, 128, False),
                                                  (1, 8, 4, 8, 200, 2880, True),
                                                  (5, 4, 2, 16, 256, 512, False),
                                                  (37, 8, 2, 16, 384, 1024, True),
                                                  (64, 16, 4, 32, 201, 2080, True),
                                                  (3, 4, 1, 64, 128, 288, False),
                                                  (100, 8, 8, 8, 256, 512, True),
                                                  (300, 6, 2, 64, 384, 1024, True),
                                                  (2048, 4, 2, 8, 128, 256, False),
                                                  (700, 2, 2, 64, 320, 544, True),
                                                  (150, 4, 2, 48, 257, 512, False),
                                                  (90, 5, 2, 1, 130, 96, True),
                                                  (50, 3, 1, 13, 128, 320, False),
                                                  (61, 128, 4, 16, 128, 256, True),
                                                  (600, 3, 2, 64, 2304, 288, True),
                                                  (200, 16, 2, 16, 2305, 544, False),
                                                  (900, 2, 1, 48, 4352, 96, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_against_64_bits(cuda_device, m, e, top_k, bs, n, k, mul, dtype):
    """Every routed slot's row; one block per expert, long runs cut into segments, layouts whose runs cross the
    segment scan's chunks, block sizes that do not divide a segment, 128 experts of which few are hit."""
    from vllm_qdq_plugin.gemm import mxfp8_moe_linear, prepare_mxfp8_moe_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    a = activation(m, k, dtype, m + e + bs, cuda_device)
    codes, scales = random_weight(e, n, k, seed=n + e, dev=cuda_device)
    w = prepare_mxfp8_moe_weight(codes, scales)
    ids, sid, eid, ntp, tw = routing(m, e, top_k, bs, m + e, cuda_device)
    rows = mxfp8_rows(a)
    for x in (a, rows):
        out = mxfp8_moe_linear(x, w, sid, eid, ntp, tw, bs, top_k, mul)
        assert out.dtype == dtype and out.shape == (m * top_k, n)
        check_moe(out, _rows_values(rows), codes, scales, ids, f"moe m={m} e={e} bs={bs}", tw if mul else None)
    _ok()


def test_moe_leaves_what_no_slot_names(cuda_device):
    """Blocks of experts outside [0, E), blocks behind num_tokens_post_padded and slots that no block names keep
    their rows; sentinels and stray slot numbers write nothing."""
    from vllm_qdq_plugin.gemm import mxfp8_moe_linear, prepare_mxfp8_moe_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    m, e, top_k, bs, n, k = 40, 4, 2, 16, 136, 256
    dev = cuda_device
    a = activation(m, k, torch.bfloat16, 1, dev)
    codes, scales = random_weight(e, n, k, seed=3, dev=dev)
    w = prepare_mxfp8_moe_weight(codes, scales)
    ids, sid, eid, ntp, tw = routing(m, e, top_k, bs, 2, dev)
    full = mxfp8_moe_linear(a, w, sid, eid, ntp, tw, bs, top_k, True)
    eid2 = eid.clone()
    eid2[0], eid2[-1] = -1, e
    sid2 = torch.cat([sid, torch.arange(2 * bs, dtype=torch.int32, device=dev)])  # live-looking, behind the end
    eid2 = torch.cat([eid2, torch.tensor([1, 2], dtype=torch.int32, device=dev)])
    sid2[bs + 3] = -7
    sid2[bs + 4] = m * top_k + 5
    held = torch.full((m * top_k + 3, n + 8), 7.0, dtype=torch.bfloat16, device=dev)
    out = held[: m * top_k, :n]
    assert mxfp8_moe_linear(mxfp8_rows(a), w, sid2, eid2, ntp, tw, bs, top_k, True, out=out) is out
    named = torch.zeros(m * top_k, dtype=torch.bool, device=dev)
    live = sid2[: int(ntp)].view(-1, bs)[1:-1].reshape(-1)
    named[live[(live >= 0) & (live < m * top_k)].long()] = True
    assert 0 < int(named.sum()) < m * top_k
    assert torch.equal(out[named], full[named]) and (out[~named] == 7.0).all()
    assert (held[m * top_k:] == 7.0).all() and (held[:, n:] == 7.0).all()
    ntp0 = torch.zeros_like(ntp)
    out.fill_(7.0)
    mxfp8_moe_linear(a, w, sid2, eid2, ntp0, tw, bs, top_k, False, out=out)
    assert (out == 7.0).all()
    _ok()


@pytest.mark.parametrize("k", [288, 2880])
def test_moe_result_independent_of_stale_workspace(cuda_device, k):
    from vllm_qdq_plugin import _native
    from vllm_qdq_plugin.gemm import prepare_mxfp8_moe_weight
    m, e, top_k, bs, n = 40, 4, 2, 16, 256
    dev = cuda_device
    a = activation(m, k, torch.bfloat16, 5, dev)
    w = prepare_mxfp8_moe_weight(*random_weight(e, n, k, seed=6, dev=dev))
    _, sid, eid, ntp, tw = routing(m, e, top_k, bs, 7, dev)
    lib, outs = _native.lib(), []
    for fill in (0x00, 0xFF, 0x7F):
        ws = torch.full((lib.fp8_moe_workspace_bytes(m, sid.numel(), bs, k),), fill, dtype=torch.uint8, device=dev)
        out = torch.zeros((m * top_k, n), dtype=torch.bfloat16, device=dev)
        _native.call("fp8_moe_mxf8", a.data_ptr(), k, None, None, 0, 0, 0, w.codes.data_ptr(), w.sf_tiled.data_ptr(), e,
                     sid.data_ptr(), eid.data_ptr(), ntp.data_ptr(), tw.data_ptr(), sid.numel(), bs, top_k, 1,
                     out.data_ptr(), n, m, n, k, ws.data_ptr(), ws.numel(), _native.stream_ptr(dev))
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and outs[0].isfinite().all()
    _ok()


def test_products_in_graphs_and_on_two_streams(cuda_device):
    """Two captured graphs and eager calls on two streams, each call with a workspace of its own."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight
    dev, m, n, k, e, top_k, bs = cuda_device, 48, 256, 512, 4, 2, 16
    a = activation(m, k, torch.bfloat16, 1, dev)
    w = prepare_mxfp8_weight(*random_weight(n, k, seed=1, dev=dev))
    wm = prepare_mxfp8_moe_weight(*random_weight(e, n, k, seed=2, dev=dev))
    _, sid, eid, ntp, tw = routing(m, e, top_k, bs, 3, dev)

    def both(x):
        return mxfp8_linear(x, w), mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, bs, top_k, True)

    want, want2 = both(a), both(a * 2)
    graphs = []
    b = a.clone()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(b)
        graphs.append((graph, out))
    for x, ref in ((a, want), (a * 2, want2), (a, want)):
        b.copy_(x)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(g, r) for g, r in zip(out, ref))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    results = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            results.append(both(a))
    torch.cuda.synchronize()
    assert all(torch.equal(g, r) for out in results for g, r in zip(out, want))
    _ok()


@pytest.mark.parametrize("m,bs", [(1, 16), (23, 16), (400, 64)])
def test_a_gated_expert_layer_stage_by_stage(cuda_device, m, bs):
    """Norm -> router -> first grouped product -> gate -> second grouped product, as a layer runs them; every stage
    is checked against 64 bits on what the stage before it really produced."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_quantize, mxfp8_rows, rmsnorm_mxfp8, silu_mul_mxfp8
    from oracle import gemm as og
    dev, hidden, inner, e, top_k = cuda_device, 320, 288, 6, 2
    x, residual = (activation(m, hidden, torch.bfloat16, s, dev) for s in (1, 2))
    weight = (1 + 0.1 * torch.randn(hidden, device=dev)).to(torch.bfloat16)
    w_attn = random_weight(hidden, hidden, seed=3, dev=dev)
    w13, w2 = random_weight(e, 2 * inner, hidden, seed=4, dev=dev), random_weight(e, hidden, inner, seed=5, dev=dev)
    router = torch.randn(e, hidden, device=dev)

    proj = mxfp8_linear(mxfp8_rows(x), prepare_mxfp8_weight(*w_attn))
    check_product(proj, _rows_values(mxfp8_rows(x)), values(*w_attn), what="projection")
    rows, h, y = rmsnorm_mxfp8(proj, weight, residual, norm_out=True)
    assert torch.equal(h, (proj.float() + residual.float()).to(torch.bfloat16))
    assert torch.equal(rows.codes, mxfp8_quantize(y)[0])
    prob, ids = torch.softmax(y.float() @ router.t(), 1).topk(top_k, 1)
    sid, eid, ntp = (torch.from_numpy(t).to(dev) for t in og.moe_align(ids.cpu().numpy(), e, bs))
    up = mxfp8_moe_linear(rows, prepare_mxfp8_moe_weight(*w13), sid, eid, ntp, None, bs, top_k, False)
    check_moe(up, _rows_values(rows), *w13, ids.cpu().numpy(), "first product")
    act = silu_mul_mxfp8(up)
    down = mxfp8_moe_linear(act, prepare_mxfp8_moe_weight(*w2), sid, eid, ntp, prob, bs, 1, True)  # a row a slot
    check_moe(down, _rows_values(act), *w2, ids.reshape(-1, 1).cpu().numpy(), "second product", prob)
    out = h + down.view(m, top_k, hidden).sum(1)
    assert out.shape == (m, hidden) and out.isfinite().all()
    _ok()


def test_refusals_name_the_argument(cuda_device):
    """Malformed calls are refused before any launch, as the other operators refuse them."""
    import dataclasses
    from vllm_qdq_plugin.gemm import (mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight)
    from vllm_qdq_plugin.qdq import Mxfp8Rows, mxfp8_rows, rmsnorm_mxfp8, silu_mul_mxfp8
    dev = cuda_device
    x = activation(8, 64, torch.bfloat16, 1, dev)
    g = torch.ones(64, dtype=torch.bfloat16, device=dev)
    rows = mxfp8_rows(x)
    w = prepare_mxfp8_weight(*random_weight(32, 64, seed=1, dev=dev))
    wm = prepare_mxfp8_moe_weight(*random_weight(2, 32, 64, seed=1, dev=dev))
    _, sid, eid, ntp, tw = routing(8, 2, 1, 16, 1, dev)
    bad = [
        lambda: mxfp8_rows(x.float()), lambda: mxfp8_rows(x[0]), lambda: mxfp8_rows(x[:, :48]),
        lambda: silu_mul_mxfp8(x[:, :63]), lambda: silu_mul_mxfp8(x[:, :32]),
        lambda: rmsnorm_mxfp8(x, g[:32]), lambda: rmsnorm_mxfp8(x, g.float()), lambda: rmsnorm_mxfp8(x, g.cpu()),
        lambda: rmsnorm_mxfp8(x, g, x[:4]), lambda: rmsnorm_mxfp8(x, g, x.half()), lambda: rmsnorm_mxfp8(x, g, x.cpu()),
        lambda: rmsnorm_mxfp8(x, g, eps=-1.0),
        lambda: rmsnorm_mxfp8(torch.zeros(1, 65568, dtype=torch.bfloat16, device=dev),
                              torch.zeros(65568, dtype=torch.bfloat16, device=dev)),
        lambda: Mxfp8Rows.from_codes(rows.codes, rows.scales[:, :1]), lambda: Mxfp8Rows.from_codes(rows.codes.view(torch.int8), rows.scales),
        lambda: Mxfp8Rows.from_codes(rows.codes, rows.scales, torch.float32),
        lambda: mxfp8_linear(x.float(), w), lambda: mxfp8_linear(x[:, :32], w), lambda: mxfp8_linear(x, w, g),
        lambda: mxfp8_linear(Mxfp8Rows(rows.codes, rows.scales.contiguous(), rows.dtype), w),
        lambda: mxfp8_linear(Mxfp8Rows(rows.codes, rows.scales[:4], rows.dtype), w),
        lambda: mxfp8_linear(Mxfp8Rows(rows.codes[:1], rows.scales[:1].contiguous().clone(), rows.dtype), w),
        lambda: mxfp8_linear(x, dataclasses.replace(w, codes=w.codes.cpu())),
        lambda: prepare_mxfp8_weight(w.codes, rows.scales), lambda: prepare_mxfp8_moe_weight(w.codes, rows.scales),
        lambda: mxfp8_moe_linear(x, wm, sid.long(), eid, ntp, tw, 16, 1, False),
        lambda: mxfp8_moe_linear(x, wm, sid, eid[:1], ntp, tw, 8, 1, False),
        lambda: mxfp8_moe_linear(x, wm, sid, eid, ntp, None, 16, 1, True),
        lambda: mxfp8_moe_linear(x, wm, sid, eid, ntp, tw[:3], 16, 1, True),
        lambda: mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, 65, 1, False),
        lambda: mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, 16, 0, False),
        lambda: mxfp8_moe_linear(x, wm, sid.cpu(), eid, ntp, tw, 16, 1, False),
        lambda: mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, 16, 1, False, out=torch.empty(8, 32, device=dev)),
        lambda: mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, 16, 1, False, out=torch.empty_like(x)),
        lambda: mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, 16, 1, False,
                                 out=torch.empty(32, 8, dtype=torch.bfloat16, device=dev).t()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((AssertionError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(AssertionError, match="2D"):
        mxfp8_rows(x[0])
    with pytest.raises(AssertionError, match="weight"):
        rmsnorm_mxfp8(x, g[:32])
    assert mxfp8_linear(x, w).isfinite().all()
    _ok()


def test_operators_trace_under_compile(cuda_device):
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import rmsnorm_mxfp8, silu_mul_mxfp8
    x = activation(8, 64, torch.bfloat16, 1, cuda_device)
    g = torch.ones(64, dtype=torch.bfloat16, device=cuda_device)
    w = prepare_mxfp8_weight(*random_weight(128, 64, seed=1, dev=cuda_device))

    def layer(x, r):
        rows, h, _ = rmsnorm_mxfp8(x, g, r)
        act = silu_mul_mxfp8(mxfp8_linear(rows, w))
        return act.codes, act.scales, h

    want = layer(x, x)
    got = torch.compile(layer, backend="eager", fullgraph=True)(x, x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_broadcast_rows_and_parameters(cuda_device):
    """Expanded activations are copied, not misread; norm weights that are parameters are taken as they are."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows, rmsnorm_mxfp8
    dev, m, k = cuda_device, 24, 96
    one = activation(1, k, torch.bfloat16, 1, dev)
    wide, dense = one.expand(m, k), one.repeat(m, 1)
    g = torch.nn.Parameter(torch.randn(k, device=dev).to(torch.bfloat16))
    assert torch.equal(mxfp8_rows(wide).codes, mxfp8_rows(dense).codes)
    assert torch.equal(rmsnorm_mxfp8(wide, g, wide)[1], rmsnorm_mxfp8(dense, g.detach(), dense)[1])
    w = prepare_mxfp8_weight(*random_weight(130, k, seed=1, dev=dev))
    assert torch.equal(mxfp8_linear(wide, w), mxfp8_linear(dense, w))
    wm = prepare_mxfp8_moe_weight(*random_weight(2, 130, k, seed=1, dev=dev))
    _, sid, eid, ntp, tw = routing(m, 2, 2, 16, 1, dev)
    both = [mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, 16, 2, True) for x in (wide, dense)]
    assert torch.equal(*both)
    _ok()


def test_chains_of_small_calls(cuda_device):
    """Many short kernels in flight behind one another, each reading what the one before wrote: eager and captured."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import rmsnorm_mxfp8, silu_mul_mxfp8
    dev, m, k = cuda_device, 4, 256
    g = torch.ones(k, dtype=torch.bfloat16, device=dev)
    ups = [prepare_mxfp8_weight(*random_weight(2 * k, k, seed=i, dev=dev)) for i in range(4)]
    downs = [prepare_mxfp8_weight(*random_weight(k, k, seed=9 + i, dev=dev)) for i in range(4)]

    def layers(x, wait):
        h = x
        for i in range(24):
            rows, h, _ = rmsnorm_mxfp8(x, g, h)
            wait()
            up = mxfp8_linear(rows, ups[i % 4])
            wait()
            act = silu_mul_mxfp8(up)
            wait()
            x = mxfp8_linear(act, downs[i % 4])
            wait()
            x = mxfp8_linear(x, downs[(i + 1) % 4])
            wait()
        return x, h

    x = activation(m, k, torch.bfloat16, 1, dev)
    want = layers(x, torch.cuda.synchronize)
    for _ in range(20):
        got = layers(x, lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layers(x, lambda: None)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want)) and want[0].isfinite().all()
    _ok()


def test_first_call_of_a_process_inside_a_capture(tmp_path):
    """Nothing has to run before a capture: not the library's load, nor a kernel's first launch."""
    import subprocess
    import sys
    from conftest import REPO
    script = tmp_path / "first.py"
    script.write_text(f"""
import sys
sys.path[:0] = [{str(REPO / "vllm-qdq-plugin_b200")!r}, {str(REPO)!r}, {str(REPO / "tests")!r}]
import torch
from mxfp8_cases import activation, random_weight, routing
from vllm_qdq_plugin.gemm import Mxfp8MoeWeight, Mxfp8Weight, mxfp8_linear, mxfp8_moe_linear
from vllm_qdq_plugin.qdq import rmsnorm_mxfp8
dev = torch.device("cuda", 0)
x = activation(40, 256, torch.bfloat16, 1, dev)
g = torch.ones(256, dtype=torch.bfloat16, device=dev)
codes, scales = random_weight(2, 512, 256, seed=1, dev=dev)
sf = torch.full((2 * 512 * 8,), 118, dtype=torch.uint8, device=dev)
w, wm = Mxfp8Weight(codes[0], sf, 512, 256), Mxfp8MoeWeight(codes, sf, 2, 512, 256)
_, sid, eid, ntp, tw = routing(40, 2, 1, 16, 1, dev)
big = activation(700, 256, torch.bfloat16, 2, dev)
torch.cuda.synchronize()
def run():
    rows = rmsnorm_mxfp8(x, g)[0]
    return mxfp8_linear(rows, w), mxfp8_linear(big, w), mxfp8_moe_linear(rows, wm, sid, eid, ntp, tw, 16, 1, True)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, run())) and all(o.isfinite().all() for o in out)
print("ok")
""")
    done = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "ok" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("m,k", [(3, 2880), (70, 352), (300, 96), (2000, 544)])
def test_padding_of_scale_rows_has_no_effect(cuda_device, m, k):
    """The bytes between rows of scales are read and must not count, whatever they are, in every form of the product."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import Mxfp8Rows, mxfp8_rows
    dev, n, e = cuda_device, 640, 3
    a = activation(m, k, torch.bfloat16, 1, dev)
    rows = mxfp8_rows(a)
    w = prepare_mxfp8_weight(*random_weight(n, k, seed=1, dev=dev))
    wm = prepare_mxfp8_moe_weight(*random_weight(e, n, k, seed=2, dev=dev))
    _, sid, eid, ntp, tw = routing(m, e, 2, 32, 1, dev)
    seen = []
    for fill in (0x00, 0xFF, 0x7F):
        stored = torch.full((m, (k // 32 + 15) // 16 * 16), fill, dtype=torch.uint8, device=dev)
        stored[:, : k // 32] = rows.scales
        r = Mxfp8Rows(rows.codes, stored[:, : k // 32], torch.bfloat16)
        seen.append((mxfp8_linear(r, w), mxfp8_moe_linear(r, wm, sid, eid, ntp, tw, 32, 2, True)))
    assert all(torch.equal(x, y) for s in seen[1:] for x, y in zip(s, seen[0])) and seen[0][0].isfinite().all()
    _ok()


@pytest.mark.parametrize("m,n,shift,gap", [(600, 328, 0, 8), (600, 328, 8, 16), (600, 328, 2, 8), (600, 328, 0, 2),
                                           (600, 328, 1, 8), (600, 328, 0, 3), (600, 326, 0, 2), (600, 325, 0, 3),
                                           (4100, 2568, 0, 8), (4100, 2568, 2, 8), (4100, 2562, 0, 6), (4100, 2563, 1, 1)])
def test_output_rows_at_any_address(cuda_device, m, n, shift, gap):
    """Products into rows that start `shift` elements into memory and `n + gap` apart: what lies between stays."""
    from vllm_qdq_plugin import _native
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    k, dev = 160, cuda_device
    rows = mxfp8_rows(activation(m, k, torch.bfloat16, n, dev))
    codes, scales = random_weight(n, k, seed=m, dev=dev)
    w = prepare_mxfp8_weight(codes, scales)
    bias = torch.randn(n, device=dev).to(torch.bfloat16)
    want = mxfp8_linear(rows, w, bias)
    check_product(want, _rows_values(rows), values(codes, scales), bias, f"{m}x{n}")
    held = torch.full((shift + m * (n + gap) + 8,), -3.0, dtype=torch.bfloat16, device=dev)
    out = held[shift : shift + m * (n + gap)].view(m, n + gap)
    lib = _native.lib()
    sf = torch.empty(lib.qdq_sf_tiled_bytes(n, k), dtype=torch.uint8, device=dev)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.qdq_sf_tile(scales.data_ptr(), sf.data_ptr(), n, k, k // 32, 32, stream) == 0
    torch.cuda.synchronize()
    assert lib.fp8_gemm_mxf8(rows.codes.data_ptr(), rows.scales.data_ptr(), rows.codes.stride(0), rows.scales.stride(0),
                             codes.data_ptr(), sf.data_ptr(), bias.data_ptr(), out.data_ptr(), m, n, k, k, n + gap, 0,
                             stream) == 0
    assert torch.equal(out[:, :n], want) and (out[:, n:] == -3).all()
    assert (held[:shift] == -3).all() and (held[shift + m * (n + gap) :] == -3).all()
    _ok()


@pytest.mark.parametrize("m,e,top_k,bs,n,k", [(400, 128, 4, 16, 2568, 96),   # pairs of few rows, many items an SM
                                              (512, 8, 2, 64, 2600, 64),     # the experts' rows in one item
                                              (911, 4, 2, 16, 390, 224),     # several items an expert
                                              (300, 4, 2, 64, 1000, 96),
                                              (1422, 64, 4, 8, 127, 192),
                                              (120, 16, 2, 64, 1312, 64)])
def test_moe_tile_choices(cuda_device, m, e, top_k, bs, n, k):
    from vllm_qdq_plugin.gemm import mxfp8_moe_linear, prepare_mxfp8_moe_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    rows = mxfp8_rows(activation(m, k, torch.bfloat16, m, cuda_device))
    codes, scales = random_weight(e, n, k, seed=n, dev=cuda_device)
    w = prepare_mxfp8_moe_weight(codes, scales)
    ids, sid, eid, ntp, tw = routing(m, e, top_k, bs, m, cuda_device)
    for mul in (False, True):
        out = mxfp8_moe_linear(rows, w, sid, eid, ntp, tw, bs, top_k, mul)
        check_moe(out, _rows_values(rows), codes, scales, ids, f"m={m} e={e} n={n}", tw if mul else None)
    _ok()


@pytest.mark.parametrize("m,n,k", [(1, 1024, 1024), (5, 640, 4128), (60, 2048, 512), (100, 512, 1024), (2100, 1280, 288)])
def test_weight_changed_by_the_kernel_before(cuda_device, m, n, k):
    """A weight's codes and scales changed in place right before each product, eager and captured."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    dev = cuda_device
    a = activation(m, k, torch.bfloat16, m, dev)
    rows = mxfp8_rows(a)
    codes, scales = random_weight(n, k, seed=3, dev=dev)
    codes.bitwise_and_(0x87)  # room for a change of the exponent that leaves no NaN
    w = prepare_mxfp8_weight(codes.clone(), scales)
    sf = w.sf_tiled.clone()
    steps = [(x, i) for i in range(1, 6) for x in (a, rows)]
    want = [mxfp8_linear(x, prepare_mxfp8_weight(codes + 8 * i, scales + i)) for x, i in steps]
    ints, tiled = codes.to(torch.int16), sf.to(torch.int16)

    def run():
        got = []
        for x, i in steps:
            torch.add(ints, 8 * i, out=w.codes)  # converting kernels, not copies
            torch.add(tiled, i, out=w.sf_tiled)
            got.append(mxfp8_linear(x, w))
            w.sf_tiled.fill_(0)
            w.codes.fill_(0x38)
            got.append(mxfp8_linear(x, w))
        return got

    torch.cuda.synchronize()
    for _ in range(3):
        got = run()
        assert all(torch.equal(g, e) for g, e in zip(got[::2], want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g, e) for g, e in zip(got[::2], want))
    _ok()


def test_weights_that_were_not_prepared_are_refused(cuda_device):
    import dataclasses
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    m, n, k, e, dev = 4, 200, 512, 2, cuda_device
    a = activation(m, k, torch.bfloat16, 1, dev)
    rows = mxfp8_rows(a)
    codes, scales = random_weight(e, n, k, seed=1, dev=dev)
    one, many = prepare_mxfp8_weight(codes[0], scales[0]), prepare_mxfp8_moe_weight(codes, scales)
    _, sid, eid, ntp, tw = routing(m, e, 1, 16, 1, dev)
    wide = torch.zeros((n, k), dtype=torch.bfloat16, device=dev)
    across = codes[0].t().contiguous().t()
    for x in (a, rows):
        for change in ({"sf_tiled": one.sf_tiled[:-1]}, {"sf_tiled": scales[0]}, {"codes": wide}, {"codes": across}):
            with pytest.raises(RuntimeError, match="weight's"):
                mxfp8_linear(x, dataclasses.replace(one, **change))
        for change in ({"sf_tiled": one.sf_tiled}, {"sf_tiled": scales[0]}, {"codes": wide.expand(e, n, k).contiguous()}):
            with pytest.raises(RuntimeError, match="weight's"):
                mxfp8_moe_linear(x, dataclasses.replace(many, **change), sid, eid, ntp, tw, 16, 1, True)
    _ok()


@pytest.mark.parametrize("m,e,top_k,bs,n,k", [(700, 9, 8, 16, 64, 2080), (4200, 3, 2, 64, 200, 2048), (1500, 6, 4, 64, 136, 3104),
                                              (130, 5, 2, 8, 640, 4128), (40, 40, 3, 64, 512, 8224), (2100, 300, 1, 1, 128, 96)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_of_16_bit_rows_is_that_of_their_mxfp8_rows(cuda_device, m, e, top_k, bs, n, k, dtype):
    """Rows that many slots share, rows split over several warps, one row a warp: the codes are always those of mxfp8_rows."""
    from vllm_qdq_plugin.gemm import mxfp8_moe_linear, prepare_mxfp8_moe_weight
    from vllm_qdq_plugin.qdq import mxfp8_rows
    a = activation(m, k, dtype, m + k, cuda_device)
    wide = torch.nn.functional.pad(a, (8, 0))[:, 8:]  # rows further apart
    codes, scales = random_weight(e, n, k, seed=n, dev=cuda_device)
    w = prepare_mxfp8_moe_weight(codes, scales)
    ids, sid, eid, ntp, tw = routing(m, e, top_k, bs, m, cuda_device)
    rows = mxfp8_rows(a)
    want = mxfp8_moe_linear(rows, w, sid, eid, ntp, tw, bs, top_k, True)
    check_moe(want, _rows_values(rows), codes, scales, ids, f"m={m} e={e} k={k}", tw)
    for x in (a, wide):
        assert torch.equal(mxfp8_moe_linear(x, w, sid, eid, ntp, tw, bs, top_k, True), want)
    _ok()
