"""GPU: every pass of the MXFP8 chains counts, not the last alone: kernels that start early must not read what the kernel
before them has yet to write."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from mxfp8_cases import activation, random_weight, routing

pytestmark = pytest.mark.gpu


def _ok():
    from vllm_qdq_plugin import _native
    assert _native.device_status() == 0


class Mismatches:
    """Counts elements that differ, on the GPU, without waiting for it between the passes."""

    def __init__(self, dev):
        self.count = torch.zeros((), dtype=torch.int64, device=dev)

    def __call__(self, got, want):
        for g, w in zip(got, want, strict=True):
            self.count += (g != w).sum()


def _moe_weight(e, n, k, seed, dev):
    from vllm_qdq_plugin.gemm import prepare_mxfp8_moe_weight
    return prepare_mxfp8_moe_weight(*random_weight(e, n, k, seed=seed, dev=dev))


@pytest.mark.parametrize("m,k", [(4, 256), (48, 512), (300, 96)])
def test_every_pass_of_a_chain(cuda_device, m, k):
    """Norm, dense product, gate and grouped products behind one another, each reading what the one before wrote."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import rmsnorm_mxfp8, silu_mul_mxfp8
    dev = cuda_device
    g = torch.ones(k, dtype=torch.bfloat16, device=dev)
    ups = [prepare_mxfp8_weight(*random_weight(2 * k, k, seed=i, dev=dev)) for i in range(2)]
    experts = [_moe_weight(3, k, k, 9 + i, dev) for i in range(2)]
    _, sid, eid, ntp, tw = routing(m, 3, 1, 16, 1, dev)

    def layers(x, wait):
        h = x
        for i in range(12):
            rows, h, y = rmsnorm_mxfp8(x, g, h, norm_out=True)
            wait()
            up = mxfp8_linear(rows, ups[i % 2])
            wait()
            act = silu_mul_mxfp8(up)
            wait()
            x = mxfp8_moe_linear(act, experts[i % 2], sid, eid, ntp, tw, 16, 1, True)
            wait()
            x = mxfp8_moe_linear(x, experts[(i + 1) % 2], sid, eid, ntp, tw, 16, 1, False)
            wait()
            x = x + mxfp8_linear(y, ups[i % 2])[:, :k]
        return x, h

    x = activation(m, k, torch.bfloat16, 1, dev)
    want = layers(x, torch.cuda.synchronize)
    assert want[0].isfinite().all()
    wrong = Mismatches(dev)
    for _ in range(20):
        wrong(layers(x, lambda: None), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layers(x, lambda: None)
    for _ in range(20):
        graph.replay()
        wrong(out, want)
        for t in out:
            t.zero_()
    assert int(wrong.count) == 0
    _ok()


@pytest.mark.parametrize("m,n,k,grouped", [(1, 1024, 1024, False), (60, 2048, 512, False), (2100, 1280, 288, False),
                                           (2, 256, 512, True), (900, 640, 288, True)])
def test_inputs_and_weights_written_just_before(cuda_device, m, n, k, grouped):
    """Activation, norm weight, codes and scales of the weight rewritten in place right before every call: few blocks of
    experts in one launch, many through the layout pass."""
    from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import rmsnorm_mxfp8
    dev, e = cuda_device, 3
    steps = 6
    sources = [activation(m, k, torch.bfloat16, i, dev) for i in range(steps)]
    gains = [torch.randn(k, device=dev).to(torch.bfloat16) for _ in range(steps)]
    made = [random_weight(e, n, k, seed=i, dev=dev) for i in range(steps)]
    _, sid, eid, ntp, tw = routing(m, e, 1, 16, 1, dev)
    if grouped:
        weights = [_moe_weight(e, n, k, i, dev) for i in range(steps)]
    else:
        weights = [prepare_mxfp8_weight(c[0], s[0]) for c, s in made]

    def product(a, w):
        return mxfp8_moe_linear(a, w, sid, eid, ntp, tw, 16, 1, True) if grouped else mxfp8_linear(a, w)

    want = []
    for i in range(steps):
        rows, _, y = rmsnorm_mxfp8(sources[i], gains[i], norm_out=True)
        torch.cuda.synchronize()
        want += [product(rows, weights[i]), product(y, weights[i]), product(sources[i], weights[i])]
        torch.cuda.synchronize()
    x, g = sources[0].clone(), gains[0].clone()
    held = dataclasses.replace(weights[0], codes=weights[0].codes.clone(), sf_tiled=weights[0].sf_tiled.clone())

    def run():
        got = []
        for i in range(steps):
            torch.mul(gains[i], 1, out=g)
            torch.mul(sources[i], 1, out=x)
            rows, _, y = rmsnorm_mxfp8(x, g, norm_out=True)
            torch.bitwise_or(weights[i].codes, 0, out=held.codes)
            torch.bitwise_or(weights[i].sf_tiled, 0, out=held.sf_tiled)
            got.append(product(rows, held))
            got.append(product(y, held))
            got.append(product(x, held))
            for t in (x, g):
                t.fill_(7)
            held.codes.fill_(0x38)
            held.sf_tiled.fill_(1)
        return got

    wrong = Mismatches(dev)
    for _ in range(5):
        wrong(run(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(10):
        graph.replay()
        wrong(out, want)
        for t in out:
            t.zero_()
    assert int(wrong.count) == 0
    _ok()
