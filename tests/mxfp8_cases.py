"""Inputs and 64-bit results of the MXFP8 row and product tests."""

from __future__ import annotations

import numpy as np
import torch

from oracle import gemm as og

# fp32 accumulation of exact products: relative to sum |a_k w_k|, as in the FP4 GEMM tests
ACC = 2.0 ** -16


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values of E4M3 codes (uint8 [..., K]) with E8M0 scales (uint8 [..., K/32])."""
    v = codes.view(torch.float8_e4m3fn).float().double()
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def random_weight(*shape: int, seed: int, dev) -> tuple[torch.Tensor, torch.Tensor]:
    g = torch.Generator(device=dev).manual_seed(seed)
    codes = (torch.randn(shape, generator=g, device=dev) * 110).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.randint(110, 124, (*shape[:-1], shape[-1] // 32), generator=g, device=dev, dtype=torch.uint8)
    return codes.view(torch.uint8), scales


def activation(m: int, k: int, dtype: torch.dtype, seed: int, dev) -> torch.Tensor:
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(m, k, generator=g, device=dev)
    return (x * torch.exp2(torch.randint(-6, 3, (m, 1), generator=g, device=dev).float())).to(dtype)


def check_product(got: torch.Tensor, a: torch.Tensor, w: torch.Tensor, bias=None, what: str = "", scale=None) -> None:
    """got [M, N] against a [M, K] . w [N, K]^T (+ bias) (x scale [M]) in float64: half a step of the
    output type, plus the fp32 accumulation bound."""
    exact, absum = a @ w.t(), a.abs() @ w.abs().t()
    if bias is not None:
        exact, absum = exact + bias.double(), absum + bias.double().abs()
    if scale is not None:
        exact, absum = exact * scale.double()[:, None], absum * scale.double().abs()[:, None]
    bound = half_step(got.dtype) * exact.abs() + ACC * absum + torch.finfo(got.dtype).tiny * half_step(got.dtype)
    bad = ~((got.double() - exact).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside tolerance, first {bad.nonzero()[0].tolist()}"


def routing(m: int, e: int, top_k: int, block: int, seed: int, dev, experts=None):
    """Distinct experts per token (out of `experts`), in vLLM's moe_align_block_size layout."""
    rng = np.random.default_rng(seed)
    pool = np.arange(e) if experts is None else np.asarray(experts)
    ids = np.stack([rng.permutation(pool)[:top_k] for _ in range(m)])
    sid, eid, ntp = og.moe_align(ids, e, block)
    w = torch.from_numpy(rng.random((m, top_k)).astype(np.float32)).to(dev)
    return ids, *(torch.from_numpy(t).to(dev) for t in (sid, eid, ntp)), w


def check_moe(out, a, codes, scales, ids, what, weights=None):
    """Every slot's row against its expert's product; `a` float64 [M, K]."""
    m, top_k = ids.shape
    flat = torch.from_numpy(ids.reshape(-1)).to(out.device)
    for e in np.unique(ids):
        slots = (flat == int(e)).nonzero()[:, 0]
        check_product(out[slots], a[slots // top_k], values(codes[e], scales[e]),
                      what=f"{what} expert {e}", scale=None if weights is None else weights.reshape(-1)[slots])
