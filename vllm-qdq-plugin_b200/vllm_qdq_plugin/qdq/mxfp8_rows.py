# SPDX-License-Identifier: Apache-2.0
"""MXFP8 rows: activations held as E4M3 codes with E8M0 scales, and the
operators that end in them.

`mxfp8_qdq` returns the values that MXFP8 leaves of an activation; these
return the codes and scales themselves, for `gemm.mxfp8_linear` and
`gemm.mxfp8_moe_linear` to multiply.  The codes are those of `mxfp8_qdq` (and
so of the reference, src/vllm_qdq_plugin/qdq/mxfp8.py:73-125) on a 16-bit
tensor that holds the operator's formula, rounded once (an unfused operator that
rounds in between stores another).  One HBM pass each
(`qdq_mxfp8_rows`, `qdq_rmsnorm_mxfp8`, `qdq_silu_mul_mxfp8` in
include/qdq_b200.h).
"""

from __future__ import annotations

import dataclasses

import torch

from .. import _native

RMSNORM_MAX_K = 65536  # QDQ_RMSNORM_MAX_K of include/qdq_b200.h
_DTYPES = (torch.bfloat16, torch.float16)


def scale_stride(k: int) -> int:
    """Scales per stored row: K / 32 rounded up to a multiple of 16."""
    return (k + 511) // 512 * 16


@dataclasses.dataclass(slots=True)
class Mxfp8Rows:
    """Rows of MXFP8: element (m, k) stands for E4M3(codes[m, k]) * 2^(scales[m, k // 32] - 127).

    The rows of `scales` lie `scale_stride(K)` bytes apart, or further, in a
    storage that holds the last one's padding too (the products read 16 scales
    at a time; `from_codes` lays scales out so).  `dtype` is the 16-bit type of
    the tensor the rows were made from, and of a product's output.
    """

    codes: torch.Tensor    # uint8 [M, K] E4M3
    scales: torch.Tensor   # uint8 [M, K / 32] E8M0, padded row stride
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> "Mxfp8Rows":
        """From codes uint8 [M, K] and scales uint8 [M, K / 32], as `mxfp8_quantize` returns them (K % 32 == 0)."""
        _native.require_cuda(codes, scales)
        _native.same_device(codes.device, scales)
        assert codes.dtype == torch.uint8 and scales.dtype == torch.uint8, (codes.dtype, scales.dtype)
        assert dtype in _DTYPES, f"MXFP8 rows stand for fp16/bf16 tensors, but got {dtype}"
        assert codes.dim() == 2 and codes.shape[1] > 0 and codes.shape[1] % 32 == 0, tuple(codes.shape)
        m, k = codes.shape
        assert tuple(scales.shape) == (m, k // 32), (tuple(codes.shape), tuple(scales.shape))
        stored = torch.empty((m, scale_stride(k)), dtype=torch.uint8, device=codes.device)[:, : k // 32]
        return cls(_native.rows16(codes), stored.copy_(scales), dtype)

    def dequantize(self) -> torch.Tensor:
        """The values in `dtype`: what `mxfp8_qdq` returns for the same tensor."""
        m, k = self.codes.shape
        scale = torch.exp2(self.scales.float() - 127)
        v = self.codes.view(torch.float8_e4m3fn).float().view(m, k // 32, 32) * scale.unsqueeze(-1)
        return v.view(m, k).to(self.dtype)


# The CUDA kernels of these schemas are csrc/torch_ops.cpp, loaded by the first call.
_LIB = torch.library.Library("qdq_b200", "FRAGMENT")
_LIB.define("mxfp8_rows(Tensor x) -> (Tensor, Tensor)")
_LIB.define("silu_mul_mxfp8(Tensor x) -> (Tensor, Tensor)")
_LIB.define("rmsnorm_mxfp8(Tensor x, Tensor weight, Tensor? residual, float eps, bool norm_out) -> Tensor[]")
_rows_op = torch.ops.qdq_b200.mxfp8_rows.default
_silu_mul_op = torch.ops.qdq_b200.silu_mul_mxfp8.default
_rmsnorm_op = torch.ops.qdq_b200.rmsnorm_mxfp8.default


def _new_rows(x: torch.Tensor, m: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    return (x.new_empty((m, k), dtype=torch.uint8),
            x.new_empty_strided((m, k // 32), (scale_stride(k), 1), dtype=torch.uint8))


@torch.library.register_fake("qdq_b200::mxfp8_rows")
def _(x):
    return _new_rows(x, x.shape[0], x.shape[1])


@torch.library.register_fake("qdq_b200::silu_mul_mxfp8")
def _(x):
    return _new_rows(x, x.shape[0], x.shape[1] // 2)


@torch.library.register_fake("qdq_b200::rmsnorm_mxfp8")
def _(x, weight, residual, eps, norm_out):
    more = int(residual is not None) + int(norm_out)
    return [*_new_rows(x, *x.shape), *(x.new_empty(x.shape) for _ in range(more))]


def _check(name: str, x: torch.Tensor, parts: int = 1) -> None:
    assert x.dim() == 2, f"{name} only supports 2D tensors, but got {x.dim()}D"
    assert x.dtype in _DTYPES, f"{name} only supports fp16/bf16 tensors, but got {x.dtype}"
    k = x.shape[1] // parts
    assert k > 0 and k % 32 == 0, f"{name}: K={k} must be a positive multiple of 32"
    _native.require_cuda(x)


# The C++ ops refuse what is malformed before any launch.  The checks here give
# the errors of the other operators (AssertionError for shapes and types); they
# run only where a call was refused, or has no CUDA tensor to dispatch on.
def mxfp8_rows(x: torch.Tensor) -> Mxfp8Rows:
    """MXFP8 rows of x [M, K] bf16/fp16 (CUDA, K % 32 == 0): the codes and scales of `mxfp8_quantize`.

    A NaN stays one.  An infinity gives its group of 32 the scale 2^-127, in which it saturates and every value beside it
    too: what the group then adds to a product is next to nothing (the rule of `mxfp8_qdq`).
    """
    try:
        _native.load_ops(x)
        return Mxfp8Rows(*_rows_op(x), x.dtype)
    except RuntimeError:
        _check("mxfp8_rows", x)
        raise


def silu_mul_mxfp8(x: torch.Tensor) -> Mxfp8Rows:
    """MXFP8 rows [M, K] of silu(x[:, :K]) * x[:, K:], the gated activation between a layer's two products.

    Args:
        x: [M, 2K] bf16/fp16 (CUDA, K % 32 == 0), gate first.

    The product is formed in fp32 and rounded to x's dtype before it is quantised.
    """
    try:
        _native.load_ops(x)
        return Mxfp8Rows(*_silu_mul_op(x), x.dtype)
    except RuntimeError:
        _check("silu_mul_mxfp8", x, 2)
        raise


def rmsnorm_mxfp8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                  norm_out: bool = False) -> tuple[Mxfp8Rows, torch.Tensor | None, torch.Tensor | None]:
    """RMSNorm in front of an MXFP8 product, with the residual's addition.

        h = x + residual              (rounded to x's dtype; h = x without a residual)
        y = h * rsqrt(mean(h^2) + eps) * weight     (fp32, rounded to x's dtype)

    The squares' sum leaves fp32's range for no finite row, bf16's largest and smallest among them.

    Args:
        x: [M, K] bf16/fp16 (CUDA), K a multiple of 32 up to 65536.
        weight: [K] of x's dtype.
        residual: [M, K] of x's dtype, or None.
        eps: added to the mean square; not negative.
        norm_out: also return y, e.g. for a router that reads it in 16 bits.

    Returns:
        (MXFP8 rows of y, h or None without a residual, y or None).
    """
    try:
        _native.load_ops(x)
        out = _rmsnorm_op(x, weight, residual, eps, norm_out)
    except RuntimeError:
        _check("rmsnorm_mxfp8", x)
        k = x.shape[1]
        assert k <= RMSNORM_MAX_K, f"rmsnorm_mxfp8: K={k} is above {RMSNORM_MAX_K}"
        assert weight.dim() == 1 and weight.shape[0] == k and weight.dtype == x.dtype, (
            f"rmsnorm_mxfp8: weight must be a [{k}] tensor of {x.dtype}")
        assert residual is None or (residual.shape == x.shape and residual.dtype == x.dtype), (
            "rmsnorm_mxfp8: residual must have x's shape and dtype")
        assert eps >= 0, f"rmsnorm_mxfp8: eps={eps} must not be negative"
        raise
    return (Mxfp8Rows(out[0], out[1], x.dtype), out[2] if residual is not None else None,
            out[-1] if norm_out else None)
