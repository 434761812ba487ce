"""CPU: what the MXFP8 row and product entry points refuse, in Python and at the C ABI, before any launch."""

from __future__ import annotations

import pytest
import torch

from vllm_qdq_plugin import _native

BF16 = torch.bfloat16



def test_cpu_tensors_are_refused():
    from vllm_qdq_plugin.gemm import Mxfp8MoeWeight, Mxfp8Weight, mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_weight
    from vllm_qdq_plugin.qdq import Mxfp8Rows, mxfp8_rows, rmsnorm_mxfp8, silu_mul_mxfp8
    x, w = torch.zeros(4, 64, dtype=BF16), torch.ones(64, dtype=BF16)
    codes, scales = torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    i32 = torch.zeros(16, dtype=torch.int32)
    weight = Mxfp8Weight(codes, scales, 8, 64)
    moe = Mxfp8MoeWeight(codes[None], scales, 1, 8, 64)
    for call in (lambda: mxfp8_rows(x), lambda: silu_mul_mxfp8(x), lambda: rmsnorm_mxfp8(x, w),
                 lambda: Mxfp8Rows.from_codes(codes, scales), lambda: prepare_mxfp8_weight(codes, scales),
                 lambda: mxfp8_linear(x, weight),
                 lambda: mxfp8_moe_linear(x, moe, i32, i32, i32, None, 16, 1, False)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_errors_of_the_native_ops_reach_python():
    """An error raised inside the C++ library is a Python exception, not the end of the process."""
    from vllm_qdq_plugin import _build, qdq  # noqa: F401  (defines the schemas)
    _native.lib()
    torch.ops.load_library(str(_build.TORCH_OPS_PATH))
    x = torch.zeros(4, 64, dtype=BF16)
    for call in (lambda: torch.ops.qdq_b200.mxfp8_rows(x), lambda: torch.ops.qdq_b200.rmsnorm_mxfp8(x, x[0], x, 1e-6, True)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_row_operators_check_shapes_and_types():
    from vllm_qdq_plugin.qdq import mxfp8_rows, rmsnorm_mxfp8, silu_mul_mxfp8
    for fn in (mxfp8_rows, silu_mul_mxfp8):
        with pytest.raises(AssertionError, match="2D"):
            fn(torch.zeros(2, 3, 64, dtype=BF16))
        with pytest.raises(AssertionError, match="fp16/bf16"):
            fn(torch.zeros(2, 64))
        with pytest.raises(AssertionError, match="multiple of 32"):
            fn(torch.zeros(2, 80, dtype=BF16))
        with pytest.raises(AssertionError, match="multiple of 32"):
            fn(torch.zeros(2, 0, dtype=BF16))
    with pytest.raises(AssertionError, match="multiple of 32"):
        rmsnorm_mxfp8(torch.zeros(2, 40, dtype=BF16), torch.zeros(40, dtype=BF16))


def test_c_abi_refuses_bad_rows():
    lib = _native.lib()
    a = 1 << 20  # an aligned address that no launch is reached with

    def norm(x=a, r=None, w=a, h=None, y=None, codes=a, scales=a, m=4, k=64, ldx=64, ldr=64, ldh=64, ldy=64, ldc=64,
             lds=16, eps=1e-6, dtype=0):
        return lib.qdq_rmsnorm_mxfp8(x, r, w, h, y, codes, scales, m, k, ldx, ldr, ldh, ldy, ldc, lds, eps, dtype, None)

    def message(st, code, text):
        assert st == code and text.encode() in lib.qdq_last_error(), (st, lib.qdq_last_error())

    assert [lib.qdq_mxfp8_scale_stride(k) for k in (-1, 0, 32, 512, 544, 4096)] == [0, 0, 16, 16, 32, 128]
    message(norm(dtype=2), 1, "dtype")
    message(norm(m=-1), 1, "negative")
    message(norm(k=40), 2, "multiple of 32")
    message(norm(x=None), 1, "null")
    message(norm(w=None), 1, "null")
    message(norm(ldx=32), 1, "stride")
    message(norm(lds=0), 1, "stride")
    message(norm(k=1024, ldx=1024, ldc=1024, lds=16), 1, "stride")
    message(norm(x=a + 2), 5, "16-byte")
    message(norm(ldx=68), 5, "16-byte")
    message(norm(w=a + 2), 5, "16-byte")
    message(norm(r=a), 1, "together")
    message(norm(r=a, h=a, ldr=32), 1, "stride")
    message(norm(y=a, ldy=8), 1, "stride")
    message(norm(eps=float("nan")), 1, "eps")
    message(norm(eps=-1.0), 1, "eps")
    message(norm(k=65568, ldx=65568, ldc=65568, lds=2064), 2, "above")
    assert norm(m=0) == 0
    for fn, width in ((lib.qdq_mxfp8_rows, 1), (lib.qdq_silu_mul_mxfp8, 2)):
        message(fn(a, a, a, 4, 64, 64 * width - 8, 64, 16, 0, None), 1, "stride")
        message(fn(a, a, a, 4, 64, 64 * width, 64, 24, 0, None), 5, "16-byte")
        message(fn(a, a + 8, a, 4, 64, 64 * width, 64, 16, 0, None), 5, "16-byte")
        assert fn(None, None, None, 0, 64, 64 * width, 64, 16, 1, None) == 0


def test_c_abi_refuses_bad_products():
    lib = _native.lib()
    a = 1 << 20

    def message(st, code, text):
        assert st == code and text.encode() in lib.qdq_last_error(), (st, lib.qdq_last_error())

    def gemm(ac=a, asc=a, lda=64, lds=16, wc=a, sf=a, bias=None, c=a, m=4, n=8, k=64, ldw=64, ldc=8, dtype=0):
        return lib.fp8_gemm_mxf8(ac, asc, lda, lds, wc, sf, bias, c, m, n, k, ldw, ldc, dtype, None)

    message(gemm(dtype=5), 1, "dtype")
    message(gemm(k=48), 2, "multiple of 32")
    message(gemm(k=0), 2, "K == 0")
    message(gemm(m=1 << 30), 2, "too large")
    message(gemm(ac=None), 1, "null")
    message(gemm(ldc=7), 1, "leading")
    message(gemm(lds=8), 1, "leading")
    message(gemm(ldw=72), 5, "16-byte")
    message(gemm(sf=a + 8), 5, "16-byte")
    message(gemm(c=a + 1), 5, "16-byte")
    assert gemm(m=0) == 0 and gemm(n=0) == 0
    need = lib.fp8_linear_workspace_bytes(4, 64)
    assert need == 512 and lib.fp8_linear_workspace_bytes(0, 64) == 0

    def linear(x=a, lda=64, ws=a, nbytes=need):
        return lib.fp8_linear_mxf8(x, lda, 0, a, a, None, a, 4, 8, 64, 64, 8, ws, nbytes, None)

    message(linear(x=None), 1, "null")
    message(linear(ws=None), 1, "workspace")
    message(linear(ws=a + 128), 1, "workspace")
    message(linear(nbytes=need - 1), 1, "workspace")
    message(linear(x=a + 2), 5, "16-byte")

    def moe(x=a, lda=64, ac=None, asc=None, ldac=0, lds=0, e=2, sid=a, eid=a, npp=a, tw=None, sorted_=32, bs=16, top_k=1,
            mul=0, c=a, ldc=8, m=4, n=8, k=64, ws=a, nbytes=1 << 20):
        return lib.fp8_moe_mxf8(x, lda, ac, asc, ldac, lds, 0, a, a, e, sid, eid, npp, tw, sorted_, bs, top_k, mul, c,
                                ldc, m, n, k, ws, nbytes, None)

    message(moe(bs=0), 2, "moe_block_size")
    message(moe(bs=65), 2, "moe_block_size")
    message(moe(top_k=0), 1, "top_k")
    message(moe(x=None), 1, "null")
    message(moe(x=None, ac=a, asc=a, ldac=64, lds=0), 1, "leading")
    message(moe(x=None, ac=a + 4, asc=a, ldac=64, lds=16), 5, "16-byte")
    message(moe(mul=1), 1, "null")
    message(moe(ldc=4), 1, "leading")
    message(moe(ws=None), 1, "workspace")
    message(moe(nbytes=64), 1, "workspace")
    message(moe(e=1 << 40), 2, "too many rows")
    assert moe(sorted_=0) == 0 and moe(m=0) == 0 and moe(e=0) == 0
    assert moe(sorted_=15) == 0  # no whole block


def test_fake_kernels_give_the_shapes():
    """The ops trace without a GPU: their fake kernels give the shapes and types of the real outputs."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(5, 544, dtype=torch.float16, device="cuda")
        codes, scales = torch.ops.qdq_b200.mxfp8_rows(x)
        assert codes.shape == (5, 544) and scales.shape == (5, 17) and codes.dtype == scales.dtype == torch.uint8
        assert scales.stride() == (32, 1)
        codes, scales = torch.ops.qdq_b200.silu_mul_mxfp8(x[:, :64])
        assert codes.shape == (5, 32) and scales.shape == (5, 1)
        out = torch.ops.qdq_b200.rmsnorm_mxfp8(x, x[0], x, 1e-6, True)
        assert [tuple(t.shape) for t in out] == [(5, 544), (5, 17), (5, 544), (5, 544)] and out[2].dtype == x.dtype
        w, sf = torch.empty(7, 544, dtype=torch.uint8, device="cuda"), torch.empty(9, dtype=torch.uint8, device="cuda")
        assert torch.ops.qdq_b200.mxfp8_linear(x, w, sf, None).shape == (5, 7)
        y = torch.ops.qdq_b200.mxfp8_linear_rows(codes, scales, w, sf, None, False)
        assert y.shape == (5, 7) and y.dtype == torch.bfloat16
        ids = torch.empty(32, dtype=torch.int32, device="cuda")
        y = torch.ops.qdq_b200.mxfp8_moe_linear(x, None, w[None], sf, ids, ids, ids, None, 16, 2, True)
        assert y.shape == (10, 7) and y.dtype == torch.float16


def test_scale_stride_is_the_c_abis():
    from vllm_qdq_plugin.qdq.mxfp8_rows import RMSNORM_MAX_K, scale_stride
    lib = _native.lib()
    assert all(scale_stride(k) == lib.qdq_mxfp8_scale_stride(k) for k in range(32, 8192, 32))
    from conftest import REPO
    assert f"QDQ_RMSNORM_MAX_K {RMSNORM_MAX_K}" in (REPO / "include" / "qdq_b200.h").read_text()
