// torch.library kernels of the MXFP8 operators: the CUDA implementations of
// the schemas that vllm_qdq_plugin/qdq/mxfp8_rows.py and gemm.py define.
// They allocate outputs and workspaces on torch's current stream and call the
// C ABI (include/qdq_b200.h).  These calls sit on the path of single tokens,
// where the host's time is the call's time, so they are C++ rather than ctypes:
// on the measured host one norm call takes 7 us instead of 25 (GPU time 2.7).
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "qdq_b200.h"

namespace {

using at::Tensor;

void check(const char* fn, int status) {
  TORCH_CHECK(status == QDQ_OK, fn, " failed with status ", status, ": ", qdq_last_error());
}

int dtype_code(const Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, "expected a bf16 or fp16 tensor");
  return t.scalar_type() == at::kHalf ? QDQ_DTYPE_FP16 : QDQ_DTYPE_BF16;
}

// The tensor, or a copy whose rows start on 16-byte boundaries with unit element stride.
Tensor rows16(const Tensor& t) {
  const bool dense = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 &&
                     (t.dim() < 2 || t.size(0) <= 1 || t.stride(0) * t.element_size() % 16 == 0);
  return dense ? t : t.clone(at::MemoryFormat::Contiguous);
}

int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* ptr(const Tensor& t) { return const_cast<void*>(t.const_data_ptr()); }
void* ptr(const std::optional<Tensor>& t) { return t.has_value() ? ptr(*t) : nullptr; }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
Tensor bytes(int64_t m, int64_t n, const Tensor& like) { return at::empty({m, n}, like.options().dtype(at::kByte)); }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

template <typename F>
std::tuple<Tensor, Tensor> rows_op(const char* name, F fn, const Tensor& x_, int64_t k) {
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows16(x_);
  const int64_t m = x.size(0), lds = qdq_mxfp8_scale_stride(k);
  Tensor codes = bytes(m, k, x), scales = bytes(m, lds, x);
  check(name, fn(ptr(x), ptr(codes), ptr(scales), m, k, ld(x), k, lds, dtype_code(x), stream()));
  return {codes, scales};
}

std::tuple<Tensor, Tensor> mxfp8_rows(const Tensor& x) {
  return rows_op("qdq_mxfp8_rows", &qdq_mxfp8_rows, x, x.size(1));
}

std::tuple<Tensor, Tensor> silu_mul_mxfp8(const Tensor& x) {
  return rows_op("qdq_silu_mul_mxfp8", &qdq_silu_mul_mxfp8, x, x.size(1) / 2);
}

std::vector<Tensor> rmsnorm_mxfp8(const Tensor& x_, const Tensor& weight, const std::optional<Tensor>& residual,
                                  double eps, bool norm_out) {
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows16(x_), w = rows16(weight);
  const int64_t m = x.size(0), k = x.size(1), lds = qdq_mxfp8_scale_stride(k);
  std::vector<Tensor> out;
  out.reserve(4);
  out.push_back(bytes(m, k, x));
  out.push_back(bytes(m, lds, x));
  Tensor r;
  void *h = nullptr, *y = nullptr;
  if (residual.has_value()) {
    r = rows16(*residual);
    out.push_back(at::empty({m, k}, x.options()));
    h = ptr(out.back());
  }
  if (norm_out) {
    out.push_back(at::empty({m, k}, x.options()));
    y = ptr(out.back());
  }
  check("qdq_rmsnorm_mxfp8",
        qdq_rmsnorm_mxfp8(ptr(x), r.defined() ? ptr(r) : nullptr, ptr(w), h, y, ptr(out[0]), ptr(out[1]), m, k, ld(x),
                          r.defined() ? ld(r) : k, k, k, k, lds, static_cast<float>(eps), dtype_code(x), stream()));
  return out;
}

Tensor mxfp8_linear(const Tensor& a_, const Tensor& w, const Tensor& sf, const std::optional<Tensor>& bias) {
  const c10::cuda::CUDAGuard guard(a_.device());
  const Tensor a = rows16(a_);
  const int64_t m = a.size(0), k = a.size(1), n = w.size(0), need = fp8_linear_workspace_bytes(m, k);
  Tensor ws = bytes(need, a), out = at::empty({m, n}, a.options());
  check("fp8_linear_mxf8", fp8_linear_mxf8(ptr(a), ld(a), dtype_code(a), ptr(w), ptr(sf), ptr(bias), ptr(out), m, n, k,
                                           ld(w), n, ptr(ws), need, stream()));
  return out;
}

Tensor mxfp8_linear_rows(const Tensor& codes, const Tensor& scales, const Tensor& w, const Tensor& sf,
                         const std::optional<Tensor>& bias, bool out_fp16) {
  const c10::cuda::CUDAGuard guard(codes.device());
  const int64_t m = codes.size(0), k = codes.size(1), n = w.size(0);
  Tensor out = at::empty({m, n}, codes.options().dtype(out_fp16 ? at::kHalf : at::kBFloat16));
  check("fp8_gemm_mxf8",
        fp8_gemm_mxf8(ptr(codes), ptr(scales), ld(codes), ld(scales), ptr(w), ptr(sf), ptr(bias), ptr(out), m, n, k,
                      ld(w), n, out_fp16 ? QDQ_DTYPE_FP16 : QDQ_DTYPE_BF16, stream()));
  return out;
}

void mxfp8_moe_linear(const Tensor& a_, const std::optional<Tensor>& a_scales, const Tensor& w, const Tensor& sf,
                      const Tensor& sorted_ids, const Tensor& expert_ids, const Tensor& num_post_padded,
                      const std::optional<Tensor>& topk_weights, int64_t block, int64_t top_k, Tensor out) {
  const c10::cuda::CUDAGuard guard(a_.device());
  const bool raw = !a_scales.has_value();
  const Tensor a = raw ? rows16(a_) : a_;
  const int64_t m = a.size(0), k = a.size(1), n = w.size(1), sorted = sorted_ids.numel();
  const int64_t need = fp8_moe_workspace_bytes(m, sorted, static_cast<int>(block), k);
  Tensor ws = bytes(need, a);
  check("fp8_moe_mxf8",
        fp8_moe_mxf8(raw ? ptr(a) : nullptr, raw ? ld(a) : 0, raw ? nullptr : ptr(a), ptr(a_scales), raw ? 0 : ld(a),
                     raw ? 0 : ld(*a_scales), dtype_code(out), ptr(w), ptr(sf), w.size(0),
                     static_cast<const int32_t*>(ptr(sorted_ids)), static_cast<const int32_t*>(ptr(expert_ids)),
                     static_cast<const int32_t*>(ptr(num_post_padded)), static_cast<const float*>(ptr(topk_weights)),
                     sorted, static_cast<int>(block), static_cast<int>(top_k), topk_weights.has_value() ? 1 : 0,
                     ptr(out), out.size(0) > 1 ? out.stride(0) : n, m, n, k, ptr(ws), need, stream()));
}

}  // namespace

TORCH_LIBRARY_IMPL(qdq_b200, CUDA, m) {
  m.impl("mxfp8_rows", &mxfp8_rows);
  m.impl("silu_mul_mxfp8", &silu_mul_mxfp8);
  m.impl("rmsnorm_mxfp8", &rmsnorm_mxfp8);
  m.impl("mxfp8_linear", &mxfp8_linear);
  m.impl("mxfp8_linear_rows", &mxfp8_linear_rows);
  m.impl("mxfp8_moe_linear", &mxfp8_moe_linear);
}
