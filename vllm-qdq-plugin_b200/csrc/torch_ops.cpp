// torch.library kernels of the MXFP8 operators: the CUDA implementations of
// the schemas that vllm_qdq_plugin/qdq/mxfp8_rows.py and gemm.py define.
// They allocate outputs and workspaces on torch's current stream and call the
// C ABI (include/qdq_b200.h).  These calls sit on the path of single tokens,
// where the host's time is the call's time, so they are C++ rather than ctypes:
// one norm call of a single row takes 10 us on the host, of which the GPU works
// 2.1, and through ctypes took 25 (a torch addition takes 4.6).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "qdq_b200.h"

// The torch that this file was compiled against, as text in the library: it is rebuilt for another.
extern "C" const char qdq_torch_ops_built_for[] = QDQ_BUILT_FOR;

namespace {

using at::Tensor;

void check(const char* fn, int status) {
  TORCH_CHECK(status == QDQ_OK, fn, " failed with status ", status, ": ", qdq_last_error());
}

int dtype_code(const Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, "expected a bf16 or fp16 tensor");
  return t.scalar_type() == at::kHalf ? QDQ_DTYPE_FP16 : QDQ_DTYPE_BF16;
}

// The tensor, or a copy whose rows are apart (not broadcast) and start on 16-byte boundaries with unit element stride.
Tensor rows16(const Tensor& t) {
  const bool dense = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 &&
                     (t.dim() < 2 || t.size(0) <= 1 ||
                      (t.stride(0) >= t.size(1) && t.stride(0) * t.element_size() % 16 == 0));
  return dense ? t : t.clone(at::MemoryFormat::Contiguous);
}

int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* ptr(const Tensor& t) { return const_cast<void*>(t.const_data_ptr()); }
void* ptr(const std::optional<Tensor>& t) { return t.has_value() ? ptr(*t) : nullptr; }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
// Straight from torch's caching allocator, without the dispatcher.
Tensor empty(at::IntArrayRef size, at::ScalarType dtype, const Tensor& like) {
  return at::detail::empty_cuda(size, dtype, like.device(), std::nullopt);
}
Tensor bytes(int64_t m, int64_t n, const Tensor& like) { return empty({m, n}, at::kByte, like); }
Tensor bytes(int64_t n, const Tensor& like) { return empty({n}, at::kByte, like); }

// What the C ABI cannot see of its pointers: shapes, types and devices.
void check_16bit(const char* name, const Tensor& x) {
  TORCH_CHECK(x.dim() == 2, name, " only supports 2D tensors, but got ", x.dim(), "D");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, name,
              " only supports fp16/bf16 tensors, but got ", x.scalar_type());
}
void check_k(const char* name, int64_t k) {
  TORCH_CHECK(k > 0 && k % 32 == 0, name, ": K=", k, " must be a positive multiple of 32");
}
void check_device(const Tensor& x, const Tensor& t) {
  TORCH_CHECK(t.device() == x.device(), "expected every tensor on ", x.device(), ", got one on ", t.device());
}
// MXFP8 rows: scales [M, K / 32] whose rows lie in storage padded to the stride the products read.
void check_rows(const char* name, const Tensor& codes, const Tensor& scales) {
  TORCH_CHECK(codes.dim() == 2 && codes.scalar_type() == at::kByte && scales.dim() == 2 &&
                  scales.scalar_type() == at::kByte && scales.size(0) == codes.size(0) &&
                  scales.size(1) * 32 == codes.size(1),
              name, ": malformed MXFP8 rows");
  const int64_t m = codes.size(0), need = qdq_mxfp8_scale_stride(codes.size(1));
  TORCH_CHECK(codes.stride(1) == 1 && (scales.size(1) == 1 || scales.stride(1) == 1), name,
              ": MXFP8 rows must be dense along K");
  const int64_t step = m > 1 ? scales.stride(0) : need;
  TORCH_CHECK(m == 0 || (step >= need && static_cast<int64_t>(scales.storage().nbytes()) >=
                                             scales.storage_offset() + (m - 1) * step + need),
              name, ": the scales' rows are not padded (make the rows with Mxfp8Rows.from_codes)");
  check_device(codes, scales);
}
int64_t scale_ld(const Tensor& scales, int64_t k) {
  return scales.size(0) > 1 ? scales.stride(0) : qdq_mxfp8_scale_stride(k);
}
// [m, k / 32] scales in storage of whole padded rows.
Tensor new_scales(int64_t m, int64_t k, const Tensor& like) {
  const int64_t lds = qdq_mxfp8_scale_stride(k);
  Tensor t = bytes(m, lds, like);
  const int64_t sizes[2] = {m, k / 32}, strides[2] = {lds, 1};
  t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes, 2), at::IntArrayRef(strides, 2));
  return t;
}
Tensor dense_as(const std::optional<Tensor>& t, at::ScalarType dtype) {
  return t.has_value() ? t->to(dtype).contiguous() : Tensor();
}
void* ptr_or_null(const Tensor& t) { return t.defined() ? ptr(t) : nullptr; }

template <typename F>
std::tuple<Tensor, Tensor> rows_op(const char* name, F fn, const Tensor& x_, int64_t k) {
  check_k(name, k);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows16(x_);
  const int64_t m = x.size(0), lds = qdq_mxfp8_scale_stride(k);
  Tensor codes = bytes(m, k, x), scales = new_scales(m, k, x);
  check(name, fn(ptr(x), ptr(codes), ptr(scales), m, k, ld(x), k, lds, dtype_code(x), stream()));
  return {codes, scales};
}

std::tuple<Tensor, Tensor> mxfp8_rows(const Tensor& x) {
  check_16bit("mxfp8_rows", x);
  return rows_op("qdq_mxfp8_rows", &qdq_mxfp8_rows, x, x.size(1));
}

std::tuple<Tensor, Tensor> silu_mul_mxfp8(const Tensor& x) {
  check_16bit("silu_mul_mxfp8", x);
  TORCH_CHECK(x.size(1) % 2 == 0, "silu_mul_mxfp8: ", x.size(1), " columns are not two halves");
  return rows_op("qdq_silu_mul_mxfp8", &qdq_silu_mul_mxfp8, x, x.size(1) / 2);
}

std::vector<Tensor> rmsnorm_mxfp8(const Tensor& x_, const Tensor& weight, const std::optional<Tensor>& residual,
                                  double eps, bool norm_out) {
  const char* name = "rmsnorm_mxfp8";
  check_16bit(name, x_);
  const int64_t m = x_.size(0), k = x_.size(1), lds = qdq_mxfp8_scale_stride(k);
  check_k(name, k);
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == k && weight.scalar_type() == x_.scalar_type(), name,
              ": weight must be a [", k, "] tensor of the activation's dtype");
  check_device(x_, weight);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows16(x_), w = rows16(weight);
  std::vector<Tensor> out;
  out.reserve(4);
  Tensor r;
  void *h = nullptr, *y = nullptr;
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), name,
                ": residual must have the activation's shape and dtype");
    check_device(x, *residual);
    r = rows16(*residual);
  }
  out.push_back(bytes(m, k, x));
  out.push_back(new_scales(m, k, x));
  if (r.defined()) {
    out.push_back(empty({m, k}, x.scalar_type(), x));
    h = ptr(out.back());
  }
  if (norm_out) {
    out.push_back(empty({m, k}, x.scalar_type(), x));
    y = ptr(out.back());
  }
  check("qdq_rmsnorm_mxfp8",
        qdq_rmsnorm_mxfp8(ptr(x), ptr_or_null(r), ptr(w), h, y, ptr(out[0]), ptr(out[1]), m, k, ld(x),
                          r.defined() ? ld(r) : k, k, k, k, lds, static_cast<float>(eps), dtype_code(x), stream()));
  return out;
}

// A weight's scales in the tiled layout.
void check_scales(const char* name, const Tensor& sf, int64_t need) {
  TORCH_CHECK(sf.element_size() == 1 && sf.is_contiguous() && sf.numel() >= need, name, ": the weight's tiled scales need ",
              need, " bytes, got ", sf.numel());
}

void check_linear(const char* name, const Tensor& a, const Tensor& w, const Tensor& sf, const std::optional<Tensor>& bias) {
  TORCH_CHECK(w.dim() == 2 && w.size(1) == a.size(1), name, ": K=", a.size(1), " of the activation is not the weight's");
  TORCH_CHECK(w.element_size() == 1 && w.stride(1) == 1, name, ": the weight's codes must be bytes, dense along K");
  check_scales(name, sf, qdq_sf_tiled_bytes(w.size(0), w.size(1)));
  check_device(a, w);
  check_device(a, sf);
  if (bias.has_value()) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == w.size(0), name, ": bias must be [", w.size(0), "]");
    check_device(a, *bias);
  }
}

Tensor mxfp8_linear(const Tensor& a_, const Tensor& w, const Tensor& sf, const std::optional<Tensor>& bias) {
  check_16bit("mxfp8_linear", a_);
  check_linear("mxfp8_linear", a_, w, sf, bias);
  const c10::cuda::CUDAGuard guard(a_.device());
  const Tensor a = rows16(a_), b = dense_as(bias, a.scalar_type());
  const int64_t m = a.size(0), k = a.size(1), n = w.size(0), need = fp8_linear_workspace_bytes(m, k);
  Tensor ws = bytes(need, a), out = empty({m, n}, a.scalar_type(), a);
  check("fp8_linear_mxf8", fp8_linear_mxf8(ptr(a), ld(a), dtype_code(a), ptr(w), ptr(sf), ptr_or_null(b), ptr(out), m, n,
                                           k, ld(w), n, ptr(ws), need, stream()));
  return out;
}

Tensor mxfp8_linear_rows(const Tensor& codes, const Tensor& scales, const Tensor& w, const Tensor& sf,
                         const std::optional<Tensor>& bias, bool out_fp16) {
  check_rows("mxfp8_linear", codes, scales);
  check_linear("mxfp8_linear", codes, w, sf, bias);
  const c10::cuda::CUDAGuard guard(codes.device());
  const auto dtype = out_fp16 ? at::kHalf : at::kBFloat16;
  const Tensor b = dense_as(bias, dtype);
  const int64_t m = codes.size(0), k = codes.size(1), n = w.size(0);
  Tensor out = empty({m, n}, dtype, codes);
  check("fp8_gemm_mxf8",
        fp8_gemm_mxf8(ptr(codes), ptr(scales), ld(codes), scale_ld(scales, k), ptr(w), ptr(sf), ptr_or_null(b), ptr(out), m, n, k,
                      ld(w), n, out_fp16 ? QDQ_DTYPE_FP16 : QDQ_DTYPE_BF16, stream()));
  return out;
}

void mxfp8_moe_linear_out(const Tensor& a_, const std::optional<Tensor>& a_scales, const Tensor& w, const Tensor& sf,
                          const Tensor& sorted_ids, const Tensor& expert_ids, const Tensor& num_post_padded,
                          const std::optional<Tensor>& topk_weights, int64_t block, int64_t top_k, Tensor out) {
  const char* name = "mxfp8_moe_linear";
  const bool raw = !a_scales.has_value();
  if (raw) check_16bit(name, a_);
  else check_rows(name, a_, *a_scales);
  TORCH_CHECK(w.dim() == 3 && w.is_contiguous() && w.size(2) == a_.size(1), name, ": K=", a_.size(1),
              " of the activation is not the weight's");
  TORCH_CHECK(w.element_size() == 1, name, ": the weight's codes must be bytes");
  check_scales(name, sf, w.size(0) * qdq_sf_tiled_bytes(w.size(1), w.size(2)));
  TORCH_CHECK(top_k >= 1 && block >= 1 && block <= 64, name, ": top_k must be positive, moe_block_size in [1, 64]");
  const int64_t slots = a_.size(0) * top_k, n = w.size(1);
  for (const Tensor* t : {&sorted_ids, &expert_ids, &num_post_padded}) {
    TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), name, ": routing tensors are dense int32");
    check_device(a_, *t);
  }
  TORCH_CHECK(num_post_padded.numel() >= 1 && expert_ids.numel() >= sorted_ids.numel() / block, name,
              ": expert_ids has one entry per block");
  TORCH_CHECK(out.dim() == 2 && out.size(0) == slots && out.size(1) == n && (n <= 1 || out.stride(1) == 1) &&
                  (!raw || out.scalar_type() == a_.scalar_type()),
              name, ": out must be [M * top_k, N] of the activation's dtype with dense rows");
  for (const Tensor* t : {&w, &sf, const_cast<const Tensor*>(&out)}) check_device(a_, *t);
  if (topk_weights.has_value()) {
    TORCH_CHECK(topk_weights->numel() == slots, name, ": topk_weights has one entry per slot");
    check_device(a_, *topk_weights);
  }
  const c10::cuda::CUDAGuard guard(a_.device());
  const Tensor a = raw ? rows16(a_) : a_, tw = dense_as(topk_weights, at::kFloat);
  const int64_t m = a.size(0), k = a.size(1), sorted = sorted_ids.numel();
  const int64_t need = fp8_moe_workspace_bytes(m, sorted, static_cast<int>(block), k);
  Tensor ws = bytes(need, a);
  check("fp8_moe_mxf8",
        fp8_moe_mxf8(raw ? ptr(a) : nullptr, raw ? ld(a) : 0, raw ? nullptr : ptr(a), ptr(a_scales), raw ? 0 : ld(a),
                     raw ? 0 : scale_ld(*a_scales, k), dtype_code(out), ptr(w), ptr(sf), w.size(0),
                     static_cast<const int32_t*>(ptr(sorted_ids)), static_cast<const int32_t*>(ptr(expert_ids)),
                     static_cast<const int32_t*>(ptr(num_post_padded)), static_cast<const float*>(ptr_or_null(tw)),
                     sorted, static_cast<int>(block), static_cast<int>(top_k), tw.defined() ? 1 : 0, ptr(out),
                     out.size(0) > 1 ? out.stride(0) : n, m, n, k, ptr(ws), need, stream()));
}

Tensor mxfp8_moe_linear(const Tensor& a, const std::optional<Tensor>& a_scales, const Tensor& w, const Tensor& sf,
                        const Tensor& sorted_ids, const Tensor& expert_ids, const Tensor& num_post_padded,
                        const std::optional<Tensor>& topk_weights, int64_t block, int64_t top_k, bool out_fp16) {
  TORCH_CHECK(a.dim() == 2 && w.dim() == 3 && top_k >= 1, "mxfp8_moe_linear: [M, K] rows, [E, N, K] weights");
  const c10::cuda::CUDAGuard guard(a.device());
  Tensor out = empty({a.size(0) * top_k, w.size(1)}, out_fp16 ? at::kHalf : at::kBFloat16, a);
  mxfp8_moe_linear_out(a, a_scales, w, sf, sorted_ids, expert_ids, num_post_padded, topk_weights, block, top_k, out);
  return out;
}

// There is no CPU fallback.
void refuse_cpu(const c10::OperatorHandle& op, torch::jit::Stack*) {
  TORCH_CHECK(false, op.schema().operator_name(), " needs CUDA tensors on an sm_100 GPU (there is no CPU fallback)");
}

}  // namespace

TORCH_LIBRARY_IMPL(qdq_b200, CPU, m) {
  for (const char* name : {"mxfp8_rows", "silu_mul_mxfp8", "rmsnorm_mxfp8", "mxfp8_linear", "mxfp8_linear_rows",
                           "mxfp8_moe_linear", "mxfp8_moe_linear_out"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse_cpu>());
}

TORCH_LIBRARY_IMPL(qdq_b200, CUDA, m) {
  m.impl("mxfp8_rows", &mxfp8_rows);
  m.impl("silu_mul_mxfp8", &silu_mul_mxfp8);
  m.impl("rmsnorm_mxfp8", &rmsnorm_mxfp8);
  m.impl("mxfp8_linear", &mxfp8_linear);
  m.impl("mxfp8_linear_rows", &mxfp8_linear_rows);
  m.impl("mxfp8_moe_linear", &mxfp8_moe_linear);
  m.impl("mxfp8_moe_linear_out", &mxfp8_moe_linear_out);
}
