// Row kernels that end in MXFP8: the activations of the MXFP8 products.
//
//   rows     y = x                                   (qdq_mxfp8_rows)
//   silu_mul y = round(silu(g) * u), x = [g | u]     (qdq_silu_mul_mxfp8)
//   rmsnorm  h = round(x + r),
//            y = round(h * rsqrt(mean(h^2) + eps) * w)   (qdq_rmsnorm_mxfp8)
//
// followed by MXFP8 of y: per 32 elements e = floor(log2 amax) - 8 and E4M3
// codes of y / 2^e (mx_quant.cuh, the rule of qdq_mxfp8).  `round` is to the
// tensors' 16-bit type: y is what the unfused operator would have stored, so
// that the codes are those of mxfp8_qdq behind it.  All sums and products
// before it are fp32.
//
// Layout: codes [M, K] row-major bytes; scales [M, lds] row-major E8M0 bytes,
// K / 32 of them followed by zeros up to a multiple of 16, so that the product
// loads 16 scales (512 elements of K) of a row at once and its last stage
// finds 2^-127 rather than a stale NaN behind K.
//
// All three are one HBM pass: a lane owns 16-byte chunks (8 elements), the
// four lanes of a group exchange their maxima by shuffles.
#include <algorithm>
#include <cstring>

#include "mx_quant.cuh"
#include "sm100.cuh"

namespace qdqb200 {
namespace {

using namespace sm100;

constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr int kRowThreads = 256;

// Scale exponent of the 32-group this lane's chunk belongs to (four
// neighbouring lanes hold the group).
template <int kDtype>
__device__ __forceinline__ int group_exp(const uint4& y) {
  uint32_t amax = absmax8(y);
  amax = max(amax, __shfl_xor_sync(kAll, amax, 1));
  amax = max(amax, __shfl_xor_sync(kAll, amax, 2));
  return mx8_exp<kDtype>(amax);
}

// Codes and scale of one chunk; chunk `col` of a row of cpr chunks.  The lane
// of the row's last group also clears the scale bytes behind K / 32.
__device__ __forceinline__ void store_chunk(uint8_t* codes_row, uint8_t* scales_row, uint32_t col, uint32_t cpr,
                                            uint2 code, int e) {
  *reinterpret_cast<uint2*>(codes_row + col * 8u) = code;
  if ((col & 3u) == 0) {
    const uint32_t g = col >> 2, gpr = cpr >> 2;
    scales_row[g] = static_cast<uint8_t>(e);
    if (g + 1 == gpr)
      for (uint32_t p = gpr; p < ((gpr + 15u) & ~15u); ++p) scales_row[p] = 0;
  }
}

// silu(g) * u without overflow of exp: t = exp(-|g|) <= 1.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float t = __expf(-fabsf(g));
  return g * __fdividef(g < 0.f ? t : 1.0f, 1.0f + t) * u;
}

// ---------------------------------------------------------------------------
// rows / silu_mul: a flat walk over the 16-byte chunks of all rows.
// ---------------------------------------------------------------------------
template <int kDtype, bool kSilu>
__global__ void __launch_bounds__(kRowThreads)
rows_mxfp8_kernel(const uint16_t* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                  uint32_t cpr, uint64_t total, int64_t ldx, int64_t ldc, int64_t lds, float zero) {
  using F = Fmt<kDtype>;
  constexpr int kU = kSilu ? 2 : 4;  // chunks in flight per lane (silu_mul: two loads each)
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t stride = static_cast<uint64_t>(gridDim.x) * blockDim.x * kU;
  const bool narrow = total <= 0xFFFFFFFFull;
  for (uint64_t base = (static_cast<uint64_t>(blockIdx.x) * blockDim.x + (threadIdx.x & ~31u)) * kU; base < total;
       base += stride) {
    uint4 v[kU], u[kU];
    uint64_t row[kU];
    uint32_t col[kU];
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      const uint64_t c = base + static_cast<uint64_t>(i) * 32u + lane;
      row[i] = narrow ? static_cast<uint32_t>(c) / cpr : c / cpr;
      col[i] = static_cast<uint32_t>(c - row[i] * cpr);
      v[i] = u[i] = make_uint4(0, 0, 0, 0);
      if (c < total) {
        const uint16_t* p = x + row[i] * ldx + col[i] * 8u;
        v[i] = ld_stream(reinterpret_cast<const uint4*>(p));
        if (kSilu) u[i] = ld_stream(reinterpret_cast<const uint4*>(p + cpr * 8u));
      }
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      if (kSilu) {
        uint32_t g4[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        const uint32_t u4[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          g4[j] = F::pack(silu_mul(F::lo(g4[j]), F::lo(u4[j])), silu_mul(F::hi(g4[j]), F::hi(u4[j])));
        v[i] = make_uint4(g4[0], g4[1], g4[2], g4[3]);
      }
      const int e = group_exp<kDtype>(v[i]);
      if (base + static_cast<uint64_t>(i) * 32u + lane < total)
        store_chunk(codes + row[i] * ldc, scales + row[i] * lds, col[i], cpr, mx8_chunk_codes<kDtype>(v[i], e, zero), e);
    }
  }
}

// ---------------------------------------------------------------------------
// rmsnorm: one row per warp (kWarpRow, up to 32 * kC chunks) or per CTA; the
// row stays in registers (kC chunks per thread) between the sum of squares
// and the output, so every input byte is read once.
// ---------------------------------------------------------------------------
template <int kDtype, int kC, bool kWarpRow>
__global__ void __launch_bounds__(kWarpRow ? kRowThreads : 1024)
rmsnorm_mxfp8_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ res, const uint16_t* __restrict__ w,
                     uint16_t* __restrict__ h_out, uint16_t* __restrict__ y_out, uint8_t* __restrict__ codes,
                     uint8_t* __restrict__ scales, int64_t M, uint32_t cpr, int64_t ldx, int64_t ldr, int64_t ldh,
                     int64_t ldy, int64_t ldc, int64_t lds, float eps, float zero) {
  using F = Fmt<kDtype>;
  __shared__ float part[32];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint32_t t = kWarpRow ? lane : threadIdx.x, step = kWarpRow ? 32u : blockDim.x;
  const int64_t row0 = kWarpRow ? static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + warp : blockIdx.x;
  const int64_t rstep = kWarpRow ? static_cast<int64_t>(gridDim.x) * (kRowThreads / 32) : gridDim.x;
  for (int64_t row = row0; row < M; row += rstep) {
    uint4 h[kC];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const uint32_t col = t + i * step;
      h[i] = col < cpr ? ld_stream(reinterpret_cast<const uint4*>(x + row * ldx + col * 8u)) : make_uint4(0, 0, 0, 0);
    }
    if (res != nullptr) {
      uint4 r[kC];
#pragma unroll
      for (int i = 0; i < kC; ++i) {
        const uint32_t col = t + i * step;
        r[i] = col < cpr ? ld_stream(reinterpret_cast<const uint4*>(res + row * ldr + col * 8u)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kC; ++i) {
        const uint32_t a4[4] = {h[i].x, h[i].y, h[i].z, h[i].w}, r4[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = F::pack(__fadd_rn(F::lo(a4[j]), F::lo(r4[j])), __fadd_rn(F::hi(a4[j]), F::hi(r4[j])));
        h[i] = make_uint4(o[0], o[1], o[2], o[3]);
        const uint32_t col = t + i * step;
        if (col < cpr) *reinterpret_cast<uint4*>(h_out + row * ldh + col * 8u) = h[i];
      }
    }
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const uint32_t a4[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = F::lo(a4[j]), b = F::hi(a4[j]);
        ss = fmaf(a, a, fmaf(b, b, ss));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kAll, ss, o);
    if (!kWarpRow) {
      // the barrier at the loop's end keeps this row's sums until every thread has read them
      if (lane == 0) part[warp] = ss;
      __syncthreads();
      ss = lane < (blockDim.x >> 5) ? part[lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kAll, ss, o);
    }
    const float rs = rsqrtf(ss / (static_cast<float>(cpr) * 8.0f) + eps);
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const uint32_t col = t + i * step;
      const uint4 wv = col < cpr ? __ldg(reinterpret_cast<const uint4*>(w + col * 8u)) : make_uint4(0, 0, 0, 0);
      const uint32_t a4[4] = {h[i].x, h[i].y, h[i].z, h[i].w}, w4[4] = {wv.x, wv.y, wv.z, wv.w};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = F::pack(F::lo(a4[j]) * rs * F::lo(w4[j]), F::hi(a4[j]) * rs * F::hi(w4[j]));
      const uint4 y = make_uint4(o[0], o[1], o[2], o[3]);
      const int e = group_exp<kDtype>(y);
      if (col < cpr) {
        if (y_out != nullptr) *reinterpret_cast<uint4*>(y_out + row * ldy + col * 8u) = y;
        store_chunk(codes + row * ldc, scales + row * lds, col, cpr, mx8_chunk_codes<kDtype>(y, e, zero), e);
      }
    }
    if (!kWarpRow) __syncthreads();
  }
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// Launch with programmatic dependent launch: the kernel may start while the
// previous one on the stream finishes; every thread passes
// griddepcontrol.wait before it reads or writes global memory.
template <typename... P, typename... A>
int launch_pdl(const char* who, void (*fn)(P...), int64_t grid, int threads, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...);
  if (e != cudaSuccess) return fail(QDQ_ERR_CUDA, "%s: launch: %s", who, cudaGetErrorString(e));
  return check_launch(who);
}

// What every row kernel asks of its sizes and outputs.
int check_rows(const char* who, const void* x, const void* codes, const void* scales, int64_t M, int64_t K,
               int64_t width, int64_t ldx, int64_t ldc, int64_t lds, int dtype) {
  if (dtype != QDQ_DTYPE_BF16 && dtype != QDQ_DTYPE_FP16)
    return fail(QDQ_ERR_INVALID_ARG, "%s: dtype must be bf16 (0) or fp16 (1)", who);
  if (M < 0 || K < 0) return fail(QDQ_ERR_INVALID_ARG, "%s: negative shape", who);
  if (K % 32 != 0) return fail(QDQ_ERR_UNSUPPORTED, "%s: K=%lld must be a multiple of 32", who, (long long)K);
  if (K > (1ll << 30) || M > (1ll << 40)) return fail(QDQ_ERR_UNSUPPORTED, "%s: dimension too large", who);
  if (M == 0 || K == 0) return QDQ_OK;
  if (!x || !codes || !scales) return fail(QDQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if (ldx < width || ldc < K || lds < qdq_mxfp8_scale_stride(K))
    return fail(QDQ_ERR_INVALID_ARG, "%s: row stride too small", who);
  if (off16(x) || ldx % 8 || off16(codes) || ldc % 16 || off16(scales) || lds % 16)
    return fail(QDQ_ERR_ALIGNMENT, "%s: rows of x, codes and scales must be 16-byte aligned", who);
  return QDQ_OK;
}

template <bool kSilu>
int rows_entry(const char* who, const void* x, void* codes, void* scales, int64_t M, int64_t K, int64_t ldx,
               int64_t ldc, int64_t lds, int dtype, void* stream) {
  if (int st = check_rows(who, x, codes, scales, M, K, kSilu ? 2 * K : K, ldx, ldc, lds, dtype)) return st;
  if (M == 0 || K == 0) return QDQ_OK;
  const uint32_t cpr = static_cast<uint32_t>(K / 8);
  const uint64_t total = static_cast<uint64_t>(M) * cpr;
  const uint64_t per = static_cast<uint64_t>(kRowThreads) * (kSilu ? 2 : 4);
  const int64_t grid = static_cast<int64_t>(std::min<uint64_t>((total + per - 1) / per, 1u << 30));
  auto fn = dtype == QDQ_DTYPE_FP16 ? &rows_mxfp8_kernel<QDQ_DTYPE_FP16, kSilu>
                                    : &rows_mxfp8_kernel<QDQ_DTYPE_BF16, kSilu>;
  return launch_pdl(who, fn, grid, kRowThreads, static_cast<cudaStream_t>(stream), static_cast<const uint16_t*>(x),
                    static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), cpr, total, ldx, ldc, lds, 0.0f);
}

}  // namespace
}  // namespace qdqb200

using namespace qdqb200;

extern "C" int64_t qdq_mxfp8_scale_stride(int64_t K) { return K <= 0 ? 0 : ((K + 31) / 32 + 15) / 16 * 16; }

extern "C" int qdq_mxfp8_rows(const void* x, void* codes, void* scales, int64_t M, int64_t K, int64_t ldx,
                              int64_t ldc, int64_t lds, int dtype, void* stream) {
  return rows_entry<false>("qdq_mxfp8_rows", x, codes, scales, M, K, ldx, ldc, lds, dtype, stream);
}

extern "C" int qdq_silu_mul_mxfp8(const void* x, void* codes, void* scales, int64_t M, int64_t K, int64_t ldx,
                                  int64_t ldc, int64_t lds, int dtype, void* stream) {
  return rows_entry<true>("qdq_silu_mul_mxfp8", x, codes, scales, M, K, ldx, ldc, lds, dtype, stream);
}

extern "C" int qdq_rmsnorm_mxfp8(const void* x, const void* residual, const void* weight, void* residual_out,
                                 void* y, void* codes, void* scales, int64_t M, int64_t K, int64_t ldx, int64_t ldr,
                                 int64_t ldh, int64_t ldy, int64_t ldc, int64_t lds, float eps, int dtype,
                                 void* stream) {
  const char* who = "qdq_rmsnorm_mxfp8";
  if (int st = check_rows(who, x, codes, scales, M, K, K, ldx, ldc, lds, dtype)) return st;
  if (K > QDQ_RMSNORM_MAX_K)
    return fail(QDQ_ERR_UNSUPPORTED, "%s: K=%lld is above %d", who, (long long)K, QDQ_RMSNORM_MAX_K);
  if (!(eps >= 0.0f)) return fail(QDQ_ERR_INVALID_ARG, "%s: eps must be >= 0", who);
  if (M == 0 || K == 0) return QDQ_OK;
  if (!weight) return fail(QDQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if ((residual != nullptr) != (residual_out != nullptr))
    return fail(QDQ_ERR_INVALID_ARG, "%s: residual and residual_out go together", who);
  if ((residual && (ldr < K || ldh < K)) || (y && ldy < K))
    return fail(QDQ_ERR_INVALID_ARG, "%s: row stride too small", who);
  if (off16(weight) || (residual && (off16(residual) || off16(residual_out) || ldr % 8 || ldh % 8)) ||
      (y && (off16(y) || ldy % 8)))
    return fail(QDQ_ERR_ALIGNMENT, "%s: rows must be 16-byte aligned", who);
  const uint32_t cpr = static_cast<uint32_t>(K / 8);
  const bool f16 = dtype == QDQ_DTYPE_FP16;
  auto go = [&](auto fn_bf16, auto fn_f16, int threads, int64_t rows_per_cta) {
    const int64_t grid = std::min<int64_t>((M + rows_per_cta - 1) / rows_per_cta, 1 << 30);
    return launch_pdl(who, f16 ? fn_f16 : fn_bf16, grid, threads, static_cast<cudaStream_t>(stream),
                      static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual),
                      static_cast<const uint16_t*>(weight), static_cast<uint16_t*>(residual_out),
                      static_cast<uint16_t*>(y), static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), M, cpr,
                      ldx, ldr, ldh, ldy, ldc, lds, eps, 0.0f);
  };
#define QDQ_NORM(C, WARP, THREADS, RPC) \
  return go(&rmsnorm_mxfp8_kernel<QDQ_DTYPE_BF16, C, WARP>, &rmsnorm_mxfp8_kernel<QDQ_DTYPE_FP16, C, WARP>, THREADS, RPC)
  if (cpr <= 32) QDQ_NORM(1, true, kRowThreads, kRowThreads / 32);
  if (cpr <= 64) QDQ_NORM(2, true, kRowThreads, kRowThreads / 32);
  if (cpr <= 128) QDQ_NORM(4, true, kRowThreads, kRowThreads / 32);
  auto threads = [&](int c) { return static_cast<int>((cpr + 32 * c - 1) / (32 * c) * 32); };
  if (cpr <= 1024) QDQ_NORM(2, false, threads(2), 1);
  if (cpr <= 4096) QDQ_NORM(4, false, threads(4), 1);
  QDQ_NORM(8, false, threads(8), 1);
#undef QDQ_NORM
}
