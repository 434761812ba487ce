// Row kernels that end in MXFP8: the activations of the MXFP8 products.
//
//   rows     y = x                                   (qdq_mxfp8_rows)
//   silu_mul y = round(silu(g) * u), x = [g | u]     (qdq_silu_mul_mxfp8)
//   rmsnorm  h = round(x + r),
//            y = round(h * rsqrt(mean(h^2) + eps) * w)   (qdq_rmsnorm_mxfp8)
//
// followed by MXFP8 of y: per 32 elements e = floor(log2 amax) - 8 and E4M3
// codes of y / 2^e (mx_quant.cuh, the rule of qdq_mxfp8).  `round` is to the
// tensors' 16-bit type, and all sums and products before it are fp32: the codes
// are those of mxfp8_qdq behind an operator that rounds this formula once.  (One
// that also rounds h * rsqrt before w, or silu(g) before u, stores another y.)
//
// Layout: codes [M, K] row-major bytes; scales row-major E8M0 bytes, K / 32 a
// row, rows lds (a multiple of 16) apart, so that the product loads 16 scales
// (512 elements of K) of a row at once; what lies between is not written.
//
// All three are one HBM pass: a lane owns units of 16 elements (two 16-byte
// loads), the two lanes of a group exchange their maxima by a shuffle.
#include <algorithm>
#include <cstring>

#include "mx_quant.cuh"
#include "sm100.cuh"

namespace qdqb200 {
namespace {

using namespace sm100;

constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr int kRowThreads = 128;  // silu_mul [4096, 14336]: 49.4 us, at 256 threads 53.2, at 64 54.8

struct Unit {  // 16 elements of a row
  uint4 a, b;
};

// One 32-byte access where every row starts on a 32-byte boundary (kWide),
// two of 16 bytes elsewhere: the halves of a sector are then fetched apart.
template <bool kWide>
__device__ __forceinline__ Unit load_unit(const uint16_t* p) {
  Unit u;
  if (kWide) {
    asm volatile("ld.global.L1::no_allocate.L2::256B.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(u.a.x), "=r"(u.a.y), "=r"(u.a.z), "=r"(u.a.w), "=r"(u.b.x), "=r"(u.b.y), "=r"(u.b.z), "=r"(u.b.w)
                 : "l"(p));
  } else {
    const uint4* q = reinterpret_cast<const uint4*>(p);
    u = {ld_stream_ordered(q), ld_stream_ordered(q + 1)};
  }
  return u;
}
template <bool kWide>
__device__ __forceinline__ void store_unit(uint16_t* p, const Unit& u) {
  if (kWide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(u.a.x), "r"(u.a.y), "r"(u.a.z),
                 "r"(u.a.w), "r"(u.b.x), "r"(u.b.y), "r"(u.b.z), "r"(u.b.w)
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = u.a;
    reinterpret_cast<uint4*>(p)[1] = u.b;
  }
}
__device__ __forceinline__ Unit zero_unit() { return {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}; }
__device__ __forceinline__ void words(const Unit& u, uint32_t (&w)[8]) {
  w[0] = u.a.x, w[1] = u.a.y, w[2] = u.a.z, w[3] = u.a.w;
  w[4] = u.b.x, w[5] = u.b.y, w[6] = u.b.z, w[7] = u.b.w;
}
__device__ __forceinline__ Unit unit_of(const uint32_t (&w)[8]) {
  return {make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
}

// MXFP8 of unit `col` of a row: codes, and from the group's first lane the
// scale.  Every lane of the warp takes part in the shuffle.
template <int kDtype>
__device__ __forceinline__ void store_mxfp8(const uint32_t (&y)[8], uint8_t* codes_row, uint8_t* scales_row,
                                            uint32_t col, bool live, float zero) {
  uint32_t amax = absmax_words<kDtype>(y);
  amax = max(amax, __shfl_xor_sync(kAll, amax, 1));
  const int e = mx8_exp<kDtype>(amax);
  if (!live) return;
  uint32_t c[4];
  mx8_codes<kDtype>(y, e, zero, c);
  *reinterpret_cast<uint4*>(codes_row + col * 16u) = make_uint4(c[0], c[1], c[2], c[3]);
  if ((col & 1u) == 0) scales_row[col >> 1] = static_cast<uint8_t>(e);
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// silu(g) * u of a pair: with h = exp(-|g| / 2), silu(g) = g (g < 0 ? h^2 : 1) /
// (1 + h^2).  Nothing overflows, and h is a normal number down to |g| = 174:
// u comes between the two factors h, so that the product is right wherever it
// is a 16-bit number, however small silu(g) alone is.  The exponent of h has no
// offset: with exp(-|g|) carried times 2^24 instead, its rounding was that of
// 24 - |g| log2(e), and of 58.7 M fp16 outputs 117 had a code other than that of
// the exact product; with h it is 27, with expf and a division in fp32 25
// ([4096, 14336] in turn: fp16 51.3 us before, 51.8 with h; bf16 51.2, 51.7).
__device__ __forceinline__ float2 silu_mul(float2 g, float2 u) {
  constexpr float kC = -0.5f * 1.44269504088896341f;
  const float2 h = make_float2(ex2_approx(kC * fabsf(g.x)), ex2_approx(kC * fabsf(g.y)));
  const float2 d = fma_f32x2(h, h, make_float2(1.0f, 1.0f));
  const float2 n = make_float2(g.x < 0.f ? h.x : 1.0f, g.y < 0.f ? h.y : 1.0f);
  const float2 s = mul_f32x2(mul_f32x2(g, make_float2(rcp_approx(d.x), rcp_approx(d.y))), n);
  return mul_f32x2(mul_f32x2(s, u), n);
}

// ---------------------------------------------------------------------------
// rows / silu_mul: `tpr` threads (a power of two, at least 2) of gridDim.y
// CTAs walk a row, the next unit's loads in flight while one is converted.
// Addresses are formed once a row: silu_mul issues 20 instructions an element,
// near what the SMs can while HBM delivers it (as a flat walk with a division
// and three row products per unit it took 27, and 55 us instead of 49 for
// [4096, 14336], where HBM alone needs 45).
// ---------------------------------------------------------------------------
template <int kDtype, bool kSilu, bool kWide>
__global__ void __launch_bounds__(kRowThreads)
rows_mxfp8_kernel(const uint16_t* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t M,
                  uint32_t upr, uint32_t tpr, int64_t ldx, int64_t ldc, int64_t lds, float zero) {
  using F = Fmt<kDtype>;
  // In this order: a dependent that starts early still finds all that was written before this kernel (the few-rows
  // product reads its weight then).
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t rpc = kRowThreads / tpr, t = threadIdx.x & (tpr - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * rpc + threadIdx.x / tpr;
  const bool in_m = row < M;
  const uint16_t* xr = x + row * ldx;
  const uint16_t* ur = xr + upr * 16u;
  uint8_t* cr = codes + row * ldc;
  uint8_t* sr = scales + row * lds;
  const uint32_t step = tpr * gridDim.y, first = tpr * blockIdx.y + t;
  Unit v = zero_unit(), u = zero_unit();
  if (in_m && first < upr) {
    v = load_unit<kWide>(xr + first * 16u);
    if (kSilu) u = load_unit<kWide>(ur + first * 16u);
  }
  for (uint32_t col0 = tpr * blockIdx.y; col0 < upr; col0 += step) {
    const uint32_t col = col0 + t, next = col + step;
    Unit vn = zero_unit(), un = zero_unit();
    if (in_m && next < upr) {
      vn = load_unit<kWide>(xr + next * 16u);
      if (kSilu) un = load_unit<kWide>(ur + next * 16u);
    }
    uint32_t y[8];
    words(v, y);
    if (kSilu) {
      uint32_t u8[8];
      words(u, u8);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 s = silu_mul(make_float2(F::lo(y[j]), F::hi(y[j])), make_float2(F::lo(u8[j]), F::hi(u8[j])));
        y[j] = F::pack(s.x, s.y);
      }
    }
    store_mxfp8<kDtype>(y, cr, sr, col, in_m && col < upr, zero);
    v = vn;
    u = un;
  }
}

// A value summed over the row's threads, the same in all of them.  The caller
// has a barrier before `part` is written again.
template <bool kWarpRow>
__device__ __forceinline__ float row_sum(float v, float* part) {
  const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  if (!kWarpRow) {
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (blockDim.x >> 5) ? part[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  }
  return v;
}

// A bf16 row whose squares leave the range of fp32 (bf16 reaches from 2^-133 to
// 2^128), from its stored h: summed as (h f)^2 with a power of two f, and
// normalised as (h f) rsqrt(mean (h f)^2 + eps f^2) w.  It reads the row again:
// scaled in the registers of the kernel below, it cost all rows the order of
// their loads ([16384, 8192] 138.5 -> 150 us).
template <bool kWarpRow>
__device__ __forceinline__ void rmsnorm_far_row(const uint16_t* h, const uint16_t* w, uint16_t* y, uint8_t* codes,
                                             uint8_t* scales, uint32_t upr, float* part, float f, float eps, float zero) {
  using F = Fmt<QDQ_DTYPE_BF16>;
  const uint32_t t = kWarpRow ? threadIdx.x & 31u : threadIdx.x, step = kWarpRow ? 32u : blockDim.x;
  const uint4 *h4 = reinterpret_cast<const uint4*>(h), *w4 = reinterpret_cast<const uint4*>(w);
  float sq = 0.f;
#pragma unroll 1
  for (uint32_t col = t; col < upr; col += step) {
    uint32_t a8[8];
    words({__ldcg(h4 + 2 * col), __ldcg(h4 + 2 * col + 1)}, a8);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = F::lo(a8[j]) * f, b = F::hi(a8[j]) * f;
      sq = fmaf(a, a, fmaf(b, b, sq));
    }
  }
  if (!kWarpRow) __syncthreads();  // the sums of the caller have been read
  const float rs = rsqrtf(row_sum<kWarpRow>(sq, part) / (static_cast<float>(upr) * 16.0f) + eps * f * f);
#pragma unroll 1
  for (uint32_t col0 = 0; col0 < upr; col0 += step) {
    const uint32_t col = col0 + t;
    uint32_t a8[8] = {}, w8[8] = {};
    if (col < upr) {
      words({__ldcg(h4 + 2 * col), __ldcg(h4 + 2 * col + 1)}, a8);
      words({__ldcg(w4 + 2 * col), __ldcg(w4 + 2 * col + 1)}, w8);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      a8[j] = F::pack(F::lo(a8[j]) * f * rs * F::lo(w8[j]), F::hi(a8[j]) * f * rs * F::hi(w8[j]));
    if (y != nullptr && col < upr) store_unit<false>(y + col * 16u, unit_of(a8));
    store_mxfp8<QDQ_DTYPE_BF16>(a8, codes, scales, col, col < upr, zero);
  }
}

template <bool kWarpRow>
__device__ __noinline__ void rmsnorm_far_row_call(const uint16_t* h, const uint16_t* w, uint16_t* y, uint8_t* codes,
                                                  uint8_t* scales, uint32_t upr, float* part, float f, float eps, float zero) {
  rmsnorm_far_row<kWarpRow>(h, w, y, codes, scales, upr, part, f, eps, zero);
}

// ---------------------------------------------------------------------------
// rmsnorm: one row per warp (kWarpRow, up to 32 * kC units) or per CTA; the
// row stays in registers (kC units per thread) between the sum of squares
// and the output, so every input byte is read once.
// ---------------------------------------------------------------------------
template <int kDtype, int kC, bool kWarpRow, bool kWide>
__global__ void __launch_bounds__(kWarpRow ? kRowThreads : 1024)
rmsnorm_mxfp8_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ res, const uint16_t* __restrict__ w,
                     uint16_t* __restrict__ h_out, uint16_t* __restrict__ y_out, uint8_t* __restrict__ codes,
                     uint8_t* __restrict__ scales, int64_t M, uint32_t upr, int64_t ldx, int64_t ldr, int64_t ldh,
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
    Unit h[kC];
    const uint16_t* xr = x + row * ldx;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const uint32_t col = t + i * step;
      h[i] = col < upr ? load_unit<kWide>(xr + col * 16u) : zero_unit();
    }
    if (res != nullptr) {
      const uint16_t* rr = res + row * ldr;
      Unit r[kC];
#pragma unroll
      for (int i = 0; i < kC; ++i) {
        const uint32_t col = t + i * step;
        r[i] = col < upr ? load_unit<kWide>(rr + col * 16u) : zero_unit();
      }
#pragma unroll
      for (int i = 0; i < kC; ++i) {
        uint32_t a8[8], r8[8];
        words(h[i], a8);
        words(r[i], r8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 s = add_f32x2(make_float2(F::lo(a8[j]), F::hi(a8[j])), make_float2(F::lo(r8[j]), F::hi(r8[j])));
          a8[j] = F::pack(s.x, s.y);
        }
        h[i] = unit_of(a8);
        const uint32_t col = t + i * step;
        if (col < upr) store_unit<kWide>(h_out + row * ldh + col * 16u, h[i]);
      }
    }
    float2 sq = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      uint32_t a8[8];
      words(h[i], a8);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 a = make_float2(F::lo(a8[j]), F::hi(a8[j]));
        sq = fma_f32x2(a, a, sq);
      }
    }
    // The barrier at the loop's end keeps this row's sums until every thread has read them.
    const float ss = row_sum<kWarpRow>(sq.x + sq.y, part);
    // Out of fp32's range, or so near its lower end that squares are lost and eps does not outweigh them.  A call of
    // its own where a thread holds two units, whose registers it would crowd ([32768, 1024] 38.3 us, inlined 40.0, without
    // the test 38.4; [16384, 8192] 145.8, 146.4, 143.4); inlined elsewhere ([777, 2880] 3.65 us, by a call 4.5).
    if (kDtype == QDQ_DTYPE_BF16 && (!(ss <= 0x1p120f) || (ss < 0x1p-90f && eps < 0x1p-60f))) {
      const uint16_t* hr = res != nullptr ? h_out + row * ldh : xr;
      uint16_t* yr = y_out != nullptr ? y_out + row * ldy : nullptr;
      const float f = ss < 1.0f ? 0x1p90f : 0x1p-80f;
      if (kC == 2)
        rmsnorm_far_row_call<kWarpRow>(hr, w, yr, codes + row * ldc, scales + row * lds, upr, part, f, eps, zero);
      else
        rmsnorm_far_row<kWarpRow>(hr, w, yr, codes + row * ldc, scales + row * lds, upr, part, f, eps, zero);
      if (!kWarpRow) __syncthreads();
      continue;
    }
    const float rs = rsqrtf(ss / (static_cast<float>(upr) * 16.0f) + eps);
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const uint32_t col = t + i * step;
      Unit wv = zero_unit();
      if (col < upr) {
        const uint4* p = reinterpret_cast<const uint4*>(w + col * 16u);
        wv = {ld_ordered(p), ld_ordered(p + 1)};
      }
      uint32_t a8[8], w8[8];
      words(h[i], a8);
      words(wv, w8);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 n = mul_f32x2(mul_f32x2(make_float2(F::lo(a8[j]), F::hi(a8[j])), make_float2(rs, rs)),
                                   make_float2(F::lo(w8[j]), F::hi(w8[j])));
        a8[j] = F::pack(n.x, n.y);
      }
      if (y_out != nullptr && col < upr) store_unit<kWide>(y_out + row * ldy + col * 16u, unit_of(a8));
      store_mxfp8<kDtype>(a8, codes + row * ldc, scales + row * lds, col, col < upr, zero);
    }
    if (!kWarpRow) __syncthreads();
  }
}

bool off(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }
bool off16(const void* p) { return off(p, 16); }

// Launch with programmatic dependent launch: the kernel may start while the
// previous one on the stream finishes; every thread passes
// griddepcontrol.wait before it reads or writes global memory.
template <typename... P, typename... A>
int launch_pdl(const char* who, void (*fn)(P...), dim3 grid, int threads, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
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
  const uint32_t upr = static_cast<uint32_t>(K / 16);
  // Threads a row: the most that keep 3/4 of themselves busy over the walk.
  uint32_t tpr = 2;
  for (uint32_t c = 4; c <= kRowThreads && c / 2 < upr; c *= 2)
    if (4 * upr >= 3 * ((upr + c - 1) / c * c)) tpr = c;
  const int64_t rpc = kRowThreads / tpr, grid = (M + rpc - 1) / rpc;
  if (grid > (1ll << 31) - 1) return fail(QDQ_ERR_UNSUPPORTED, "%s: too many rows", who);
  // Few rows: a row's walk is split over CTAs, up to a few CTAs per SM (silu_mul [1, 14336]: 4.4 -> 2.6 us).
  const int64_t walks = (upr + tpr - 1) / tpr, room = 4 * device_sm_count();
  const int64_t split = std::max<int64_t>(1, std::min<int64_t>(walks, room / grid));
  // K % 32 == 0, so silu_mul's second half starts as aligned as the first
  const bool wide = !off(x, 32) && ldx % 16 == 0;
  auto fn = dtype == QDQ_DTYPE_FP16
                ? (wide ? &rows_mxfp8_kernel<QDQ_DTYPE_FP16, kSilu, true> : &rows_mxfp8_kernel<QDQ_DTYPE_FP16, kSilu, false>)
                : (wide ? &rows_mxfp8_kernel<QDQ_DTYPE_BF16, kSilu, true> : &rows_mxfp8_kernel<QDQ_DTYPE_BF16, kSilu, false>);
  return launch_pdl(who, fn, dim3(static_cast<unsigned>(grid), static_cast<unsigned>(split)), kRowThreads, static_cast<cudaStream_t>(stream), static_cast<const uint16_t*>(x),
                    static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), M, upr, tpr, ldx, ldc, lds, 0.0f);
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
  const uint32_t upr = static_cast<uint32_t>(K / 16);
  const bool f16 = dtype == QDQ_DTYPE_FP16;
  const bool wide = !(off(x, 32) || ldx % 16 || (residual && (off(residual, 32) || ldr % 16 || off(residual_out, 32) || ldh % 16)) ||
                      (y && (off(y, 32) || ldy % 16)));
  auto go = [&](auto bf16, auto f16w, auto bf16n, auto f16n, int threads, int64_t rows_per_cta) {
    const int64_t grid = std::min<int64_t>((M + rows_per_cta - 1) / rows_per_cta, 1 << 30);
    return launch_pdl(who, f16 ? (wide ? f16w : f16n) : (wide ? bf16 : bf16n), dim3(static_cast<unsigned>(grid)), threads, static_cast<cudaStream_t>(stream),
                      static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual),
                      static_cast<const uint16_t*>(weight), static_cast<uint16_t*>(residual_out),
                      static_cast<uint16_t*>(y), static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), M, upr,
                      ldx, ldr, ldh, ldy, ldc, lds, eps, 0.0f);
  };
#define QDQ_NORM(C, WARP, THREADS, RPC) \
  return go(&rmsnorm_mxfp8_kernel<QDQ_DTYPE_BF16, C, WARP, true>, &rmsnorm_mxfp8_kernel<QDQ_DTYPE_FP16, C, WARP, true>, \
            &rmsnorm_mxfp8_kernel<QDQ_DTYPE_BF16, C, WARP, false>, &rmsnorm_mxfp8_kernel<QDQ_DTYPE_FP16, C, WARP, false>, THREADS, RPC)
  // Units per thread: one for few rows, whose latency is the sync's and the reduction's ([1, 4096] 2.0 us, with two
  // 2.4; [777, 2880] 4.8 and 6.0), two where rows queue for the SMs and bytes in flight count ([16384, 8192] 137 us,
  // with one 147).
  if (upr <= 32) QDQ_NORM(1, true, kRowThreads, kRowThreads / 32);
  if (upr <= 64) QDQ_NORM(2, true, kRowThreads, kRowThreads / 32);
  auto threads = [&](int c) { return static_cast<int>((upr + 32 * c - 1) / (32 * c) * 32); };
  if (upr <= 1024 && M <= 8 * device_sm_count()) QDQ_NORM(1, false, threads(1), 1);
  if (upr <= 2048) QDQ_NORM(2, false, threads(2), 1);
  QDQ_NORM(4, false, threads(4), 1);
#undef QDQ_NORM
}
