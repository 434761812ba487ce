// MX group quantisation shared by the QDQ kernels and the fused linears: the
// reference's per-dtype exponent / scale rules and the codes of one group,
// MXFP4 (vllm_qdq_plugin/qdq/mxfp4.py:98-156), NVFP4 and MXFP8
// (vllm_qdq_plugin/qdq/mxfp8.py:73-125).  Everything here reproduces the
// reference bit for bit.
#pragma once

#include "common.cuh"

namespace qdqb200 {
namespace {

// ---------------------------------------------------------------------------
// per-dtype pieces
// ---------------------------------------------------------------------------
template <int kDtype>
struct Fmt;

template <>
struct Fmt<QDQ_DTYPE_BF16> {
  __device__ static float lo(uint32_t w) { return bf16lo(w); }
  __device__ static float hi(uint32_t w) { return bf16hi(w); }
  __device__ static float one(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }
  __device__ static uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  __device__ static uint16_t pack1(float a) { return static_cast<uint16_t>(pack_bf16x2(a, 0.f) & 0xFFFFu); }
  __device__ static float amax_value(uint32_t bits) { return __uint_as_float(bits << 16); }
  // E8M0 exponent of the group scale from the group's max |x| bit pattern:
  // round the mantissa up at 0.75 (`+0x20 & 0xFF80`, mxfp4.py:138-140), then
  // clamp(floor(log2) + 127 - 2, 0, 254) (mxfp4.py:142-145).  A rounded max of
  // zero, inf or NaN makes the reference's float->int32 cast of +-inf land on
  // the lower clamp, i.e. exponent 0.
  __device__ static int mx_exp(uint32_t amax_bits) {
    const uint32_t r = (amax_bits + 0x20u) & 0xFF80u;
    const int ef = static_cast<int>((r >> 7) & 0xFFu);
    return (ef == 0 || ef == 255) ? 0 : max(ef - 2, 0);
  }
  // 2^(e-127) as the reference holds it in bf16 (mxfp4.py:146): always exact.
  __device__ static float mx_scale(int e) {
    return e ? __uint_as_float(static_cast<uint32_t>(e) << 23) : __uint_as_float(0x00400000u);
  }
  static constexpr bool kScaleCanBeZero = false;
};

template <>
struct Fmt<QDQ_DTYPE_FP16> {
  __device__ static float lo(uint32_t w) { return f16lo(w); }
  __device__ static float hi(uint32_t w) { return f16hi(w); }
  __device__ static float one(uint16_t b) { return __half2float(__ushort_as_half(b)); }
  __device__ static uint32_t pack(float a, float b) { return pack_f16x2(a, b); }
  __device__ static uint16_t pack1(float a) { return static_cast<uint16_t>(pack_f16x2(a, 0.f) & 0xFFFFu); }
  __device__ static float amax_value(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
  // fp16 variant of the same rule (`+0x100 & 0xFC00`, exponent bias 15).
  __device__ static int mx_exp(uint32_t amax_bits) {
    const uint32_t r = (amax_bits + 0x100u) & 0xFC00u;
    const int ef = static_cast<int>((r >> 10) & 0x1Fu);
    return (ef == 0 || ef == 31) ? 0 : ef + 110;
  }
  // In fp16, 2^(e-127) underflows to 0 for e == 0 and is exact otherwise
  // (e >= 111 for every finite non-tiny group).
  __device__ static float mx_scale(int e) {
    return e ? __uint_as_float(static_cast<uint32_t>(e) << 23) : 0.0f;
  }
  static constexpr bool kScaleCanBeZero = true;
};

// fp16 groups whose scale is 0: the reference divides by zero, turning x != 0
// into +-inf and +-0 into a NaN whose sign on x86 is negative; the E2M1
// simulation maps both to +-6 and the final multiply by the zero scale leaves
// a signed zero.  Result: copysign(0, x) for x != 0, -0 for x == +-0.
__device__ __forceinline__ uint16_t fp16_zero_scale_result(uint16_t xb) {
  return ((xb & 0x7FFFu) == 0) ? static_cast<uint16_t>(0x8000u) : static_cast<uint16_t>(xb & 0x8000u);
}
__device__ __forceinline__ uint32_t fp16_zero_scale_word(uint32_t w) {
  return static_cast<uint32_t>(fp16_zero_scale_result(static_cast<uint16_t>(w & 0xFFFFu))) |
         (static_cast<uint32_t>(fp16_zero_scale_result(static_cast<uint16_t>(w >> 16))) << 16);
}

// E2M1 byte holding two signed zeros with the signs of an fp16x2 word.
__device__ __forceinline__ uint32_t zero_codes_of(uint32_t w) {
  return ((w >> 12) & 0x8u) | ((w >> 24) & 0x80u);
}

__device__ __forceinline__ uint32_t absmax8(const uint4& v) {
  const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                              __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
  return max(m & 0xFFFFu, m >> 16);
}

// MXFP4 codes of one 32-element group held as four 16-byte chunks (8
// elements each): returns the E8M0 exponent byte and writes the four code
// words (element 2j of a chunk in the low nibble of byte j).  These are the
// codes the QDQ kernel emits for the same group.
template <int kDtype>
__device__ __forceinline__ int mx_group_codes(const uint4 (&v)[4], uint32_t (&code)[4]) {
  using F = Fmt<kDtype>;
  const uint32_t amax = max(max(absmax8(v[0]), absmax8(v[1])), max(absmax8(v[2]), absmax8(v[3])));
  const int e = F::mx_exp(amax);
  const float inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);  // 1/scale, exact
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
    if (F::kScaleCanBeZero && e == 0) {
      uint32_t cw = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) cw |= zero_codes_of(fp16_zero_scale_word(w[j])) << (8 * j);
      code[c] = cw;
    } else {
      float sv[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = mul_f32x2(make_float2(F::lo(w[j]), F::hi(w[j])), make_float2(inv, inv));
        sv[2 * j] = t.x;
        sv[2 * j + 1] = t.y;
      }
      code[c] = cvt_e2m1x8(sv[0], sv[1], sv[2], sv[3], sv[4], sv[5], sv[6], sv[7]);
    }
  }
  return e;
}


// ---------------------------------------------------------------------------
// NVFP4 group math (nvfp4_emulation_utils.py:439-452 and :474-476)
// ---------------------------------------------------------------------------
constexpr float kRecip6 = 1.0f / 6.0f;  // fp32 value of vLLM's FLOAT4_E2M1_MAX_RECIPROCAL

struct NvGroup {
  float out_scale;  // 1 / (scale * (1/gs))  with vLLM's zero-safe reciprocal
  float deq;        // scale / gs
  uint32_t sbyte;   // E4M3 byte of the block scale
};

__device__ __forceinline__ float zero_safe_recip(float t) {
  // get_reciprocal(t) = 1 / (t + (t == 0) * 1e8)   (nvfp4_emulation_utils.py:415-418)
  return __fdiv_rn(1.0f, __fadd_rn(t, t == 0.0f ? 1e8f : 0.0f));
}

__device__ __forceinline__ NvGroup nv_group(float vec_max, float gs, float rgs) {
  float s = __fmul_rn(gs, __fmul_rn(vec_max, kRecip6));
  s = fminf(fmaxf(s, -448.0f), 448.0f);
  NvGroup g;
  g.sbyte = e4m3_byte(s);
  s = round_e4m3(s);
  g.out_scale = zero_safe_recip(__fmul_rn(s, rgs));
  g.deq = __fdiv_rn(s, gs);
  return g;
}

// Codes of two elements x*out_scale.  The reference clamps to +-6 and rounds
// to nearest-even (nvfp4_emulation_utils.py:450-451, :425-436): the
// satfinite E2M1 conversion does both.  cast_to_fp4 multiplies by
// torch.sign(), which is +0 for a -0 product (x == -0, or an underflow), so a
// zero product is encoded as +0.
__device__ __forceinline__ uint32_t nv_codes(float xa, float xb, float out_scale) {
  const float2 p = mul_f32x2(make_float2(xa, xb), make_float2(out_scale, out_scale));
  uint32_t byte = cvt_e2m1x2(p.x, p.y);
  if (p.x == 0.0f) byte &= 0xF7u;
  if (p.y == 0.0f) byte &= 0x7Fu;
  return byte;
}

// With out_scale >= 2^-16 no nonzero bf16 or fp16 input (smallest magnitude
// 2^-133, resp. 2^-24) has a product below the smallest fp32 subnormal
// 2^-149, so the only zero products are those of x == +-0.
constexpr float kNoUnderflowScale = 0x1p-16f;

// x * out_scale for 8 elements, with a zero product made +0 (see nv_codes):
// the product is formed as fma(x, out_scale, zero) with `zero` = +0.0 passed
// in as a kernel argument (an operand the compiler cannot treat as a
// constant), so an exact -0 product becomes -0 + +0 = +0 under RN while every
// other product is rounded exactly once, as by a plain multiply.
__device__ __forceinline__ void nv_scale8(const uint32_t (&w)[4], float out_scale, float zero, float (&sv)[8],
                                          bool fp16) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = fp16 ? f16lo(w[j]) : bf16lo(w[j]);
    const float b = fp16 ? f16hi(w[j]) : bf16hi(w[j]);
    const float2 t = fma_f32x2(make_float2(a, b), make_float2(out_scale, out_scale), make_float2(zero, zero));
    sv[2 * j] = t.x;
    sv[2 * j + 1] = t.y;
  }
}

// NVFP4 codes of one 16-element group (two 16-byte chunks of bf16/fp16, in
// order) with the per-tensor global scale gs (rgs = its zero-safe
// reciprocal): the codes and E4M3 scale byte of vLLM's NVFP4 quantisation,
// as nvfp4_vec_kernel computes them.  code[c] holds chunk c's eight codes.
template <int kDtype>
__device__ __forceinline__ uint32_t nv_group_codes(const uint4 (&v)[2], float gs, float rgs, float zero,
                                                   uint32_t (&code)[2]) {
  using F = Fmt<kDtype>;
  const uint32_t amax = max(absmax8(v[0]), absmax8(v[1]));
  const NvGroup g = nv_group(F::amax_value(amax), gs, rgs);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
    if (g.out_scale >= kNoUnderflowScale) {
      float sv[8];
      nv_scale8(w, g.out_scale, zero, sv, kDtype == QDQ_DTYPE_FP16);
      code[c] = cvt_e2m1x8(sv[0], sv[1], sv[2], sv[3], sv[4], sv[5], sv[6], sv[7]);
    } else {
      uint32_t cw = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) cw |= nv_codes(F::lo(w[j]), F::hi(w[j]), g.out_scale) << (8 * j);
      code[c] = cw;
    }
  }
  return g.sbyte;
}

// ---------------------------------------------------------------------------
// MXFP8 group math (vllm_qdq_plugin/qdq/mxfp8.py:73-125), bit-exact
// ---------------------------------------------------------------------------
// Scale exponent 127 + floor(log2(max(amax, FLT_MIN))) - 8, clamped to
// [0, 254] (mxfp8.py:104-112).  For a bf16/fp16 maximum, floor(log2) is the
// fp32 exponent field (their mantissas are too short for log2 to round up to
// the next integer); a zero or sub-FLT_MIN maximum sits at FLT_MIN (-126);
// inf / NaN give 0, the x86 float->int32 cast of +-inf / NaN.
template <int kDtype>
__device__ __forceinline__ int mx8_exp(uint32_t amax_bits) {
  const uint32_t b = __float_as_uint(Fmt<kDtype>::amax_value(amax_bits));
  const int ef = static_cast<int>(b >> 23);
  if (ef == 255) return 0;
  return min(max((ef == 0 ? -126 : ef - 127) + 119, 0), 254);
}
__device__ __forceinline__ float pow2f(int e) {  // 2^e, e in [-127, 127]
  return __uint_as_float(e > -127 ? static_cast<uint32_t>(e + 127) << 23 : 0x00400000u);
}
// The reference's E4M3 grid (mxfp8.py:40-70) is round-to-nearest-even with
// saturation at 448, except that its subnormal branch is clamped to 7 * 2^-9
// (:57): magnitudes in [7.5, 8) * 2^-9 give 7 * 2^-9 where RNE gives 2^-6.
// Lowering [7, 8) * 2^-9 to 7 * 2^-9 before the hardware conversion
// reproduces that.
__device__ __forceinline__ float mx8_sub_clamp(float v) {
  const uint32_t u = __float_as_uint(v);
  return ((u & 0x7FFFFFFFu) - 0x3C600000u < 0x00200000u) ? __uint_as_float((u & 0x80000000u) | 0x3C600000u) : v;
}
// Two values -> E4M3 pair (a in the low byte) and its exact fp16x2 decode.
__device__ __forceinline__ uint32_t e4m3x2_roundtrip(float a, float b, uint32_t& h) {
  uint32_t out;
  asm("{\n\t.reg .b16 t;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 t, %3, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, t;\n\t"
      "cvt.u32.u16 %0, t;\n\t}"
      : "=r"(out), "=r"(h)
      : "f"(a), "f"(b));
  return out;
}
// The same two steps on an f16x2 pair of quotients: magnitudes in
// [7, 8) * 2^-9 (fp16 0x2300 .. 0x23FF) lose their low mantissa bits, which
// leaves 7 * 2^-9 with the sign; then E4M3 with the exact fp16x2 decode.  The
// quotients of the fast path fit fp16 exactly: |x / scale| < 2^9, at most 11
// significant bits, and those below 2^-14 (fp16 subnormals, rounded) are far
// below 2^-10, where every E4M3 code is zero.
__device__ __forceinline__ uint32_t mx8_pair_f16(uint32_t h, uint32_t& dec) {
  uint32_t eq, out;
  asm("{\n\t.reg .b32 m;\n\t"
      "and.b32 m, %1, 0x7F007F00;\n\t"
      "set.eq.u32.f16x2 %0, m, %2;\n\t}"
      : "=r"(eq)
      : "r"(h), "r"(0x23002300u));
  h &= ~(eq & 0x00FF00FFu);
  asm("{\n\t.reg .b16 t;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 t, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, t;\n\t"
      "cvt.u32.u16 %0, t;\n\t}"
      : "=r"(out), "=r"(dec)
      : "r"(h));
  return out;
}
// x / scale for a pair.  torch.sign makes a zero quotient +0 (mxfp8.py:46,
// :70): with fma(x, inv, zero), zero = +0.0 a kernel argument, an exact -0
// becomes +0.  That covers every zero quotient while no nonzero input can
// underflow: inv >= 2^-16 (scale exponent <= 143), always so for fp16.
// Above it, zero quotients are cleared by comparison.
__device__ __forceinline__ float2 mx8_scaled(float a, float b, float inv, float zero, bool fast) {
  if (fast) return fma_f32x2(make_float2(a, b), make_float2(inv, inv), make_float2(zero, zero));
  float2 t = mul_f32x2(make_float2(a, b), make_float2(inv, inv));
  if (t.x == 0.0f) t.x = 0.0f;
  if (t.y == 0.0f) t.y = 0.0f;
  return t;
}

// E4M3 codes of a bf16 pair, w = x * inv with inv >= 2^-16 a power of two (as
// a bf16 pair): the product is exact in bf16 where it is a normal number, and
// below that, far under 2^-10, it rounds to a value of its own sign whose code
// is the zero of that sign, as that of the exact quotient; fma(x, inv, +0)
// makes a -0 quotient +0.  Magnitudes in [7, 8) * 2^-9 (bf16 0x3C60 .. 0x3C7F)
// lose their low mantissa bits as in mx8_pair_f16.
__device__ __forceinline__ uint32_t mx8_pair_bf16(uint32_t x, uint32_t inv2, uint32_t zero2) {
  uint32_t t, eq, out;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(t) : "r"(x), "r"(inv2), "r"(zero2));
  asm("{\n\t.reg .b32 m;\n\t"
      "and.b32 m, %1, 0x7FE07FE0;\n\t"
      "set.eq.u32.f16x2 %0, m, %2;\n\t}"  // equal bits: both are ordinary f16 numbers where they are equal
      : "=r"(eq)
      : "r"(t), "r"(0x3C603C60u));
  t &= ~(eq & 0x001F001Fu);
  asm("{\n\t.reg .b16 p;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 p, %2, %1;\n\t"
      "cvt.u32.u16 %0, p;\n\t}"
      : "=r"(out)
      : "f"(bf16lo(t)), "f"(bf16hi(t)));
  return out;
}

// E4M3 codes of the elements in kW words (two each) of a 32-group with scale
// exponent e, four per output word: the codes mxfp8_vec_kernel emits.
template <int kDtype, int kW>
__device__ __forceinline__ void mx8_codes(const uint32_t (&w)[kW], int e, float zero, uint32_t (&code)[kW / 2]) {
  using F = Fmt<kDtype>;
  const float inv = pow2f(127 - e);
  uint32_t p[kW];
  if (e <= 143) {
    if (kDtype == QDQ_DTYPE_BF16) {
      const uint32_t inv2 = pack_bf16x2(inv, inv), zero2 = __float_as_uint(zero);
#pragma unroll
      for (int j = 0; j < kW; ++j) p[j] = mx8_pair_bf16(w[j], inv2, zero2);
    } else {
#pragma unroll
      for (int j = 0; j < kW; ++j) {
        const float2 t = mx8_scaled(F::lo(w[j]), F::hi(w[j]), inv, zero, true);
        uint32_t h;
        p[j] = mx8_pair_f16(pack_f16x2(t.x, t.y), h);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kW; ++j) {
      const float2 t = mx8_scaled(F::lo(w[j]), F::hi(w[j]), inv, zero, false);
      uint32_t h;
      p[j] = e4m3x2_roundtrip(mx8_sub_clamp(t.x), mx8_sub_clamp(t.y), h);
    }
  }
#pragma unroll
  for (int j = 0; j < kW / 2; ++j) code[j] = __byte_perm(p[2 * j], p[2 * j + 1], 0x5410);
}

// Maximum magnitude bits of the 16-bit elements in kW words; a NaN gives an
// all-ones exponent, as an infinity does.
template <int kDtype, int kW>
__device__ __forceinline__ uint32_t absmax_words(const uint32_t (&w)[kW]) {
  uint32_t m = w[0];
#pragma unroll
  for (int j = 1; j < kW; ++j) {  // |m| = max(|m|, |w|); the sign is dropped below
    if (kDtype == QDQ_DTYPE_BF16) asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[j]));
    else asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[j]));
  }
  m &= 0x7FFF7FFFu;
  return max(m & 0xFFFFu, m >> 16);
}

}  // namespace
}  // namespace qdqb200
