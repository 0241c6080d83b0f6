// Microscaled 4-bit floating point: sizes of the layout, and the arithmetic that every kernel applies when it
// makes or reads codes and block scales.
#pragma once
#include "common.cuh"
#include "spconvb_fp4.h"

namespace spconvb {
namespace fp4 {

__host__ __device__ inline uint32_t cpad(uint32_t channels) { return (channels + 63u) & ~63u; }
__host__ __device__ inline uint32_t code_pitch(uint32_t channels) { return cpad(channels) / 2; }
__host__ __device__ inline uint32_t scale_pitch(int format, uint32_t channels) {
  return format == SPCONVB_MXFP4 ? 4u * ((cpad(channels) + 127u) / 128u) : cpad(channels) / 16u;
}
inline bool format_ok(int f) { return f == SPCONVB_MXFP4 || f == SPCONVB_NVFP4; }
inline bool channels_ok(int c) { return c >= 1 && c <= SPCONVB_FP4_MAX_CHANNELS; }
// A tensor scale is a positive, finite, normal number; the format without one takes 1.
inline bool tensor_scale_ok(int format, float g) {
  return format == SPCONVB_MXFP4 ? g == 1.f : g >= 1.17549435e-38f && g <= 3.4e38f / 448.f;
}

// K is walked in chunks of 256 channels (128 bytes of codes a row), four MMAs of 64 channels each.  An MMA reads the
// scales of its 64 channels as bytes of one 32-bit word a row: four of 16 channels (NVFP4), or two of 32
// (MXFP4), in the lower or the upper half of a word that covers 128 channels.  Rows of 64 channels have their word for themselves.
constexpr uint32_t kChunkK = 256;
constexpr uint32_t kAtomBytes = 512;  // the scale words of 128 rows: word of row r at (r % 32) * 16 + (r / 32) * 4
__host__ __device__ inline uint32_t steps_per_word(int format, uint32_t cp) {
  return format == SPCONVB_MXFP4 && cp != 64u ? 2u : 1u;
}
__host__ __device__ inline uint32_t words_per_chunk(int format, uint32_t cp) {
  return 4u / steps_per_word(format, cp);
}

// 32, 16 and 8 bytes in program order.
__device__ __forceinline__ void st32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "l"(p)
               : "memory");
}
__device__ __forceinline__ void ld32(const void* p, uint32_t* v) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ uint4 ld16(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld8(const void* p) {
  uint2 v;
  asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}

// Two fp32 numbers in an instruction, each rounded as by itself: what these kernels spend is issue slots.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// The largest magnitude of m >= 0 and two more; and the same where a NaN counts as the largest.
__device__ __forceinline__ float max_abs(float m, float a, float b) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

__device__ __forceinline__ float max_abs_nan(float m, float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// The block scale of a block whose largest magnitude is `amax` (the bits of a float >= 0, infinity or NaN): its byte,
// and S in fp32.  x / S of MXFP4 is a multiplication by a power of two.
__device__ __forceinline__ uint32_t scale_mx(uint32_t amax_bits, float& s) {
  const uint32_t e = amax_bits >> 23;  // 0 for zero and subnormals, whose scale is the smallest one anyway
  const uint32_t byte = e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
  s = byte == 0u ? 5.8774717541114375e-39f : __uint_as_float(byte << 23);  // 2^-127 is a subnormal number
  return byte;
}
// A quotient x / d, correctly rounded, from the product with the reciprocal r of d and one correction by the exact remainder
// (Markstein 1990): where x is the product of d and a short number, as on the border between two codes, the corrected quotient is
// that number, and anywhere else it is within a last bit of the division's.  d between 2^-90 and 2^90 and |x / d| below 2^100, so that nothing overflows and no remainder loses bits.
__device__ __forceinline__ float quotient(float x, float d, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-q, d, x), r, q);
}
__device__ __forceinline__ F2 quotient2(F2 x, F2 minus_d, F2 r) {  // (d is given with its sign turned)
  const F2 q = mul2(x, r);
  return fma2(fma2(q, minus_d, x), r, q);
}
__host__ __device__ inline bool in_range(float d) { return d > 8.1e-28f && d < 1.2e27f; }

// What a tensor scale g gives to all blocks: 6 g and its reciprocal, 0 where that is out of range.
struct TensorScale {
  float g, six, inv_six;
};
inline TensorScale tensor_scale_of(float g) {
  TensorScale t{g, 6.f * g, 0.f};
  if (in_range(t.six)) t.inv_six = 1.f / t.six;
  return t;
}
__device__ __forceinline__ uint32_t scale_nv(uint32_t amax_bits, const TensorScale& t, float& s) {
  const float amax = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u) {
    s = 0.f;
    return 0x7fu;
  }
  const bool fast = t.inv_six != 0.f && amax * t.inv_six < 1e30f;  // (a quotient beyond fp32 is for the division: infinity, then 448)
  const float ratio = fast ? quotient(amax, t.six, t.inv_six) : __fdiv_rn(amax, t.six);
  uint16_t two;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.f), "f"(ratio));
  uint32_t half2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(half2) : "h"(two));
  s = __fmul_rn(__half2float(__ushort_as_half((uint16_t)half2)), t.g);
  return two & 0xffu;
}
// S of a stored byte.
__device__ __forceinline__ float scale_value(int format, uint32_t byte, float tensor_scale) {
  if (format == SPCONVB_MXFP4)
    return byte == 255u ? __uint_as_float(0x7fffffffu)
                        : (byte == 0u ? 5.8774717541114375e-39f : __uint_as_float(byte << 23));
  uint32_t half2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(half2) : "h"((uint16_t)byte));
  return __fmul_rn(__half2float(__ushort_as_half((uint16_t)half2)), tensor_scale);
}

// Eight values, already divided by S, to eight codes: round to nearest even, saturate at 6.
__device__ __forceinline__ uint32_t codes8(const float (&q)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return r;
}
// Eight codes to fp16 pairs (exact).
__device__ __forceinline__ void values8(uint32_t codes, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}

// N values of a block (a multiple of 8) to codes.  `s` and `amax_bits` are the block's.
template <int N>
__device__ __forceinline__ void codes_of(bool mx, const float* x, float s, uint32_t amax_bits, uint32_t* c) {
  if (amax_bits >= 0x7f800000u || s == 0.f) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) c[i] = 0u;
    return;
  }
  const float amax = __uint_as_float(amax_bits);
  float r;
  bool fast;
  if (mx) {
    // times 2^-e, exact; e = -127 .. 125, so its exponent field lies in 2 .. 254
    r = s < 1.1754944e-38f ? 1.7014118346046923e38f : __uint_as_float((254u << 23) - __float_as_uint(s));
    fast = true;
  } else {
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));  // (subnormal scales are out of range)
    fast = in_range(s) && amax * r < 1e30f;
  }
  if (fast) {
    const F2 r2(r, r), d2(-s, -s);
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      float q[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const F2 x2(x[8 * i + j], x[8 * i + j + 1]);
        (mx ? mul2(x2, r2) : quotient2(x2, d2, r2)).get(q[j], q[j + 1]);
      }
      c[i] = codes8(q);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      float q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = __fdiv_rn(x[8 * i + j], s);
      c[i] = codes8(q);
    }
  }
}

}  // namespace fp4
}  // namespace spconvb
