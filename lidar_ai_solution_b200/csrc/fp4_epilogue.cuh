// What both products do with their sums: a lane owns a row, 32 channels at a time.
#pragma once
#include "fp4.cuh"
#include "pdl.cuh"

namespace spconvb {
namespace fp4 {

struct Output {
  const float* bias;
  const __half* res;   // NULL: none
  uint8_t* out;
  uint8_t* out_scales;
  uint32_t cout, cpitch, spitch;
  float alpha;
  TensorScale ts;  // of 4-bit output
  int act, res_relu;
  int mode;    // 0: fp16, 1: MXFP4, 2: NVFP4
  int access;  // bytes of an fp16 row that may be stored (and of the residual, read) at once: 32, 16 or 2
};

// The residual's 32 channels from `col` on, as pairs (channels that do not exist: 0).  Read in program order: it may be what the
// launch before wrote.
__device__ __forceinline__ void load_residual(const Output& o, uint64_t row, uint32_t col, uint32_t (&r)[16]) {
  const __half* p = o.res + row * o.cout + col;
  if (o.access == 32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (col + 16u * i < o.cout) {
        ld32(p + 16 * i, r + 8 * i);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[8 * i + j] = 0u;
      }
    }
  } else if (o.access == 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (col + 8u * i < o.cout) v = ld16(p + 8 * i);
      r[4 * i] = v.x;
      r[4 * i + 1] = v.y;
      r[4 * i + 2] = v.z;
      r[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      r[i] = 0u;
      if (col + 2u * i < o.cout) r[i] = (uint32_t)load_in_order((const uint16_t*)p + 2 * i);
      if (col + 2u * i + 1u < o.cout) r[i] |= (uint32_t)load_in_order((const uint16_t*)p + 2 * i + 1) << 16;
    }
  }
}

// 32 channels of one row, from fp32 sums to memory.  `col` is a multiple of 32 below cout rounded up to 64; the row exists.
// A NaN passes through ReLU (fmaxf would drop it).
template <bool RES>
__device__ __forceinline__ void emit32(const Output& o, float (&y)[32], uint64_t row, uint32_t col,
                                       const uint32_t (&res)[16]) {
  const float lo = o.act == SPCONVB_ACT_RELU ? 0.f : -INFINITY;
  auto above = [](float v, float least) { return v < least ? least : v; };
  if (o.bias && col + 32u <= o.cout && ((uintptr_t)o.bias & 15u) == 0u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = __ldg((const float4*)(o.bias + col) + i);
      y[4 * i] = above(fmaf(y[4 * i], o.alpha, b.x), lo);
      y[4 * i + 1] = above(fmaf(y[4 * i + 1], o.alpha, b.y), lo);
      y[4 * i + 2] = above(fmaf(y[4 * i + 2], o.alpha, b.z), lo);
      y[4 * i + 3] = above(fmaf(y[4 * i + 3], o.alpha, b.w), lo);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      y[i] = col + i < o.cout ? above(fmaf(y[i], o.alpha, o.bias ? __ldg(o.bias + col + i) : 0.f), lo) : 0.f;
  }
  if (RES) {
    const float lo2 = o.res_relu ? 0.f : -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 r = __half22float2(*(const __half2*)&res[i]);
      y[2 * i] = above(__fadd_rn(__half2float(__float2half_rn(y[2 * i])), r.x), lo2);
      y[2 * i + 1] = above(__fadd_rn(__half2float(__float2half_rn(y[2 * i + 1])), r.y), lo2);
    }
  }
  if (o.mode == 0) {
    __half* p = (__half*)o.out + row * o.cout + col;
    uint32_t h[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __half2 two = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
      h[i] = *(const uint32_t*)&two;
    }
    if (o.access == 32) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (col + 16u * i < o.cout) st32(p + 16 * i, h + 8 * i);
    } else if (o.access == 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col + 8u * i < o.cout)
          ((uint4*)p)[i] = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (col + i < o.cout) ((uint16_t*)p)[i] = (uint16_t)(h[i / 2] >> (16 * (i % 2)));
    }
    return;
  }
  uint32_t amax[2] = {0u, 0u}, c[4], byte[2];
#pragma unroll
  for (int i = 0; i < 32; ++i) amax[i / 16] = max(amax[i / 16], __float_as_uint(y[i]) & 0x7fffffffu);
  const bool mx = o.mode == 1;
  if (mx) amax[0] = amax[1] = max(amax[0], amax[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float s;
    byte[h] = mx ? scale_mx(amax[h], s) : scale_nv(amax[h], o.ts, s);
    codes_of<16>(mx, y + 16 * h, s, amax[h], c + 2 * h);
  }
  *(uint4*)(o.out + row * o.cpitch + col / 2u) = make_uint4(c[0], c[1], c[2], c[3]);
  uint8_t* so = o.out_scales + row * o.spitch;
  if (mx) {
    so[col / 32u] = (uint8_t)byte[0];
    // the bytes behind the last block of rows of an odd number of 64 channels
    if (col / 2u + 16u == o.cpitch && (o.cpitch & 32u)) so[col / 32u + 1u] = so[col / 32u + 2u] = 0;
  } else {
    *(uint16_t*)(so + col / 16u) = (uint16_t)(byte[0] | byte[1] << 8);
  }
}

// Host: the output's part of a call's parameters; false where they are not valid.
inline bool make_output(const spconvb_fp4_params& p, const float* bias, void* out, Output& o) {
  if (p.act != SPCONVB_ACT_NONE && p.act != SPCONVB_ACT_RELU) return false;
  if (p.out_fp4 && (!p.out_scales || !format_ok(p.out_format) || !tensor_scale_ok(p.out_format, p.out_tensor_scale)))
    return false;
  if ((uintptr_t)out & (p.out_fp4 ? 15u : 1u) || (p.out_fp4 && (uintptr_t)p.out_scales & 15u) || (uintptr_t)bias & 3u ||
      (uintptr_t)p.res & 1u)
    return false;
  o = Output{};
  o.bias = bias;
  o.res = (const __half*)p.res;
  o.out = (uint8_t*)out;
  o.out_scales = (uint8_t*)p.out_scales;
  o.cout = (uint32_t)p.cout;
  o.alpha = p.alpha;
  o.act = p.act;
  o.res_relu = p.res_relu;
  if (p.out_fp4) {
    o.mode = p.out_format == SPCONVB_MXFP4 ? 1 : 2;
    o.ts = tensor_scale_of(p.out_tensor_scale);
    o.cpitch = code_pitch(o.cout);
    o.spitch = scale_pitch(p.out_format, o.cout);
  }
  const uint64_t bits = (uint64_t)(uintptr_t)p.res | 2ull * o.cout | (p.out_fp4 ? 0ull : (uint64_t)(uintptr_t)out);
  o.access = bits % 32u == 0u ? 32 : (bits % 16u == 0u ? 16 : 2);
  return true;
}

}  // namespace fp4
}  // namespace spconvb
