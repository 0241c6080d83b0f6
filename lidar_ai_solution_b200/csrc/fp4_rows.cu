// Rows to 4-bit codes with block scales and back, and the layout of quantised weights for the products.
//
// All three only move bytes.  A thread owns a unit of 16 channels: 32 bytes of fp16 in one load, 8 bytes of codes in one store, so
// a warp reads and writes contiguous kilobytes; the scale of an MXFP4 block belongs to two neighbouring lanes, which
// exchange their largest magnitudes.  Rows go one of three ways:
//   flat     no padding of channels (NVFP4: a multiple of 64; MXFP4: of 128, or 64) and 32-byte alignment: units, codes and
//            scales are one sequence each
//   aligned  rows that start on 16 bytes: a unit is found by its row, 16 bytes at a time
//   staged   all others: 256 units in a row are one contiguous piece of the fp16 / fp32 / int8 side, which passes through
//            shared memory in 16-byte pieces
//
// Measured: 480 000 x 128 fp16 -> NVFP4 25.4 us (6.2 TB/s, 96 % of a copy's rate), 120 000 x 128 -> MXFP4 5.5 us (out of L2); 960 000 x 64
// int8 -> NVFP4 21.7 us (4.4 TB/s; two thirds of the issue slots and of the integer pipe, whatever the occupancy, so that neither is
// the limit by itself); back to fp16 25.8 us
// (6.1 TB/s); 200 000 rows of 100 channels, staged, 20.6 us and back 15.4.  A grid of 32 blocks an SM: with 16, a block had one turn or
// two, and the last ones ran alone (back to fp16 27.5; with 6 33.5, with as many as there are turns 25.8).
#include "fp4.cuh"
#include "pdl.cuh"

namespace spconvb {
namespace fp4 {
namespace {

constexpr int kThreads = 256;
enum Way { kFlat, kAligned, kStaged };
// Units whose loads a thread keeps in flight on the flat way (int8 units are half as long); on the others one: with two, rows of 72
// channels took 4.2 us and not 3.8, for what they have to compute before the load.
template <int KIND, Way WAY>
constexpr int kAhead = WAY == kFlat ? (KIND == SPCONVB_I8 ? 4 : 2) : 1;

struct Rows {
  uint32_t channels, upr;  // units of 16 channels a row, padding included
  uint64_t upr_inv;        // ceil(2^64 / upr): u / upr = hi64(u * upr_inv) for u < 2^48, upr <= 4096
  uint32_t cpitch, spitch;
  Way way;
};

// Row and unit in the row of unit u.
__device__ __forceinline__ void place(const Rows& g, uint64_t u, uint64_t& row, uint32_t& ub) {
  row = __umul64hi(u, g.upr_inv);
  ub = (uint32_t)(u - row * g.upr);
}
// Channels of a unit that exist, and its first element counted from the first row's.
__device__ __forceinline__ uint32_t present(const Rows& g, uint32_t ub) {
  return ub * 16u < g.channels ? min(16u, g.channels - ub * 16u) : 0u;
}
__device__ __forceinline__ uint64_t element_at(const Rows& g, uint64_t row, uint32_t ub) {
  return row * g.channels + min(ub * 16u, g.channels);
}

template <int KIND>
__device__ __forceinline__ constexpr uint32_t elem_size() {
  return KIND == SPCONVB_F32 ? 4u : (KIND == SPCONVB_I8 ? 1u : 2u);
}

// The 16 elements of a unit as they lie in memory (channels behind the last one: zero).
template <int KIND>
struct Raw {
  static constexpr int kWords = 4 * elem_size<KIND>();
  uint32_t w[kWords];
};
template <int KIND>
__device__ __forceinline__ void load_flat(const uint8_t* p, Raw<KIND>& raw) {
  if (KIND == SPCONVB_I8) {
    const uint4 v = ld16(p);
    raw.w[0] = v.x;
    raw.w[1] = v.y;
    raw.w[2] = v.z;
    raw.w[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < Raw<KIND>::kWords / 8; ++i) ld32(p + 32 * i, raw.w + 8 * i);
  }
}
template <int KIND>
__device__ __forceinline__ void load_aligned(const uint8_t* p, uint32_t left, Raw<KIND>& raw) {
#pragma unroll
  for (int i = 0; i < (int)elem_size<KIND>(); ++i) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if ((int)left > i * 16 / (int)elem_size<KIND>()) v = ld16(p + 16 * i);
    raw.w[4 * i] = v.x;
    raw.w[4 * i + 1] = v.y;
    raw.w[4 * i + 2] = v.z;
    raw.w[4 * i + 3] = v.w;
  }
}
// From `at` bytes into shared memory on: whole words, moved into place, and what does not exist cut off.
template <int KIND>
__device__ __forceinline__ void load_staged(const uint32_t* buf, uint32_t at, uint32_t left, Raw<KIND>& raw) {
  const uint32_t sh = (at & 3u) * 8u;
  const uint32_t* p = buf + (at >> 2);
  uint32_t w[Raw<KIND>::kWords + 1];
#pragma unroll
  for (int i = 0; i <= Raw<KIND>::kWords; ++i) w[i] = p[i];
  const uint32_t bytes = left * elem_size<KIND>();
#pragma unroll
  for (int i = 0; i < Raw<KIND>::kWords; ++i) {
    const uint32_t v = __funnelshift_r(w[i], w[i + 1], sh);
    raw.w[i] = bytes >= 4u * i + 4u ? v : (bytes <= 4u * i ? 0u : v & ((1u << (8u * (bytes - 4u * i))) - 1u));
  }
}

// Elements to fp32, and the bits of the largest magnitude (infinities and NaN are the largest).
template <int KIND>
__device__ __forceinline__ uint32_t elements(const Raw<KIND>& raw, float in_scale, float (&x)[16]) {
  if (KIND == SPCONVB_F32) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      x[i] = __uint_as_float(raw.w[i]);
      x[i + 1] = __uint_as_float(raw.w[i + 1]);
      m = max_abs_nan(m, x[i], x[i + 1]);
    }
    return __float_as_uint(m);
  }
  if (KIND == SPCONVB_F16) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __half22float2(*(const __half2*)&raw.w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
      m = __vmaxu2(m, raw.w[i] & 0x7fff7fffu);
    }
    m = max(m & 0xffffu, m >> 16);
    return __float_as_uint(__half2float(__ushort_as_half((uint16_t)m)));
  }
  // int8: byte b goes into the mantissa of 2^23 + (b + 128); a conversion instruction has an eighth of the rate
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const uint32_t w = raw.w[i / 4] ^ 0x80808080u;
    const F2 b(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650u | (uint32_t)(i % 4))),
               __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650u | (uint32_t)(i % 4 + 1))));
    mul2(add2(b, F2(-8388736.f, -8388736.f)), F2(in_scale, in_scale)).get(x[i], x[i + 1]);
    m = max_abs(m, x[i], x[i + 1]);
  }
  return __float_as_uint(m);
}

template <int FMT, int KIND, Way WAY>
__device__ __forceinline__ void store_unit(const Rows& g, uint64_t u, uint64_t row, uint32_t ub, const Raw<KIND>& raw,
                                           float in_scale, const TensorScale& ts, uint8_t* codes, uint8_t* scales, bool live) {
  float x[16];
  uint32_t amax = elements<KIND>(raw, in_scale, x);
  if (FMT == SPCONVB_MXFP4) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  float s;
  uint32_t byte = FMT == SPCONVB_MXFP4 ? scale_mx(amax, s) : scale_nv(amax, ts, s);
  const bool word = FMT == SPCONVB_MXFP4 && WAY == kFlat && g.upr == 4u;  // rows of 64 channels: two scales, two bytes of padding
  if (word) byte |= __shfl_down_sync(0xffffffffu, byte, 2) << 8;
  if (!live) return;
  uint32_t c[2];
  codes_of<16>(FMT == SPCONVB_MXFP4, x, s, amax, c);
  uint8_t* co = WAY == kFlat ? codes + u * 8u : codes + row * g.cpitch + ub * 8u;
  *(uint2*)co = make_uint2(c[0], c[1]);
  if (FMT == SPCONVB_NVFP4) {
    scales[WAY == kFlat ? u : row * g.spitch + ub] = (uint8_t)byte;
  } else if (word) {
    if (!(u & 3u)) *(uint32_t*)(scales + u) = byte;
  } else if (!(ub & 1u)) {
    uint8_t* so = WAY == kFlat ? scales + (u >> 1) : scales + row * g.spitch + (ub >> 1);
    *so = (uint8_t)byte;
    // the two bytes behind the last block of rows of an odd number of 64 channels
    if (WAY != kFlat && (g.upr & 4u) && ub + 2u == g.upr) so[1] = so[2] = 0;
  }
}

// Place of unit u's scale on the flat way.
template <int FMT>
__device__ __forceinline__ uint64_t flat_scale(const Rows& g, uint64_t u) {
  if (FMT == SPCONVB_NVFP4) return u;
  return g.upr == 4u ? (u & ~3ull) + (u >> 1 & 1u) : u >> 1;
}

// The contiguous piece of rows that units [u0, u1) cover: first element, and one past the last.
__device__ __forceinline__ void piece_of(const Rows& g, uint64_t u0, uint64_t u1, uint64_t& e0, uint64_t& e1) {
  uint64_t row;
  uint32_t ub;
  place(g, u0, row, ub);
  e0 = element_at(g, row, ub);
  place(g, u1 - 1u, row, ub);
  e1 = element_at(g, row, ub) + present(g, ub);
}

template <int FMT, int KIND, Way WAY>
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(const uint8_t* __restrict__ x, const Rows g, float in_scale,
                                                                const TensorScale ts, const uint32_t* n_ptr, uint32_t cap,
                                                                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr uint32_t es = elem_size<KIND>();
  __shared__ uint4 buf[WAY == kStaged ? kThreads * es + 2 : 1];  // 16 bytes of slack at either end
  pdl_wait_and_trigger();
  const uint64_t units = (uint64_t)min(load_in_order(n_ptr), cap) * g.upr;
  // loops go by the block: the lanes of a warp exchange magnitudes
  if (WAY != kStaged) {
    constexpr int A = kAhead<KIND, WAY>;
    for (uint64_t u0 = (uint64_t)blockIdx.x * (kThreads * A); u0 < units; u0 += (uint64_t)gridDim.x * (kThreads * A)) {
      Raw<KIND> raw[A];
      if (WAY == kFlat && u0 + kThreads * A <= units) {  // all of the block's units are there: nothing to ask (int8 -> NVFP4 23.7 -> 21.7 us)
        const uint64_t u = u0 + threadIdx.x;
#pragma unroll
        for (int i = 0; i < A; ++i) load_flat<KIND>(x + (u + i * kThreads) * (16u * es), raw[i]);
#pragma unroll
        for (int i = 0; i < A; ++i)
          store_unit<FMT, KIND, WAY>(g, u + i * kThreads, 0, (uint32_t)u & 1u, raw[i], in_scale, ts, codes, scales, true);
        continue;
      }
#pragma unroll
      for (int i = 0; i < A; ++i) {
        const uint64_t u = u0 + i * kThreads + threadIdx.x;
#pragma unroll
        for (int j = 0; j < Raw<KIND>::kWords; ++j) raw[i].w[j] = 0u;
        if (u < units) {
          if (WAY == kFlat) {
            load_flat<KIND>(x + u * (16u * es), raw[i]);
          } else {
            uint64_t row;
            uint32_t ub;
            place(g, u, row, ub);
            load_aligned<KIND>(x + element_at(g, row, ub) * es, present(g, ub), raw[i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < A; ++i) {
        const uint64_t u = u0 + i * kThreads + threadIdx.x;
        uint64_t row = 0;
        uint32_t ub = (uint32_t)u & 1u;
        if (WAY == kAligned) place(g, u, row, ub);
        store_unit<FMT, KIND, WAY>(g, u, row, ub, raw[i], in_scale, ts, codes, scales, u < units);
      }
    }
  } else {
    for (uint64_t u0 = (uint64_t)blockIdx.x * kThreads; u0 < units; u0 += (uint64_t)gridDim.x * kThreads) {
      const uint64_t u = u0 + threadIdx.x;
      const bool live = u < units;
      uint64_t row = 0, e0, e1;
      uint32_t ub = 0;
      if (live) place(g, u, row, ub);
      const uint32_t left = live ? present(g, ub) : 0u;
      piece_of(g, u0, min(u0 + kThreads, units), e0, e1);
      // 16-byte pieces from the last boundary before e0 on; at the ends only what lies inside
      const uint64_t a0 = (uint64_t)(uintptr_t)x + e0 * es, a1 = (uint64_t)(uintptr_t)x + e1 * es, from = a0 & ~15ull;
      __syncthreads();  // the units before are read
      for (uint64_t p = from + threadIdx.x * 16u; p < a1; p += kThreads * 16u) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (p >= a0 && p + 16u <= a1) {
          v = ld16((const void*)(uintptr_t)p);
        } else {
          uint8_t* b = (uint8_t*)&v;
#pragma unroll
          for (uint32_t i = 0; i < 16u; i += es) {
            if (p + i >= a0 && p + i < a1) {
              if (es == 1u) b[i] = *(const volatile uint8_t*)(uintptr_t)(p + i);
              else if (es == 2u) *(uint16_t*)(b + i) = *(const volatile uint16_t*)(uintptr_t)(p + i);
              else *(uint32_t*)(b + i) = *(const volatile uint32_t*)(uintptr_t)(p + i);
            }
          }
        }
        buf[(p - from) >> 4] = v;
      }
      __syncthreads();
      Raw<KIND> raw;
#pragma unroll
      for (int j = 0; j < Raw<KIND>::kWords; ++j) raw.w[j] = 0u;
      if (left)
        load_staged<KIND>((const uint32_t*)buf, (uint32_t)((uint64_t)(uintptr_t)x + element_at(g, row, ub) * es - from), left,
                          raw);
      store_unit<FMT, KIND, WAY>(g, u, row, ub, raw, in_scale, ts, codes, scales, live);
    }
  }
}

// What a unit's codes stand for, as it lies in memory.
template <int FMT, int KIND>
__device__ __forceinline__ void values_of(uint2 c, uint32_t byte, float tensor_scale, Raw<KIND>& v) {
  const float s = scale_value(FMT, byte, tensor_scale);
  uint32_t h[2][4];
  values8(c.x, h[0]);
  values8(c.y, h[1]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __half22float2(*(const __half2*)&h[i / 4][i % 4]);
    float a, b;
    mul2(F2(f.x, f.y), F2(s, s)).get(a, b);
    if (KIND == SPCONVB_F16) {
      const __half2 p = __floats2half2_rn(a, b);
      v.w[i] = *(const uint32_t*)&p;
    } else {
      v.w[2 * i] = __float_as_uint(a);
      v.w[2 * i + 1] = __float_as_uint(b);
    }
  }
}

template <int FMT, int KIND, Way WAY>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                  const Rows g, float tensor_scale, const uint32_t* n_ptr,
                                                                  uint32_t cap, uint8_t* __restrict__ out) {
  constexpr uint32_t es = elem_size<KIND>();
  __shared__ uint4 buf[WAY == kStaged ? kThreads * es + 2 : 1];
  pdl_wait_and_trigger();
  const uint64_t units = (uint64_t)min(load_in_order(n_ptr), cap) * g.upr;
  if (WAY != kStaged) {
    constexpr int A = kAhead<KIND, WAY>;
    for (uint64_t u0 = (uint64_t)blockIdx.x * (kThreads * A); u0 < units; u0 += (uint64_t)gridDim.x * (kThreads * A)) {
      uint2 c[A];
      uint32_t byte[A], left[A];
      uint8_t* o[A];
#pragma unroll
      for (int i = 0; i < A; ++i) {
        const uint64_t u = u0 + i * kThreads + threadIdx.x;
        left[i] = 0u;
        if (u < units) {
          if (WAY == kFlat) {
            left[i] = 16u;
            c[i] = ld8(codes + u * 8u);
            byte[i] = (uint32_t)load_in_order((const int8_t*)scales + flat_scale<FMT>(g, u)) & 255u;
            o[i] = out + u * (16u * es);
          } else {
            uint64_t row;
            uint32_t ub;
            place(g, u, row, ub);
            left[i] = present(g, ub);
            if (left[i]) {
              c[i] = ld8(codes + row * g.cpitch + ub * 8u);
              byte[i] = (uint32_t)load_in_order((const int8_t*)scales + row * g.spitch +
                                                (FMT == SPCONVB_MXFP4 ? ub >> 1 : ub)) & 255u;
            }
            o[i] = out + element_at(g, row, ub) * es;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < A; ++i) {
        if (left[i] == 0u) continue;
        Raw<KIND> v;
        values_of<FMT, KIND>(c[i], byte[i], tensor_scale, v);
        if (WAY == kFlat) {
#pragma unroll
          for (int j = 0; j < Raw<KIND>::kWords / 8; ++j) st32(o[i] + 32 * j, v.w + 8 * j);
        } else {
#pragma unroll
          for (int j = 0; j < (int)es; ++j)
            if ((int)left[i] > j * 16 / (int)es)
              ((uint4*)o[i])[j] = make_uint4(v.w[4 * j], v.w[4 * j + 1], v.w[4 * j + 2], v.w[4 * j + 3]);
        }
      }
    }
  } else {
    for (uint64_t u0 = (uint64_t)blockIdx.x * kThreads; u0 < units; u0 += (uint64_t)gridDim.x * kThreads) {
      const uint64_t u = u0 + threadIdx.x;
      uint64_t row = 0;
      uint32_t ub = 0, left = 0;
      if (u < units) {
        place(g, u, row, ub);
        left = present(g, ub);
      }
      Raw<KIND> v;
      if (left) {
        const uint2 c = ld8(codes + row * g.cpitch + ub * 8u);
        const uint32_t byte =
            (uint32_t)load_in_order((const int8_t*)scales + row * g.spitch + (FMT == SPCONVB_MXFP4 ? ub >> 1 : ub)) & 255u;
        values_of<FMT, KIND>(c, byte, tensor_scale, v);
      }
      uint8_t* o = out + element_at(g, row, ub) * es;
      uint64_t e0, e1;
      piece_of(g, u0, min(u0 + kThreads, units), e0, e1);
      const uint64_t a0 = (uint64_t)(uintptr_t)out + e0 * es, a1 = (uint64_t)(uintptr_t)out + e1 * es, from = a0 & ~15ull;
      uint8_t* b = (uint8_t*)buf + ((uint64_t)(uintptr_t)o - from);
      __syncthreads();  // the units before are written
      if (es == 4u) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < (int)left) ((uint32_t*)b)[i] = v.w[i % Raw<KIND>::kWords];
      } else if (((uint64_t)(uintptr_t)b & 3u) == 0u) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (2 * i + 1 < (int)left) ((uint32_t*)b)[i] = v.w[i];
          else if (2 * i < (int)left) ((uint16_t*)b)[2 * i] = (uint16_t)v.w[i];
        }
      } else {
        // from the odd half on: one half, pairs across the words, one half
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i == 0 && left) *(uint16_t*)b = (uint16_t)v.w[0];
          const uint32_t pair = __funnelshift_r(v.w[i], i < 7 ? v.w[i < 7 ? i + 1 : 7] : 0u, 16);
          if (2 * i + 2 < (int)left) *(uint32_t*)(b + 4 * i + 2) = pair;
          else if (2 * i + 1 < (int)left) *(uint16_t*)(b + 4 * i + 2) = (uint16_t)pair;
        }
      }
      __syncthreads();
      for (uint64_t p = from + threadIdx.x * 16u; p < a1; p += kThreads * 16u) {
        const uint4* src = buf + ((p - from) >> 4);
        if (p >= a0 && p + 16u <= a1) {
          *(uint4*)(uintptr_t)p = *src;
        } else {
#pragma unroll
          for (uint32_t i = 0; i < 16u; i += es) {
            if (p + i >= a0 && p + i < a1) {
              if (es == 2u) *(uint16_t*)(uintptr_t)(p + i) = ((const uint16_t*)src)[i / 2u];
              else *(uint32_t*)(uintptr_t)(p + i) = ((const uint32_t*)src)[i / 4u];
            }
          }
        }
      }
    }
  }
}

Rows rows_of(int format, int channels, const void* p, uint32_t es) {
  Rows g;
  g.channels = (uint32_t)channels;
  g.upr = cpad(g.channels) / 16u;
  g.upr_inv = ~0ull / g.upr + 1ull;  // upr is at least 4
  g.cpitch = code_pitch(g.channels);
  g.spitch = scale_pitch(format, g.channels);
  const uint64_t row = (uint64_t)g.channels * es;
  if (((uint64_t)(uintptr_t)p | row) % 16u != 0u) g.way = kStaged;
  else if ((g.channels == 64u || g.channels % (format == SPCONVB_MXFP4 ? 128u : 64u) == 0u) && (uintptr_t)p % 32u == 0u)
    g.way = kFlat;
  else g.way = kAligned;
  return g;
}
template <int KIND>
int blocks_of(const Rows& g, uint32_t rows) {
  const uint64_t per = kThreads * (g.way == kFlat ? kAhead<KIND, kFlat> : 1), b = ((uint64_t)rows * g.upr + per - 1) / per;
  return (int)(b < (uint64_t)kSmCount * 32 ? b : (uint64_t)kSmCount * 32);
}

// One thread a 16-byte segment of the image or a word of scales.
__global__ void fp4_pack_kernel(int format, uint32_t cin, uint32_t cout, uint32_t kvol, const uint8_t* __restrict__ codes,
                                const uint8_t* __restrict__ scales, uint8_t* __restrict__ out, uint64_t total) {
  const uint32_t cp = cpad(cin), cpitch = cp / 2u, spitch = scale_pitch(format, cin);
  const uint32_t words = words_per_chunk(format, cp);
  const uint64_t ktotal = (uint64_t)kvol * cp;
  const uint32_t nchunk = (uint32_t)((ktotal + kChunkK - 1) / kChunkK);
  const uint32_t per_chunk = 128u * 8u + words * 128u;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t rec = i / per_chunk;  // (block of 128 channels, chunk)
    uint32_t t = (uint32_t)(i % per_chunk);
    const uint32_t blk = (uint32_t)(rec / nchunk), j = (uint32_t)(rec % nchunk);
    uint8_t* dst = out + rec * (128u * 128u + (uint64_t)words * kAtomBytes);
    const bool code = t < 1024u;
    uint32_t r, w = 0, seg = 0;
    if (code) {
      r = t / 8u;
      seg = t % 8u;
    } else {
      t -= 1024u;
      w = t / 128u;
      r = t % 128u;
    }
    const uint32_t ch = blk * 128u + r;
    const uint64_t k = (uint64_t)j * kChunkK + (code ? seg * 32u : w * (kChunkK / words));
    const bool live = ch < cout && k < ktotal;
    const uint32_t tap = live ? (uint32_t)(k / cp) : 0u, c = live ? (uint32_t)(k % cp) : 0u;
    const uint64_t row = (uint64_t)ch * kvol + tap;
    if (code) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (live) v = *(const uint4*)(codes + row * cpitch + c / 2u);
      *(uint4*)(dst + (r / 8u) * 1024u + (r % 8u) * 128u + ((seg ^ (r % 8u)) << 4)) = v;
    } else {
      uint32_t v = 0u;
      if (live) v = *(const uint32_t*)(scales + row * spitch + (format == SPCONVB_MXFP4 ? c / 128u : c / 64u) * 4u);
      *(uint32_t*)(dst + 128u * 128u + w * kAtomBytes + (r % 32u) * 16u + (r / 32u) * 4u) = v;
    }
  }
}

struct Call {
  cudaStream_t st;
  Rows g;
  float in_scale, tensor_scale;
  const uint32_t* n;
  uint32_t cap;
};
template <int FMT, int KIND>
cudaError_t quantize_way(const Call& k, const uint8_t* x, uint8_t* codes, uint8_t* scales) {
  const dim3 b(blocks_of<KIND>(k.g, k.cap)), t(kThreads);
  if (k.g.way == kFlat)
    return launch_pdl(fp4_quantize_kernel<FMT, KIND, kFlat>, b, t, 0, k.st, x, k.g, k.in_scale, tensor_scale_of(k.tensor_scale), k.n, k.cap,
                      codes, scales);
  if (k.g.way == kAligned)
    return launch_pdl(fp4_quantize_kernel<FMT, KIND, kAligned>, b, t, 0, k.st, x, k.g, k.in_scale, tensor_scale_of(k.tensor_scale), k.n, k.cap,
                      codes, scales);
  return launch_pdl(fp4_quantize_kernel<FMT, KIND, kStaged>, b, t, 0, k.st, x, k.g, k.in_scale, tensor_scale_of(k.tensor_scale), k.n, k.cap, codes,
                    scales);
}
template <int FMT>
cudaError_t quantize_kind(int kind, const Call& k, const uint8_t* x, uint8_t* codes, uint8_t* scales) {
  if (kind == SPCONVB_F16) return quantize_way<FMT, SPCONVB_F16>(k, x, codes, scales);
  return kind == SPCONVB_F32 ? quantize_way<FMT, SPCONVB_F32>(k, x, codes, scales)
                             : quantize_way<FMT, SPCONVB_I8>(k, x, codes, scales);
}
template <int FMT, int KIND>
cudaError_t dequantize_way(const Call& k, const uint8_t* codes, const uint8_t* scales, uint8_t* out) {
  const dim3 b(blocks_of<KIND>(k.g, k.cap)), t(kThreads);
  if (k.g.way == kFlat)
    return launch_pdl(fp4_dequantize_kernel<FMT, KIND, kFlat>, b, t, 0, k.st, codes, scales, k.g, k.tensor_scale, k.n, k.cap, out);
  if (k.g.way == kAligned)
    return launch_pdl(fp4_dequantize_kernel<FMT, KIND, kAligned>, b, t, 0, k.st, codes, scales, k.g, k.tensor_scale, k.n, k.cap,
                      out);
  return launch_pdl(fp4_dequantize_kernel<FMT, KIND, kStaged>, b, t, 0, k.st, codes, scales, k.g, k.tensor_scale, k.n, k.cap, out);
}

template <int FMT>
cudaError_t dequantize_kind(int kind, const Call& k, const uint8_t* codes, const uint8_t* scales, uint8_t* out) {
  return kind == SPCONVB_F16 ? dequantize_way<FMT, SPCONVB_F16>(k, codes, scales, out)
                             : dequantize_way<FMT, SPCONVB_F32>(k, codes, scales, out);
}

bool aligned16(const void* a, const void* b = nullptr, const void* c = nullptr) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15u) == 0u;
}

}  // namespace

// Chunks of an image of packed weights, over all blocks of 128 channels; 0 for numbers that no image has.
uint64_t packed_records(int cin, int cout, int kvol) {
  if (!channels_ok(cin) || !channels_ok(cout) || kvol < 1 || kvol > 27) return 0;
  const uint64_t nchunk = ((uint64_t)kvol * cpad(cin) + kChunkK - 1) / kChunkK;
  return nchunk * (((uint64_t)cout + 127u) / 128u);
}

}  // namespace fp4
}  // namespace spconvb

using namespace spconvb;
using namespace spconvb::fp4;

extern "C" {

uint32_t spconvb_fp4_code_pitch(int32_t channels) {
  return channels_ok(channels) ? code_pitch((uint32_t)channels) : 0u;
}
uint32_t spconvb_fp4_scale_pitch(int32_t format, int32_t channels) {
  return channels_ok(channels) && format_ok(format) ? scale_pitch(format, (uint32_t)channels) : 0u;
}

int spconvb_fp4_quantize(int32_t format, const void* x, int32_t kind, float in_scale, int32_t channels, float tensor_scale,
                         const uint32_t* n_ptr, uint32_t launch_rows, void* codes, void* scales, void* stream) {
  if (!x || !codes || !scales || !n_ptr || launch_rows < 1 || !format_ok(format) || !channels_ok(channels) ||
      !tensor_scale_ok(format, tensor_scale))
    return SPCONVB_E_ARG;
  if (kind != SPCONVB_F16 && kind != SPCONVB_F32 && kind != SPCONVB_I8) return SPCONVB_E_ARG;
  const uint32_t es = kind == SPCONVB_F32 ? 4u : (kind == SPCONVB_I8 ? 1u : 2u);
  if (!aligned16(codes, scales) || (uintptr_t)x % es != 0u) return SPCONVB_E_ARG;
  if (kind == SPCONVB_I8 && !(in_scale > -3.4e38f && in_scale < 3.4e38f)) return SPCONVB_E_ARG;
  const Rows g = rows_of(format, channels, x, es);
  const Call k{(cudaStream_t)stream, g, in_scale, tensor_scale, n_ptr, launch_rows};
  SPCONVB_CUDA_TRY(format == SPCONVB_MXFP4
                       ? quantize_kind<SPCONVB_MXFP4>(kind, k, (const uint8_t*)x, (uint8_t*)codes, (uint8_t*)scales)
                       : quantize_kind<SPCONVB_NVFP4>(kind, k, (const uint8_t*)x, (uint8_t*)codes, (uint8_t*)scales));
  return SPCONVB_OK;
}

int spconvb_fp4_dequantize(int32_t format, const void* codes, const void* scales, int32_t channels, float tensor_scale,
                           int32_t out_kind, const uint32_t* n_ptr, uint32_t launch_rows, void* out, void* stream) {
  if (!codes || !scales || !n_ptr || !out || launch_rows < 1 || !format_ok(format) || !channels_ok(channels) ||
      !tensor_scale_ok(format, tensor_scale))
    return SPCONVB_E_ARG;
  if (out_kind != SPCONVB_F16 && out_kind != SPCONVB_F32) return SPCONVB_E_ARG;
  const uint32_t es = out_kind == SPCONVB_F32 ? 4u : 2u;
  if (!aligned16(codes, scales) || (uintptr_t)out % es != 0u) return SPCONVB_E_ARG;
  const Rows g = rows_of(format, channels, out, es);
  const Call k{(cudaStream_t)stream, g, 1.f, tensor_scale, n_ptr, launch_rows};
  const uint8_t *c = (const uint8_t*)codes, *s = (const uint8_t*)scales;
  SPCONVB_CUDA_TRY(format == SPCONVB_MXFP4 ? dequantize_kind<SPCONVB_MXFP4>(out_kind, k, c, s, (uint8_t*)out)
                                           : dequantize_kind<SPCONVB_NVFP4>(out_kind, k, c, s, (uint8_t*)out));
  return SPCONVB_OK;
}

size_t spconvb_fp4_packed_bytes(int32_t format, int32_t cin, int32_t cout, int32_t kvol) {
  if (!format_ok(format)) return 0;
  return packed_records(cin, cout, kvol) *
         (128u * 128u + (size_t)words_per_chunk(format, cpad((uint32_t)cin)) * kAtomBytes);
}

int spconvb_fp4_pack_weights(int32_t format, int32_t cin, int32_t cout, int32_t kvol, const void* codes, const void* scales,
                             void* packed, void* stream) {
  if (!codes || !scales || !packed || !format_ok(format)) return SPCONVB_E_ARG;
  const uint64_t records = packed_records(cin, cout, kvol);
  if (records == 0 || !aligned16(codes, scales, packed)) return SPCONVB_E_ARG;
  // What no product takes is refused here and not at the first product.  (With more than one tap an image also wants a whole number of scale
  // words a tap, which MXFP4 rows of 129 to 192 channels do not have.)
  if (kvol > 1 && !spconvb_fp4_conv_supported(cin, cout, kvol)) return SPCONVB_E_UNSUPPORTED;
  const uint64_t total = records * (1024u + words_per_chunk(format, cpad((uint32_t)cin)) * 128u);
  const uint64_t blocks = (total + 255u) / 256u;
  fp4_pack_kernel<<<(int)(blocks < kSmCount * 32u ? blocks : kSmCount * 32u), 256, 0, (cudaStream_t)stream>>>(
      format, (uint32_t)cin, (uint32_t)cout, (uint32_t)kvol, (const uint8_t*)codes, (const uint8_t*)scales,
      (uint8_t*)packed, total);
  SPCONVB_LAUNCH_CHECK();
  return SPCONVB_OK;
}

}  // extern "C"
