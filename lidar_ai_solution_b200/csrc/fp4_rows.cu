// Rows to 4-bit codes with block scales and back, and the layout of quantised weights for the products.
//
// All three only move bytes.  A thread owns a unit of 16 channels: 32 bytes of fp16 in one load, 8 bytes of codes in one store, so
// a warp reads and writes contiguous kilobytes; the scale of an MXFP4 block belongs to two neighbouring lanes, which
// exchange their largest magnitudes.
#include "fp4.cuh"
#include "pdl.cuh"

namespace spconvb {
namespace fp4 {
namespace {

constexpr int kThreads = 256;

struct Rows {
  uint32_t channels, upr;  // units of 16 channels a row, padding included
  uint64_t upr_inv;        // ceil(2^64 / upr): u / upr = hi64(u * upr_inv) for u < 2^48, upr <= 4096
  uint32_t cpitch, spitch;
  int flat;                // no padding anywhere: units, codes and scales are one sequence
  int aligned;             // of a row's first element: 32, 16, or 0 (that of the element)
};

// Row and unit in the row of unit u.
__device__ __forceinline__ void place(const Rows& g, uint64_t u, uint64_t& row, uint32_t& ub) {
  row = __umul64hi(u, g.upr_inv);
  ub = (uint32_t)(u - row * g.upr);
}

__device__ __forceinline__ void ld32(const void* p, uint32_t (&v)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void st32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "l"(p)
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

template <int KIND>
__device__ __forceinline__ constexpr uint32_t elem_size() {
  return KIND == SPCONVB_F32 ? 4u : (KIND == SPCONVB_I8 ? 1u : 2u);
}

// The 16 elements of a unit as they lie in memory (channels behind the last one: zero).
template <int KIND>
struct Raw {
  uint32_t w[4 * elem_size<KIND>()];
};
template <int KIND>
__device__ __forceinline__ void load_raw(const Rows& g, const uint8_t* x, uint64_t row, uint32_t ub,
                                         Raw<KIND>& raw) {
  constexpr uint32_t es = elem_size<KIND>();
  const uint8_t* p = x + (row * g.channels + ub * 16u) * es;
  const uint32_t c0 = ub * 16u;
  const uint32_t left = c0 < g.channels ? min(16u, g.channels - c0) : 0u;
  if (left == 16u && g.aligned == 32 && es >= 2u) {
#pragma unroll
    for (int i = 0; i < (int)(es / 2u); ++i) {
      uint32_t v[8];
      ld32(p + 32 * i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) raw.w[8 * i + j] = v[j];
    }
  } else if (g.aligned != 0) {
    // whole 16-byte pieces: rows that start on one end on one
#pragma unroll
    for (uint32_t i = 0; i < es; ++i) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (i * (16u / es) < left) v = ld16(p + 16u * i);
      raw.w[4u * i] = v.x;
      raw.w[4u * i + 1u] = v.y;
      raw.w[4u * i + 2u] = v.z;
      raw.w[4u * i + 3u] = v.w;
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4u * es; ++i) raw.w[i] = 0u;
#pragma unroll
    for (uint32_t i = 0; i < 16u; ++i) {
      if (i < left) {
        if (KIND == SPCONVB_F32) raw.w[i] = load_in_order((const uint32_t*)p + i);
        else if (KIND == SPCONVB_F16)
          raw.w[i / 2u] |= (uint32_t)load_in_order((const uint16_t*)p + i) << (16u * (i % 2u));
        else
          raw.w[i / 4u] |= ((uint32_t)load_in_order((const int8_t*)p + i) & 255u) << (8u * (i % 4u));
      }
    }
  }
}
template <int KIND>
__device__ __forceinline__ float element(const Raw<KIND>& raw, int i, float in_scale) {
  if (KIND == SPCONVB_F32) return __uint_as_float(raw.w[i]);
  if (KIND == SPCONVB_F16)
    return __half2float(__ushort_as_half((uint16_t)(raw.w[i / 2] >> (16 * (i % 2)))));
  return __fmul_rn((float)(int8_t)(raw.w[i / 4] >> (8 * (i % 4))), in_scale);
}

template <int FMT, int KIND>
__device__ __forceinline__ void store_unit(const Rows& g, uint64_t row, uint32_t ub, uint64_t u, const Raw<KIND>& raw,
                                           float in_scale, float tensor_scale, uint8_t* codes,
                                           uint8_t* scales, bool live) {
  float x[16];
  uint32_t amax = 0u;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = element<KIND>(raw, i, in_scale);
    amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
  }
  if (FMT == SPCONVB_MXFP4) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  if (!live) return;
  float s;
  const uint32_t byte = FMT == SPCONVB_MXFP4 ? scale_mx(amax, s) : scale_nv(amax, tensor_scale, s);
  const bool none = amax >= 0x7f800000u || s == 0.f;
  const Divider d = divider(FMT, s, amax);
  uint32_t c[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = divide(d, x[8 * h + i]);
    c[h] = none ? 0u : codes8(q);
  }
  uint8_t* co = g.flat ? codes + u * 8u : codes + row * g.cpitch + ub * 8u;
  *(uint2*)co = make_uint2(c[0], c[1]);
  if (FMT == SPCONVB_NVFP4) {
    scales[g.flat ? u : row * g.spitch + ub] = (uint8_t)byte;
  } else if (!(ub & 1u)) {
    uint8_t* so = g.flat ? scales + (u >> 1) : scales + row * g.spitch + (ub >> 1);
    *so = (uint8_t)byte;
    // the two bytes behind the last block of rows of an odd number of 64 channels
    if (!g.flat && (g.upr & 4u) && ub + 2u == g.upr) so[1] = so[2] = 0;
  }
}

template <int FMT, int KIND>
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(const uint8_t* __restrict__ x, Rows g, float in_scale,
                                                                float tensor_scale, const uint32_t* n_ptr, uint32_t cap,
                                                                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  pdl_wait_and_trigger();
  const uint64_t units = (uint64_t)min(load_in_order(n_ptr), cap) * g.upr;
  const uint64_t step = (uint64_t)gridDim.x * kThreads;
  // the bound is the same for all lanes of a warp: they exchange magnitudes
  for (uint64_t first = (uint64_t)blockIdx.x * kThreads + (threadIdx.x & ~31u); first < units; first += step) {
    const uint64_t u = first + (threadIdx.x & 31u);
    const bool live = u < units;
    uint64_t row = 0;
    uint32_t ub = 0;
    if (live) {
      if (g.flat) ub = (uint32_t)(u & 1u);
      else place(g, u, row, ub);
    }
    Raw<KIND> raw;
    if (g.flat && live) {
      Rows one = g;
      one.channels = 16u;
      load_raw<KIND>(one, x, u, 0u, raw);
    } else if (live) {
      load_raw<KIND>(g, x, row, ub, raw);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 4u * elem_size<KIND>(); ++i) raw.w[i] = 0u;
    }
    store_unit<FMT, KIND>(g, row, ub, u, raw, in_scale, tensor_scale, codes, scales, live);
  }
}

template <int FMT, int KIND>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                  Rows g, float tensor_scale, const uint32_t* n_ptr,
                                                                  uint32_t cap, uint8_t* __restrict__ out) {
  pdl_wait_and_trigger();
  const uint64_t units = (uint64_t)min(load_in_order(n_ptr), cap) * g.upr;
  const uint64_t step = (uint64_t)gridDim.x * kThreads;
  constexpr uint32_t es = elem_size<KIND>();
  for (uint64_t u = (uint64_t)blockIdx.x * kThreads + threadIdx.x; u < units; u += step) {
    uint64_t row = 0;
    uint32_t ub = 0;
    place(g, u, row, ub);
    if (ub * 16u >= g.channels) continue;
    const uint32_t left = min(16u, g.channels - ub * 16u);
    const uint2 c = ld8(codes + row * g.cpitch + ub * 8u);
    const uint32_t byte =
        (uint32_t)load_in_order((const int8_t*)scales + row * g.spitch + (FMT == SPCONVB_MXFP4 ? ub >> 1 : ub)) & 255u;
    const float s = scale_value(FMT, byte, tensor_scale);
    uint32_t h[2][4], v[4 * es];
    values8(c.x, h[0]);
    values8(c.y, h[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __half22float2(*(const __half2*)&h[i / 4][i % 4]);
      const float a = __fmul_rn(f.x, s), b = __fmul_rn(f.y, s);
      if (KIND == SPCONVB_F16) {
        const __half2 p = __floats2half2_rn(a, b);
        v[i] = *(const uint32_t*)&p;
      } else {
        v[2 * i] = __float_as_uint(a);
        v[2 * i + 1] = __float_as_uint(b);
      }
    }
    uint8_t* o = out + (row * g.channels + ub * 16u) * es;
    if (left == 16u && g.aligned == 32) {
#pragma unroll
      for (uint32_t i = 0; i < es / 2u; ++i) {
        uint32_t t[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) t[j] = v[8u * i + j];
        st32(o + 32u * i, t);
      }
    } else if (g.aligned != 0) {
#pragma unroll
      for (uint32_t i = 0; i < es; ++i)
        if (i * (16u / es) < left)
          ((uint4*)o)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 16u; ++i)
        if (i < left) {
          if (KIND == SPCONVB_F32) ((uint32_t*)o)[i] = v[i];
          else ((uint16_t*)o)[i] = (uint16_t)(v[i / 2u] >> (16u * (i % 2u)));
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
  g.flat = g.channels % (format == SPCONVB_MXFP4 ? 128u : 64u) == 0u;
  const uint64_t bits = (uint64_t)(uintptr_t)p | (uint64_t)g.channels * es;
  g.aligned = bits % 32u == 0u ? 32 : (bits % 16u == 0u ? 16 : 0);
  return g;
}
int blocks_of(const Rows& g, uint32_t rows) {
  const uint64_t b = ((uint64_t)rows * g.upr + kThreads - 1) / kThreads;
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
    const uint32_t ch = cout <= 64u ? r % 64u : blk * 128u + r;
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

template <int FMT>
cudaError_t quantize_kind(int kind, int blocks, cudaStream_t st, const uint8_t* x, const Rows& g, float in_scale, float ts,
                          const uint32_t* n, uint32_t cap, uint8_t* codes, uint8_t* scales) {
  const dim3 b(blocks), t(kThreads);
  if (kind == SPCONVB_F16)
    return launch_pdl(fp4_quantize_kernel<FMT, SPCONVB_F16>, b, t, 0, st, x, g, in_scale, ts, n, cap, codes, scales);
  if (kind == SPCONVB_F32)
    return launch_pdl(fp4_quantize_kernel<FMT, SPCONVB_F32>, b, t, 0, st, x, g, in_scale, ts, n, cap, codes, scales);
  return launch_pdl(fp4_quantize_kernel<FMT, SPCONVB_I8>, b, t, 0, st, x, g, in_scale, ts, n, cap, codes, scales);
}
template <int FMT>
cudaError_t dequantize_kind(int kind, int blocks, cudaStream_t st, const uint8_t* codes, const uint8_t* scales, const Rows& g,
                            float ts, const uint32_t* n, uint32_t cap, uint8_t* out) {
  const dim3 b(blocks), t(kThreads);
  if (kind == SPCONVB_F16)
    return launch_pdl(fp4_dequantize_kernel<FMT, SPCONVB_F16>, b, t, 0, st, codes, scales, g, ts, n, cap, out);
  return launch_pdl(fp4_dequantize_kernel<FMT, SPCONVB_F32>, b, t, 0, st, codes, scales, g, ts, n, cap, out);
}

bool aligned16(const void* a, const void* b = nullptr, const void* c = nullptr) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15u) == 0u;
}

}  // namespace

// Elements of an image of packed weights and its size; 0 for shapes that no product takes.
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
  const Rows g = rows_of(format, channels, x, es);
  const int blocks = blocks_of(g, launch_rows);
  if (format == SPCONVB_MXFP4)
    SPCONVB_CUDA_TRY(quantize_kind<SPCONVB_MXFP4>(kind, blocks, (cudaStream_t)stream, (const uint8_t*)x, g, in_scale,
                                                  tensor_scale, n_ptr, launch_rows, (uint8_t*)codes, (uint8_t*)scales));
  else
    SPCONVB_CUDA_TRY(quantize_kind<SPCONVB_NVFP4>(kind, blocks, (cudaStream_t)stream, (const uint8_t*)x, g, in_scale,
                                                  tensor_scale, n_ptr, launch_rows, (uint8_t*)codes, (uint8_t*)scales));
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
  const int blocks = blocks_of(g, launch_rows);
  if (format == SPCONVB_MXFP4)
    SPCONVB_CUDA_TRY(dequantize_kind<SPCONVB_MXFP4>(out_kind, blocks, (cudaStream_t)stream, (const uint8_t*)codes,
                                                    (const uint8_t*)scales, g, tensor_scale, n_ptr, launch_rows, (uint8_t*)out));
  else
    SPCONVB_CUDA_TRY(dequantize_kind<SPCONVB_NVFP4>(out_kind, blocks, (cudaStream_t)stream, (const uint8_t*)codes,
                                                    (const uint8_t*)scales, g, tensor_scale, n_ptr, launch_rows, (uint8_t*)out));
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
  const uint64_t total = records * (1024u + words_per_chunk(format, cpad((uint32_t)cin)) * 128u);
  const uint64_t blocks = (total + 255u) / 256u;
  fp4_pack_kernel<<<(int)(blocks < kSmCount * 32u ? blocks : kSmCount * 32u), 256, 0, (cudaStream_t)stream>>>(
      format, (uint32_t)cin, (uint32_t)cout, (uint32_t)kvol, (const uint8_t*)codes, (const uint8_t*)scales,
      (uint8_t*)packed, total);
  SPCONVB_LAUNCH_CHECK();
  return SPCONVB_OK;
}

}  // extern "C"
