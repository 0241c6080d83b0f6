// What both products do with their sums: a lane owns a row, 32 channels at a time.
#pragma once
#include "fp4_umma.cuh"
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
  int bulk;    // fp16: whole patches go out as tensor copies
  int access;  // bytes of an fp16 row that may be stored (and of the residual, read) at once: 16, 4 or 2
};

// A warp's 32 rows x 32 channels of fp16 between its lanes and memory by way of 2 KB of shared memory: a lane has a row
// there, and a quarter of a row on the way to memory, where eight rows go at a time (a lane's own 32 bytes of 32 rows touch 32
// lines an instruction and not 8).  Piece c (16 bytes) of row r lies at piece c ^ (r / 2 + r / 8) % 4 of its 64 bytes: free of bank conflicts
// for lanes that have rows 0, 1, 2, ... and for lanes that have rows 0, 8, 16, 24, 1, 9, ...
constexpr uint32_t kPatchBytes = 2048, kBiasBytes = 128;
__device__ __forceinline__ uint32_t staged_at(uint32_t r, uint32_t c) {
  return r * 64u + ((c ^ ((r >> 1 ^ r >> 3) & 3u)) << 4);
}
__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// Where a warp's 32 rows x 32 channels are: four times eight rows from row0 on, which begin APART rows from each other (those below `rows`
// exist; row `own` of the 32 is this lane's), channels col ..
struct Patch {
  uint64_t row0, rows;
  template <int APART>
  __device__ __forceinline__ uint64_t row(uint32_t r) const {
    return row0 + (APART == 8 ? r : r / 8u * APART + r % 8u);
  }
  uint32_t col, own, lane, stage, bias;  // (the last two: addresses in shared memory)
};

// Of fp16 results, a patch all of whose rows exist leaves as one tensor copy of 32 x 32, which the next patch waits for before it writes
// there: the lanes' four loads and stores and the wait between them are out of the way of the next tile (32 400 x 256 -> 512 12.3 us, this way
// 9.8; 120 000 x 256 -> 256 19.9 and 15.6; 100 x 256 -> 128 3.8 and 3.6).  Its pieces lie as that copy wants them: piece c of row r
// at c ^ (r / 2) % 4.  (Rows that begin 32 from each other leave as four copies of eight.)
__device__ __forceinline__ uint32_t copied_at(uint32_t r, uint32_t c) { return r * 64u + ((c ^ (r >> 1 & 3u)) << 4); }
template <int APART>
__device__ __forceinline__ bool patch_whole(const Patch& p) {  // every box of it: there, or not there
  if (APART == 8) return p.row0 + 32u <= p.rows;
  bool whole = true;
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    const uint64_t row = p.row<APART>(8u * k);
    whole = whole && (row + 8u <= p.rows || row >= p.rows);
  }
  return whole;
}
template <int APART>
__device__ __forceinline__ void store_patch(const CUtensorMap* map, const Patch& p) {
#pragma unroll
  for (uint32_t k = 0; k < (APART == 8 ? 1u : 4u); ++k) {
    const uint64_t row = p.row<APART>(8u * k);
    if (k == 0 || row < p.rows)
      asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map),
                   "r"((int32_t)p.col), "r"((int32_t)row), "r"(p.stage + k * 512u)
                   : "memory");
  }
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// By all lanes: what this warp has stored has left shared memory; and, before the CTA ends, has been written.
template <bool BULK>
__device__ __forceinline__ void patch_free(const Output& o, const Patch& p) {
  if (BULK && o.bulk && p.lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void stores_done(const Output& o, const Patch& p) {
  if (o.bulk && p.lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// The patch's bias on its way into shared memory (zeros where there is none): a load that the epilogue would wait for is made long
// before it.  (Read where it is used, 14 000 rows 64 -> 64 took 8.8 us and not 6.5.)
__device__ __forceinline__ float load_bias(const Output& o, const Patch& p) {
  return o.bias && p.col + p.lane < o.cout ? __uint_as_float(load_in_order((const uint32_t*)o.bias + p.col + p.lane)) : 0.f;
}
__device__ __forceinline__ void stage_bias(const Patch& p, float b) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(p.bias + 4u * p.lane), "f"(b) : "memory");
}

// The residual on its way into the patch's shared memory, in program order: it may be what the launch before wrote.  (Rows that do
// not start on 16 bytes go by pairs of channels, two rows an instruction, or by single ones.)
template <bool BULK, int APART>
__device__ __forceinline__ void prefetch_residual(const Output& o, const Patch& p) {
  patch_free<BULK>(o, p);  // what was there is read
  if (o.access >= 16) {
    const uint32_t c = p.col + 8u * (p.lane % 4u);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t r = 8u * k + p.lane / 4u;
      const bool there = p.row<APART>(r) < p.rows && c < o.cout;
      cp_async16(p.stage + staged_at(r, p.lane % 4u), o.res + (there ? p.row<APART>(r) * o.cout + c : 0u), there ? 16u : 0u);
    }
    return;
  }
  const uint32_t per = o.access == 4 ? 2u : 1u, lanes = 32u / per;  // channels a lane, lanes a row
  const uint32_t at = p.lane % lanes * per;
#pragma unroll 8
  for (uint32_t k = 0; k < lanes; ++k) {
    const uint32_t r = k * per + p.lane / lanes;
    const bool there = p.row<APART>(r) < p.rows && p.col + at < o.cout;
    const __half* from = o.res + p.row<APART>(r) * o.cout + p.col + at;
    const uint32_t to = p.stage + staged_at(r, at / 8u) + at % 8u * 2u;
    if (per == 2u) {
      const uint32_t v = there ? load_in_order((const uint32_t*)from) : 0u;
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(v) : "memory");
    } else {
      const uint16_t v = there ? (uint16_t)load_in_order((const uint16_t*)from) : (uint16_t)0;
      asm volatile("st.shared.b16 [%0], %1;" ::"r"(to), "h"(v) : "memory");
    }
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN stays one
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// Two sums at a time: a * b + c, each rounded once.
__device__ __forceinline__ void fma2(uint32_t& x, uint32_t& y, float b, uint32_t c0, uint32_t c1) {
  asm("{\n\t.reg .b64 v, w, u;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 w, {%2, %2};\n\tmov.b64 u, {%3, %4};\n\t"
      "fma.rn.f32x2 v, v, w, u;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+r"(x), "+r"(y)
      : "f"(b), "r"(c0), "r"(c1));
}
__device__ __forceinline__ uint32_t halves_of(uint32_t x, uint32_t y) {
  const __half2 h = __floats2half2_rn(__uint_as_float(x), __uint_as_float(y));
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}

// Sums of 32 channels of this lane's row to results in memory: alpha, bias, activation, residual, fp16 or 4 bits.
// `col` is a multiple of 32 below cout rounded up to 64.
template <bool RES, bool BULK, int APART>
__device__ __forceinline__ void emit32(const Output& o, uint32_t (&v)[32], const Patch& p, const CUtensorMap* out_map) {
  const uint64_t row = p.row<APART>(p.own);
  const bool live = row < p.rows;
  if (RES) cp_async_wait_all();
  patch_free<BULK>(o, p);  // residual and bias are there, and what was there is read
  // step by step over all 32 channels, so that the loads of a step are in flight together
  {
    uint4 b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = ld_shared16(p.bias + 16u * i);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      fma2(v[4 * i], v[4 * i + 1], o.alpha, b[i].x, b[i].y);
      fma2(v[4 * i + 2], v[4 * i + 3], o.alpha, b[i].z, b[i].w);
    }
  }
  const bool relu = o.act == SPCONVB_ACT_RELU;
  if (RES || o.mode == 0) {
    // fp16 from here on (the sum with a residual is rounded as if it had been stored); ReLU before or after a rounding is the same
    uint32_t h[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) h[i] = halves_of(v[2 * i], v[2 * i + 1]);
    if (relu) {
#pragma unroll
      for (int i = 0; i < 16; ++i) h[i] = max_nan2(h[i], 0u);
    }
    if (RES) {
      uint32_t r[16];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 t = ld_shared16(p.stage + staged_at(p.own, c));
        r[4 * c] = t.x; r[4 * c + 1] = t.y; r[4 * c + 2] = t.z; r[4 * c + 3] = t.w;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x = __half22float2(*(const __half2*)&h[i]), y = __half22float2(*(const __half2*)&r[i]);
        v[2 * i] = __float_as_uint(__fadd_rn(x.x, y.x));
        v[2 * i + 1] = __float_as_uint(__fadd_rn(x.y, y.y));
        if (o.mode == 0) h[i] = halves_of(v[2 * i], v[2 * i + 1]);
      }
      if (o.res_relu && o.mode == 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = max_nan2(h[i], 0u);
      }
    }
    if (o.mode == 0) {
      if (BULK && o.bulk && patch_whole<APART>(p)) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          st_shared16(p.stage + copied_at(p.own, c), h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
        fence_proxy_async();
        __syncwarp();
        if (p.lane == 0 && p.col < o.cout) store_patch<APART>(out_map, p);
        return;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
        st_shared16(p.stage + staged_at(p.own, c), h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
      __syncwarp();
      if (o.access < 16) {
        const uint32_t per = o.access == 4 ? 2u : 1u, lanes = 32u / per;
        const uint32_t at = p.lane % lanes * per;
        if (p.col + at >= o.cout) return;
#pragma unroll 8
        for (uint32_t k = 0; k < lanes; ++k) {
          const uint32_t r = k * per + p.lane / lanes;
          if (p.row<APART>(r) >= p.rows) break;
          __half* to = (__half*)o.out + p.row<APART>(r) * o.cout + p.col + at;
          const uint32_t from = p.stage + staged_at(r, at / 8u) + at % 8u * 2u;
          if (per == 2u) {
            uint32_t v;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
            *(uint32_t*)to = v;
          } else {
            uint16_t v;
            asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
            *(uint16_t*)to = v;
          }
        }
        return;
      }
      uint4 t[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) t[k] = ld_shared16(p.stage + staged_at(8u * k + p.lane / 4u, p.lane % 4u));
      const uint32_t c = p.col + 8u * (p.lane % 4u);
      const uint64_t at = p.row0 + p.lane / 4u;
      const uint32_t left = c < o.cout && at < p.rows ? (uint32_t)min(p.rows - at, (uint64_t)(4 * APART)) : 0u;
      __half* to = (__half*)o.out + at * o.cout + c;
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)
        if (APART * k < left) *(uint4*)(to + APART * k * o.cout) = t[k];
      return;
    }
  }
  if (RES ? o.res_relu != 0 : relu) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(max_nan(__uint_as_float(v[i]), 0.f));
  }
  if (p.col + 32u > o.cout) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = p.col + i < o.cout ? v[i] : 0u;
  }
  if (!live) return;
  uint32_t amax[2], c[4], byte[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) m = max_abs_nan(m, __uint_as_float(v[16 * h + i]), __uint_as_float(v[16 * h + i + 1]));
    amax[h] = __float_as_uint(m);
  }
  const bool mx = o.mode == 1;
  if (mx) amax[0] = amax[1] = max(amax[0], amax[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float s, y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(v[16 * h + i]);
    byte[h] = mx ? scale_mx(amax[h], s) : scale_nv(amax[h], o.ts, s);
    codes_of<16>(mx, y, s, amax[h], c + 2 * h);
  }
  *(uint4*)(o.out + row * o.cpitch + p.col / 2u) = make_uint4(c[0], c[1], c[2], c[3]);
  uint8_t* so = o.out_scales + row * o.spitch;
  if (mx) {
    so[p.col / 32u] = (uint8_t)byte[0];
    // the bytes behind the last block of rows of an odd number of 64 channels
    if (p.col / 2u + 16u == o.cpitch && (o.cpitch & 32u)) so[p.col / 32u + 1u] = so[p.col / 32u + 2u] = 0;
  } else {
    *(uint16_t*)(so + p.col / 16u) = (uint16_t)(byte[0] | byte[1] << 8);
  }
}

// Host: the output's part of a call's parameters; false where they are not valid.
inline bool make_output(const spconvb_fp4_params& p, const float* bias, void* out, Output& o) {
  if (p.act != SPCONVB_ACT_NONE && p.act != SPCONVB_ACT_RELU) return false;
  if (!(p.alpha >= -3.4028235e38f && p.alpha <= 3.4028235e38f)) return false;  // times a sum of 0 it would be a NaN
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
  o.access = bits % 16u == 0u ? 16 : (bits % 4u == 0u ? 4 : 2);
  return true;
}

// Host: the map of fp16 results, where their rows can be copied so.
inline bool encode_out(CUtensorMap& map, const Output& o, uint32_t rows, uint32_t box_rows) {
  return o.mode == 0 && o.access == 16 && o.cout >= 32u &&
         encode_map(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, o.out, o.cout, rows, 32, box_rows, CU_TENSOR_MAP_SWIZZLE_64B);
}

}  // namespace fp4
}  // namespace spconvb
