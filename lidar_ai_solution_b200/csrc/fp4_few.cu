// The linear layer of a few rows (single tokens, pooled features): out[r, c] = act(alpha * sum_k x[r, k] W[c, k] + bias[c]) for up to
// eight rows, on the CUDA cores.
//
// All of it is reading the weights once, and a tile of the tensor cores would be 120 empty rows: what counts is that the
// whole GPU reads at once and that little comes before and after.  A CTA owns 8 output channels, one row group of the
// weights' image, and its warps share K: a chunk of the group is 1 KB in a row, 32 bytes a lane (4 lanes a channel), read in one piece.  Codes
// become fp16 in pairs; the products of two codes are multiples of 1/4 up to 36, so the sums of 8 of them are exact in
// fp16, and a block of 16 channels is 8 two-way multiply-adds; times both block scales it goes into fp32.
// The lanes of a channel and then the warps are added in a fixed order.  Measured, NVFP4, us a launch in a chain: 1 row x 4 096 -> 4 096
// 5.1 (9.5 MB; 2.4 of it are a launch that reads next to nothing), 1 x 8 192 -> 8 192 12.2 (3.1 TB/s): what bounds it there is the
// conversion of codes, done again for every channel on the rows' side.  A long K stays with 16 warps, 0.5 to 0.6 us a chunk of each and row (1 x 65 536 -> 128
// 12.5, 2 x 18.6): the linear layer's rule sends longer shares elsewhere.
#include "fp4_epilogue.cuh"

namespace spconvb {
namespace fp4 {
namespace {

struct FewArgs {
  const uint8_t *codes, *scales;
  uint32_t cpitch, spitch, nchunk;
  uint64_t k;         // stored channels
  const uint32_t* n_ptr;
  uint32_t cap;
  const uint8_t* wpk;
  uint32_t record, words;
  Output o;
};

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Sum of 16 products of codes (two words of eight each), exact.
__device__ __forceinline__ float dot16(const uint32_t (&a)[2], const uint32_t (&b)[2][4]) {
  uint32_t s = 0u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h[4];
    values8(a[i], h);
#pragma unroll
    for (int j = 0; j < 4; ++j) s = hfma2(h[j], b[i][j], s);
  }
  const float2 f = __half22float2(*(const __half2*)&s);
  return f.x + f.y;
}

// The scale that a sum is multiplied by first, and the one after it.  Powers of two between 2^-127 and 2^127: times the smaller one a sum (a
// multiple of 1/4 up to 576) loses no bit, and is infinite only where the product of all three is.  (A NaN is the larger one.)  e4m3
// numbers are far from either end, in any order.
template <int FMT>
__device__ __forceinline__ float first_of(float s, float x) { return FMT == SPCONVB_MXFP4 ? fminf(s, x) : s; }
template <int FMT>
__device__ __forceinline__ float then_of(float s, float x) { return FMT == SPCONVB_MXFP4 ? max_nan(s, x) : x; }

template <int FMT, int R>
__global__ void __launch_bounds__(512) fp4_few_kernel(const FewArgs a) {
  __shared__ float sums[16][R][8];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t r8 = lane >> 2, quarter = lane & 3u;   // channel of the group, 32 bytes of its 128
  const uint32_t group = blockIdx.x, blk = group / 16u, row_in_blk = group % 16u * 8u + r8;
  pdl_wait_and_trigger();
  const uint32_t n = min(load_in_order(a.n_ptr), a.cap);
  float acc[R] = {};
  const uint8_t* image = a.wpk + (uint64_t)blk * a.nchunk * a.record;
#pragma unroll 2
  for (uint32_t c = warp; c < a.nchunk; c += warps) {
    const uint8_t* rec = image + (uint64_t)c * a.record;
    uint32_t w[8];
    ld32(rec + (group % 16u) * 1024u + lane * 32u, w);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t seg = (quarter * 2u + h) ^ r8;     // 32 channels of the chunk; the image is swizzled
      const uint64_t k = (uint64_t)c * kChunkK + seg * 32u;
      if (k >= a.k) continue;                           // padding of the last chunk
      // the scales of the weights' two blocks of 16 (or one of 32), in the word of their channel
      const uint8_t* sw = rec + 128u * 128u + (row_in_blk % 32u) * 16u + (row_in_blk / 32u) * 4u;
      uint32_t sb;
      if (FMT == SPCONVB_NVFP4)
        sb = (uint32_t)load_in_order((const uint16_t*)(sw + (seg / 2u) * kAtomBytes + (seg % 2u) * 2u));
      else
        sb = (uint32_t)load_in_order((const int8_t*)(sw + (a.words == 2u ? seg / 4u : seg / 2u) * kAtomBytes +
                                                     (a.words == 2u ? seg % 4u : seg % 2u))) & 255u;
      uint32_t b[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) values8(w[4u * h + i], b[i]);
      const float s0 = scale_value(FMT, sb & 255u, 1.f), s1 = FMT == SPCONVB_NVFP4 ? scale_value(FMT, sb >> 8, 1.f) : s0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= (int)n) break;
        const uint4 x = ld16(a.codes + (uint64_t)r * a.cpitch + k / 2u);
        uint32_t xb;
        if (FMT == SPCONVB_NVFP4) xb = (uint32_t)load_in_order((const uint16_t*)(a.scales + (uint64_t)r * a.spitch + k / 16u));
        else xb = (uint32_t)load_in_order((const int8_t*)(a.scales + (uint64_t)r * a.spitch + k / 32u)) & 255u;
        const uint32_t lo[2] = {x.x, x.y}, hi[2] = {x.z, x.w};
        const uint32_t b0[2][4] = {{b[0][0], b[0][1], b[0][2], b[0][3]}, {b[1][0], b[1][1], b[1][2], b[1][3]}};
        const uint32_t b1[2][4] = {{b[2][0], b[2][1], b[2][2], b[2][3]}, {b[3][0], b[3][1], b[3][2], b[3][3]}};
        const float d0 = dot16(lo, b0), d1 = dot16(hi, b1);
        const float x0 = scale_value(FMT, xb & 255u, 1.f), x1 = FMT == SPCONVB_NVFP4 ? scale_value(FMT, xb >> 8, 1.f) : x0;
        // (a sum and two scales are at most 20 bits: exact, and a sum of 0 stays one where the scales' product would overflow)
        acc[r] = fmaf(__fmul_rn(d0, first_of<FMT>(s0, x0)), then_of<FMT>(s0, x0), acc[r]);
        acc[r] = fmaf(__fmul_rn(d1, first_of<FMT>(s1, x1)), then_of<FMT>(s1, x1), acc[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], 1);
    acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], 2);
    if (quarter == 0u) sums[warp][r][r8] = acc[r];
  }
  __syncthreads();
  const uint32_t r = threadIdx.x / 8u, c = group * 8u + threadIdx.x % 8u;
  if (r < R && r < n && c < a.o.cout) {
    float y = 0.f;
    for (uint32_t w = 0; w < warps; ++w) y += sums[w][r][threadIdx.x % 8u];
    y = fmaf(y, a.o.alpha, a.o.bias ? __uint_as_float(load_in_order((const uint32_t*)a.o.bias + c)) : 0.f);
    if (a.o.act == SPCONVB_ACT_RELU) y = max_nan(y, 0.f);
    ((__half*)a.o.out)[(uint64_t)r * a.o.cout + c] = __float2half_rn(y);
  }
}

template <int FMT>
cudaError_t launch_few(const FewArgs& a, uint32_t rows, cudaStream_t st) {
  const uint32_t warps = a.nchunk < 16u ? a.nchunk : 16u;
  const dim3 grid((a.o.cout + 7u) / 8u), block(32u * (warps < 2u ? 2u : warps));
  if (rows <= 1u) return launch_pdl(fp4_few_kernel<FMT, 1>, grid, block, 0, st, a);
  if (rows <= 2u) return launch_pdl(fp4_few_kernel<FMT, 2>, grid, block, 0, st, a);
  if (rows <= 4u) return launch_pdl(fp4_few_kernel<FMT, 4>, grid, block, 0, st, a);
  return launch_pdl(fp4_few_kernel<FMT, 8>, grid, block, 0, st, a);
}

}  // namespace

int linear_few(int format, const void* codes, const void* scales, uint32_t cin, const uint32_t* n_ptr, uint32_t cap,
               const void* packed, const Output& o, cudaStream_t st) {
  FewArgs a{};
  const uint32_t cp = cpad(cin);
  a.codes = (const uint8_t*)codes;
  a.scales = (const uint8_t*)scales;
  a.cpitch = code_pitch(cin);
  a.spitch = scale_pitch(format, cin);
  a.nchunk = (cp + kChunkK - 1) / kChunkK;
  a.k = cp;
  a.n_ptr = n_ptr;
  a.cap = cap;
  a.wpk = (const uint8_t*)packed;
  a.words = words_per_chunk(format, cp);
  a.record = 128u * 128u + a.words * kAtomBytes;
  a.o = o;
  SPCONVB_CUDA_TRY(format == SPCONVB_MXFP4 ? launch_few<SPCONVB_MXFP4>(a, cap, st) : launch_few<SPCONVB_NVFP4>(a, cap, st));
  return SPCONVB_OK;
}

}  // namespace fp4
}  // namespace spconvb
