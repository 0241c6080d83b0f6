// The block-scaled tensor-core instructions of the 4-bit products, and the tensor-memory copy of their scales.
#pragma once
#include <cuda.h>

#include <utility>

#include "fp4.cuh"
#include "umma_common.cuh"

namespace spconvb {
namespace fp4 {

using namespace umma_detail;

// Instruction descriptor of kind::mxf4 / kind::mxf4nvf4: [4,6) half of the scale word of B, [7,10) A format and [10,12)
// B format (1 = e2m1), [17,23) N >> 3, [23] scale format (0 = e4m3, 1 = e8m0), [27,29) M >> 7, [29,31) half of the scale
// word of A; both operands K-major, K = 64.
template <int FMT>
__device__ __forceinline__ constexpr uint32_t idesc_of(uint32_t n, uint32_t sf_id, uint32_t m = 128) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) |
         ((FMT == SPCONVB_MXFP4 ? 1u : 0u) << 23) | ((m >> 7) << 27) | (sf_id << 29);
}

// One MMA, K = 64, by predicate from one lane of a converged warp: M = 128 on this SM, or with PAIR M = 256 on the two SMs of a
// cluster of two.  Of a pair, each SM holds its own 128 rows of A, its half of B's columns, the scales of its rows and those of all
// columns, at the same places in both; one SM issues for both, here and in the two functions below.
#define FP4_MMA(GROUP, KIND)                                                                                               \
  asm volatile(                                                                                                            \
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\t"                                               \
      "setp.ne.b32 q, %6, 0;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"                                          \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], da, db, %4, [%7], [%8], p;\n\t}" ::"r"(d_tmem),            \
      "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate), "r"(issue), "r"(sfa), "r"(sfb)                      \
      : "memory")
template <int FMT, bool PAIR = false>
__device__ __forceinline__ void umma_scaled_if(uint32_t issue, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                               uint32_t desc_hi, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                               uint32_t accumulate) {
  if (FMT == SPCONVB_MXFP4) {
    if (PAIR)
      FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
    else
      FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
  } else {
    if (PAIR)
      FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else
      FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  }
}
#undef FP4_MMA

// 128 rows of scale words (512 bytes: row r's word at (r % 32) * 16 + (r / 32) * 4) into four columns of tensor memory, the
// word of row r in lane r % 32 (of every quadrant of lanes) and column r / 32.  With PAIR each SM of the pair copies its own.
#define FP4_COPY(GROUP)                                                            \
  asm volatile(                                                                    \
      "{\n\t.reg .pred q;\n\t.reg .b64 d;\n\tsetp.ne.b32 q, %3, 0;\n\tmov.b64 d, {%1, %2};\n\t" \
      "@q tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [%0], d;\n\t}" ::"r"(tmem), \
      "r"(desc_lo), "r"(desc_hi), "r"(issue)                                       \
      : "memory")
template <bool PAIR = false>
__device__ __forceinline__ void copy_scales_if(uint32_t issue, uint32_t tmem, uint32_t desc_lo, uint32_t desc_hi) {
  if (PAIR)
    FP4_COPY("2");
  else
    FP4_COPY("1");
}
#undef FP4_COPY
// Its shared-memory descriptor: no swizzle, groups of 8 rows of 16 bytes 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) |
         ((uint64_t)1 << 46);
}

// Commits what this thread issued for the pair to the barrier at the same place in both of its CTAs.
__device__ __forceinline__ void tc_commit_pair_if(uint32_t issue, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b16 m;\n\tsetp.ne.b32 q, %1, 0;\n\tmov.b16 m, 3;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar),
      "r"(issue)
      : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void commit_if(uint32_t issue, uint32_t bar) {
  if (PAIR)
    tc_commit_pair_if(issue, bar);
  else
    tc_commit_if(issue, bar);
}
// All of an SM's tensor memory, by one warp; of a pair, one in either CTA.  The address is left at `holder` in shared memory.
constexpr uint32_t kTmemCols = 512;
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc_all(uint32_t holder) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(holder), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(holder), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free_all(uint32_t tmem) {
  if (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrives on the barrier at the same place in CTA `rank` of the cluster.  What it tells of is tensor memory, or shared memory of the
// arriving CTA whose writers have fenced it for the tensor core of that SM, which is what reads it; a release at the scope of the cluster
// would wait for the thread's global stores too, and cost 1 200 cycles.
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar, uint32_t rank) {
  asm volatile(
      "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\t"
      "mbarrier.arrive.shared::cluster.b64 _, [r];\n\t}" ::"r"(bar),
      "r"(rank)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

// A map of a matrix that is copied in boxes; false where there is none to be had.
inline bool encode_map(CUtensorMap& map, CUtensorMapDataType type, uint32_t size, const void* at, uint64_t columns, uint64_t rows,
                       uint32_t box_columns, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  const EncodeTiled encode = encode_tiled();
  const cuuint64_t dims[2] = {columns, rows}, strides[1] = {columns * size};
  const cuuint32_t box[2] = {box_columns, box_rows}, ones[2] = {1, 1};
  return encode && encode(&map, type, 2, const_cast<void*>(at), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A launch in clusters of `ctas` (1: none) that may begin while the kernel before it ends.
template <typename... P, typename... A>
cudaError_t launch_clusters(void (*kernel)(P...), uint32_t grid, uint32_t ctas, uint32_t threads, size_t smem, cudaStream_t st,
                            A&&... args) {
  cudaLaunchAttribute at[2] = {};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = ctas;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = ctas > 1u ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

}  // namespace fp4
}  // namespace spconvb
