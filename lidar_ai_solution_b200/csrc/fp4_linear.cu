// 4-bit rows times 4-bit weights:  out[r, c] = act(alpha * sum_k x[r, k] W[c, k] + bias[c]).
//
// A tile is 128 rows (M, accumulator lanes) by 128 output channels (N, accumulator columns) on one SM, or 256 by 256 on two: a
// cluster of two CTAs, each with 128 rows, whose tensor cores share the weights, half of them in either's shared memory.  K goes by
// chunks of 256 channels: 128 bytes of codes a row, which is one swizzle atom, and four MMAs of 64 channels.  Roles of the warps of a
// CTA (one an SM, walking over tiles):
//
//   0-15   epilogue: a lane owns a row, a warp its quadrant of 32 and 32 or 64 channels
//   16     allocates tensor memory; copies the chunk's scales there and issues its MMAs, of a pair those of both CTAs.  In the second
//          CTA of a pair it tells the first one that its stage is full
//   17     one lane: TMA of the rows' codes
//   18-21  the rows' scales, a row a lane: four chunks ahead in registers, then as words into the order that the
//          copy to tensor memory wants.  (They are kept row by row in memory, so that a convolution can gather them.)
//   22     one lane: bulk copies of the weights' image (codes and scales lie ready in it)
//
// Scales in tensor memory have a place for every stage of the ring: a stage is filled again only when the MMAs that
// read its scales are complete, so no copy overwrites scales that are in use.
//
// A tile of 64 channels was slower also for 64 channels (1 row x 256 -> 64 4.3 us, with half of a tile of 128 empty 3.6): it takes as
// many instructions.  A chunk of a pair brings 38 KB into an SM and is four times the work of one of 128 x 128, which brings 36, on twice
// the SMs.  But its accumulator is the only one (two and the scales are more than tensor memory holds), drained with no MMA beside it, and
// its channels are twice as many to write before the next tile's: measured, a tile takes about 5 000 cycles and 580 a chunk, one of 128
// 2 000 and 600, a launch in pairs 1 500 more, and the launch takes what costs less over its rounds of tiles (us, pairs / not: 32 400 x
// 256 -> 512 11.8 / 9.8, x 1 024 15.5 / 16.6; 8 192 x 4 096 -> 4 096 56 / 88; 200 x 8 192 -> 8 192 18.9 / 16.6, x 16 384 -> 16 384
// 37 / 53).  With a tile of 128 rows x 256 channels on one SM, 54 KB a chunk, 8 192 x 4 096 -> 4 096 took 65.
//
// What bounds it: short K, the epilogue and the writing of fp16 rows (1 900 cycles for 32 KB a tile and SM; 32 400 x 256 -> 512 takes 9.8
// us, and 6.7 without results).  Long K, several things at once: 8 192 x 4 096 -> 4 096 takes 55 us (5.0 PFLOP/s), 5 less with no code
// copied at all, 5 less on zeros (the power limit then lowers the clock less).  Of 13 100 cycles a tile the MMAs are 8 500, 1 900 the
// exchange of the accumulator; shared memory takes in 38 KB a chunk and gives them to the tensor core, at 66 + 62 of its 128 bytes a
// cycle when the MMAs run at their full rate.
//
// Few tiles and a long K: K is split over the CTAs of a cluster, whose sums the first one collects through distributed shared memory,
// always in the same order.  That costs 5 us and a chunk takes 0.32, so it begins at 32 chunks (64 rows -> 64 channels, us, split / not:
// x 4 096 11.3 / 8.6, x 16 384 13.3 / 24.6).
#include "fp4_epilogue.cuh"

namespace spconvb {
namespace fp4 {

int linear_few(int format, const void* codes, const void* scales, uint32_t cin, const uint32_t* n_ptr, uint32_t cap,
               const void* packed, const Output& o, cudaStream_t st);

namespace {

// What goes to the CUDA cores: up to 8 rows, as long as the products are few (us there / here: 1 x 4 096 -> 4 096 5.2 / 8.8, 4 x
// 4 096 -> 4 096 8.9 / 8.8, 8 x 4 096 -> 512 5.8 / 8.6, 8 x 4 096 -> 4 096 13.9 / 8.8, 1 x 8 192 -> 8 192 12.2 / 15.5), and as long as
// a warp's share of K is short: 16 warps have 8 channels' whole K there, however few channels there are, and it is split over SMs here.  A chunk a warp
// costs 0.2 + 0.42 a row there (NVFP4; MXFP4 0.4 + 0.48), 0.55 here, and 7.8 to 8.1 more for the split (rows x chunks a warp, us there / here, NVFP4 and MXFP4: 1 x 16
// 12.5 / 19.0 and 16.2 / 19.0; 2 x 9 11.4 / 15.2 and 13.7 / 15.1; 2 x 12 14.4 / 16.8 and 17.5 / 16.7; 3 x 6 10.8 / 13.6 and 13.8 / 13.5; 4 x 4 9.4 / 12.6 and 11.5 / 12.6;
// 5 x 4 12.2 / 12.5 and 14.0 / 12.4; 8 x 2 9.7 / 11.5 and 10.8 / 11.4; 8 x 3 12.9 / 11.9 and 14.6 / 11.9; 4 x 8 16.5 / 14.8 and 20.8 / 14.8).
constexpr uint32_t kFewRows = 8;
constexpr uint64_t kFewProducts = 1ull << 26;
inline bool short_share(int format, uint32_t rows, uint32_t nchunk) {
  const uint32_t share = (nchunk + 15u) / 16u;
  return share * (format == SPCONVB_NVFP4 ? 42u * rows - 35u : 48u * rows - 15u) <= 810u;  // hundredths of a us
}
constexpr int kEpiWarps = 16, kMmaWarp = 16, kLoadWarp = 17, kScaleWarp0 = 18, kWeightWarp = 22;
constexpr int kCtaThreads = 32 * 23;
constexpr uint32_t kTileM = 128;

struct LinearArgs {
  const uint8_t* scales;
  uint32_t spitch, nchunk, last_steps;
  const uint32_t* n_ptr;
  uint32_t cap;
  const uint8_t* wpk;
  uint32_t record;  // bytes of a block of 128 channels of a chunk in the weights' image
  uint32_t* status;
  Output o;
  uint32_t split;     // CTAs of a cluster that share a tile's K
  int wait_test;
};

template <int FMT, int TN>
struct Shape {
  static constexpr bool kPair = TN == 256;  // two CTAs of a cluster, on two SMs, share a tile of 256 rows
  static constexpr uint32_t kCtas = kPair ? 2 : 1;
  static constexpr uint32_t kRows = kCtas * kTileM;                 // of a tile
  static constexpr uint32_t kWords = FMT == SPCONVB_MXFP4 ? 2 : 4;  // scale words a row and chunk
  static constexpr uint32_t kBlocks = TN > 128 ? TN / 128 : 1;      // blocks of 128 channels of the image
  static constexpr uint32_t kSf = kWords * kAtomBytes;
  static constexpr uint32_t kA = kTileM * 128, kB = 128 * 128;
  static constexpr uint32_t kOffB = kA, kOffSfb = kA + kB, kOffSfa = kOffSfb + kBlocks * kSf;
  static constexpr uint32_t kStage = kOffSfa + kSf;  // a multiple of 1024
  static constexpr uint32_t kStages = 5;
  static constexpr uint32_t kBuffers = TN == 256 ? 1 : 2;  // accumulators
  static constexpr uint32_t kSfCols = kWords * 4 * (1 + kBlocks);
  static constexpr uint32_t kPatches = TN == 256 ? 2 : 1;            // of 32 channels a warp
  static constexpr uint32_t kRing = kStages * kStage;
  static constexpr uint32_t kSmem = kRing + kEpiWarps * (kPatchBytes + kBiasBytes) + 1024 + 512;
  static_assert(kStage % 1024 == 0, "stages start on swizzle atoms");
  static_assert(kBuffers * TN + kStages * kSfCols <= kTmemCols, "tensor memory");
  static_assert(kSmem <= 232448, "shared memory");
};

__device__ __forceinline__ float ld_peer(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// SPLIT: the CTAs of a cluster share a tile's K (a kernel of its own: the sums kept for it would be spilled in the other).
template <int FMT, int TN, bool SPLIT>
__global__ void __launch_bounds__(kCtaThreads, 1)
fp4_linear_kernel(const LinearArgs a, const __grid_constant__ CUtensorMap rows_map, const __grid_constant__ CUtensorMap out_map) {
  using S = Shape<FMT, TN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t s0 = smem_u32(smem);
  uint64_t* bars = (uint64_t*)(smem + S::kRing + kEpiWarps * (kPatchBytes + kBiasBytes));
  uint32_t* tmem_holder = (uint32_t*)(bars + 2 * S::kStages + 4);
  volatile uint32_t* abort_flag = tmem_holder + 1;
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * S::kStages;
  const uint32_t bar_tfull = bar_empty + 8 * S::kStages, bar_tempty = bar_tfull + 16;
  // Warp index, row count and tensor-memory address are made the same for all lanes where the compiler sees it: what is computed from
  // them, and the loops they bound, then stay in uniform registers, which is where the tensor-core instructions take their operands.
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t cta = S::kPair ? blockIdx.x % 2u : 0u;  // of the pair; the first issues the MMAs of both

  if (threadIdx.x < S::kStages) {
    // two with copies, the four scale warps; of a pair, the second CTA, whose warp 16 passes on that its stage is full
    mbar_init(bar_full + 8 * threadIdx.x, 2 + 4 + (S::kPair && cta == 0u ? 1 : 0));
    mbar_init(bar_empty + 8 * threadIdx.x, 1);
    if (threadIdx.x < 2) {
      mbar_init(bar_tfull + 8 * threadIdx.x, 1);
      mbar_init(bar_tempty + 8 * threadIdx.x, S::kCtas * kEpiWarps);
    }
    if (threadIdx.x == 0) *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == kMmaWarp) {
    tmem_alloc_all<S::kPair>(smem_u32(tmem_holder));
  }
  pdl_wait_and_trigger();
  const uint32_t n = __shfl_sync(0xffffffffu, min(load_in_order(a.n_ptr), a.cap), 0);
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (S::kPair) cluster_sync();  // the other CTA's barriers are there
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_holder, 0);

  const uint32_t tiles_n = (a.o.cout + TN - 1) / TN;
  const uint32_t tiles = ((n + S::kRows - 1) / S::kRows) * tiles_n;
  // this CTA's tiles and its part of K
  const uint32_t split = SPLIT ? a.split : 1u;
  const uint32_t rank = SPLIT ? blockIdx.x % split : 0u;
  const uint32_t tile0 = SPLIT ? blockIdx.x / split : blockIdx.x / S::kCtas;
  const uint32_t tile_step = SPLIT ? gridDim.x / split : gridDim.x / S::kCtas;
  const uint32_t c0 = a.nchunk * rank / split, c1 = a.nchunk * (rank + 1u) / split;
  uint32_t part[32];  // with a split: this thread's sums, over the cluster's barrier

  if (warp == kLoadWarp || warp == kWeightWarp) {
    if (lane == 0) {
      uint32_t s = 0, ph = 1, it = 0;
      bool on = true;
      for (uint32_t tile = tile0; on && tile < tiles; tile += tile_step) {
        const uint32_t blk = tile % tiles_n * S::kBlocks;
        const int32_t row = (int32_t)(tile / tiles_n * S::kRows + cta * kTileM);
        const uint64_t block = (uint64_t)a.nchunk * a.record;  // of 128 channels
        const uint8_t* w = a.wpk + blk * block + (uint64_t)c0 * a.record;
        // of a pair, the codes of this CTA's block and the scales of both (the last tile may have one only)
        const bool two = S::kPair && blk * 128u + 128u < a.o.cout;
        const bool own = cta == 0u || two;
        for (uint32_t c = c0; c < c1; ++c, ++it, w += a.record) {
          if (!mbar_wait(bar_empty + 8 * s, ph, abort_flag, a.status, 21u) ||
              (a.wait_test > 0 && it + 1u >= (uint32_t)a.wait_test)) {
            on = false;
            break;
          }
          const uint32_t st = s0 + s * S::kStage, bar = bar_full + 8 * s;
          if (warp == kLoadWarp) {
            mbar_expect_tx(bar, S::kA);
            tma_load_2d(st, &rows_map, (int32_t)(c * 128u), row, bar);
          } else if (S::kPair) {
            mbar_expect_tx(bar, (own ? S::kB : 0u) + (two ? 2u : 1u) * S::kSf);
            if (own) bulk_g2s(st + S::kOffB, cta == 0u ? w : w + block, S::kB, bar);
            bulk_g2s(st + S::kOffSfb, w + 128u * 128u, S::kSf, bar);
            if (two) bulk_g2s(st + S::kOffSfb + S::kSf, w + block + 128u * 128u, S::kSf, bar);
          } else {
            mbar_expect_tx(bar, S::kB + S::kSf);
            bulk_g2s(st + S::kOffB, w, S::kB + S::kSf, bar);
          }
          if (++s == S::kStages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      if (S::kPair) {  // the last commits of the first CTA land here before this one leaves
        for (uint32_t i = 0; on && i < S::kStages; ++i) {
          on = mbar_wait(bar_empty + 8 * s, ph, abort_flag, a.status, 21u);
          if (++s == S::kStages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp >= kScaleWarp0) {
    const uint32_t r = threadIdx.x - 32u * kScaleWarp0;
    const uint32_t dst = S::kOffSfa + (r % 32u) * 16u + (r / 32u) * 4u;
    constexpr uint32_t W = S::kWords;
    const bool vec = a.spitch % (4u * W) == 0u;  // a chunk's words lie whole inside the row
    // a cursor for the loads, four chunks ahead of the one for the stages; of its tile, the row's words, or none
    uint32_t lt = tile0, lc = c0, tile = tile0, c = c0, s = 0, ph = 1;
    const uint8_t* words = nullptr;
    auto find = [&] {
      const uint64_t row = (uint64_t)(lt / tiles_n) * S::kRows + cta * kTileM + r;
      words = lt < tiles && row < n ? a.scales + row * a.spitch : nullptr;
    };
    find();
    auto load = [&](uint32_t (&v)[W]) {
#pragma unroll
      for (uint32_t w = 0; w < W; ++w) v[w] = 0u;
      if (words) {
        const uint8_t* p = words + lc * (4u * W);
        if (vec && W == 4) {
          asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v[0]), "=r"(v[1]), "=r"(v[W - 2]), "=r"(v[W - 1])
                       : "l"(p)
                       : "memory");
        } else if (vec) {
          asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "l"(p) : "memory");
        } else {
#pragma unroll
          for (uint32_t w = 0; w < W; ++w)
            if (lc * (4u * W) + 4u * w < a.spitch) v[w] = load_in_order((const uint32_t*)p + w);
        }
      }
      if (++lc == c1) {
        lc = c0;
        lt += tile_step;
        find();
      }
    };
    auto step = [&](uint32_t (&v)[W]) -> bool {
      if (tile >= tiles) return false;
      // as one warp: where a wait runs out, it may have for some lanes and not for others
      if (!__all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph, abort_flag, a.status, 22u))) return false;
      const uint32_t at = s0 + s * S::kStage + dst;
#pragma unroll
      for (uint32_t w = 0; w < W; ++w)
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + w * kAtomBytes), "r"(v[w]) : "memory");
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_full + 8 * s);
      load(v);
      if (++c == c1) {
        c = c0;
        tile += tile_step;
      }
      if (++s == S::kStages) {
        s = 0;
        ph ^= 1u;
      }
      return true;
    };
    if (c0 < c1) {
      uint32_t v0[W], v1[W], v2[W], v3[W];
      load(v0);
      load(v1);
      load(v2);
      load(v3);
      while (step(v0) && step(v1) && step(v2) && step(v3)) {
      }
    }
  } else if (S::kPair && warp == kMmaWarp && cta != 0u) {
    if (lane == 0) {
      uint32_t s = 0, ph = 0;
      bool on = true;
      for (uint32_t tile = tile0; on && tile < tiles; tile += tile_step) {
        for (uint32_t c = c0; c < c1; ++c) {
          on = mbar_wait_spin(bar_full + 8 * s, ph, abort_flag, a.status, 24u);
          if (!on) break;
          mbar_arrive_at(bar_full + 8 * s, 0u);
          if (++s == S::kStages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    auto wait = [&](uint32_t bar, uint32_t parity, uint32_t where) {
      return mbar_test_wait(bar, parity) || mbar_wait_spin(bar, parity, abort_flag, a.status, where);
    };
    const bool leader = elect_one();
    const uint64_t d0 = make_smem_desc(s0);
    const uint32_t desc_hi = (uint32_t)(d0 >> 32);
    const uint64_t f0 = scale_desc(s0);
    const uint32_t sf_hi = (uint32_t)(f0 >> 32);
    bool alive = true;
    uint32_t s = 0, ph = 0, tl = 0;
    for (uint32_t tile = tile0; tile < tiles; tile += tile_step, ++tl) {
      const uint32_t buf = S::kBuffers == 1 ? 0u : tl & 1u, use = S::kBuffers == 1 ? tl : tl >> 1;
      alive = alive && wait(bar_tempty + 8 * buf, (use & 1u) ^ 1u, 23u);
      __syncwarp();
      tc_fence_after();
      const uint32_t d_tmem = tmem + buf * TN;
      uint32_t accumulate = 0u;
      for (uint32_t c = c0; c < c1; ++c) {
        alive = alive && wait(bar_full + 8 * s, ph, 24u);
        __syncwarp();
        const uint32_t issue = leader && alive ? 1u : 0u;
        tc_fence_after();
        const uint32_t st = s * S::kStage;
        const uint32_t sf_lo = (uint32_t)f0 + (st >> 4);
        const uint32_t sfa = tmem + S::kBuffers * TN + s * S::kSfCols, sfb = sfa + S::kWords * 4u;
#pragma unroll
        for (uint32_t w = 0; w < S::kWords; ++w) {
          copy_scales_if<S::kPair>(issue, sfa + 4u * w, sf_lo + ((S::kOffSfa + w * kAtomBytes) >> 4), sf_hi);
#pragma unroll
          for (uint32_t b = 0; b < S::kBlocks; ++b)
            copy_scales_if<S::kPair>(issue, sfb + 4u * (w * S::kBlocks + b),
                           sf_lo + ((S::kOffSfb + b * S::kSf + w * kAtomBytes) >> 4), sf_hi);
        }
        const uint32_t steps = c + 1u == a.nchunk ? a.last_steps : 4u;
        const uint32_t a_lo = (uint32_t)d0 + (st >> 4), b_lo = a_lo + (S::kOffB >> 4);
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
          constexpr uint32_t kPer = FMT == SPCONVB_MXFP4 ? 2u : 1u;
          const uint32_t w = k / kPer;
          umma_scaled_if<FMT, S::kPair>(issue && k < steps ? 1u : 0u, d_tmem, a_lo + 2u * k, b_lo + 2u * k, desc_hi,
                              idesc_of<FMT>(TN, (k % kPer) * 2u, S::kRows), sfa + 4u * w,
                              sfb + 4u * w * S::kBlocks, k == 0 ? accumulate : 1u);
        }
        accumulate = 1u;
        commit_if<S::kPair>(issue, bar_empty + 8 * s);
        if (++s == S::kStages) {
          s = 0;
          ph ^= 1u;
        }
      }
      commit_if<S::kPair>(leader && alive ? 1u : 0u, bar_tfull + 8 * buf);
    }
    __syncwarp();
  } else {
    const uint32_t q = (uint32_t)warp & 3u, set = (uint32_t)warp >> 2;
    const uint32_t first = set * (32u * S::kPatches);  // channel of the tile
    Patch p;
    p.own = p.lane = lane;
    p.stage = s0 + S::kRing + (uint32_t)warp * kPatchBytes;
    p.bias = s0 + S::kRing + kEpiWarps * kPatchBytes + (uint32_t)warp * kBiasBytes;
    p.rows = n;
    uint32_t tl = 0;
    for (uint32_t tile = tile0; tile < tiles; tile += tile_step, ++tl) {
      const uint32_t buf = S::kBuffers == 1 ? 0u : tl & 1u, use = S::kBuffers == 1 ? tl : tl >> 1;
      p.row0 = (uint64_t)(tile / tiles_n) * S::kRows + cta * kTileM + 32u * q;
      const uint32_t col = (tile % tiles_n) * TN + first;
      float bias[S::kPatches];
#pragma unroll
      for (uint32_t g = 0; g < S::kPatches; ++g) {
        p.col = col + 32u * g;
        bias[g] = load_bias(a.o, p);
      }
      uint32_t ok = 1u;
      if (lane == 0) ok = mbar_wait(bar_tfull + 8 * buf, use & 1u, abort_flag, a.status, 25u) ? 1u : 0u;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      uint32_t v[S::kPatches][32];
#pragma unroll
      for (uint32_t g = 0; g < S::kPatches; ++g)
        tmem_ld32(tmem + ((32u * q) << 16) + buf * TN + first + 32u * g, v[g]);
      tmem_ld_wait();
      tc_fence_before();  // no more reads of this accumulator by this warp
      __syncwarp();
      if (lane == 0) {
        if (S::kPair && cta != 0u)
          mbar_arrive_at(bar_tempty + 8 * buf, 0u);
        else
          mbar_arrive(bar_tempty + 8 * buf);
      }
      if (SPLIT) {
#pragma unroll
        for (int i = 0; i < 32; ++i) part[i] = v[0][i];
      } else {
#pragma unroll
        for (uint32_t g = 0; g < S::kPatches; ++g) {
          p.col = col + 32u * g;
          __syncwarp();  // the bias before is read
          stage_bias(p, bias[g]);
          if (p.row0 < n && p.col < ((a.o.cout + 63u) & ~63u)) emit32<false, !SPLIT, 8>(a.o, v[g], p, &out_map);
        }
      }
    }
    if (!SPLIT) stores_done(a.o, p);
  }

  // A split's sums: every CTA but the first leaves its part in its own shared memory (no copy into it is in flight:
  // the MMAs have read all there was), the first adds them up in the order of the ranks.
  if (SPLIT) {
    const bool epi = warp < kEpiWarps && tile0 < tiles;
    const uint32_t q = (uint32_t)warp & 3u, set = (uint32_t)warp >> 2, lane_row = 32u * q + lane;
    Patch p;
    p.row0 = (uint64_t)(tile0 / tiles_n) * kTileM + 32u * q;
    p.rows = n;
    p.col = (tile0 % tiles_n) * TN + set * 32u;
    p.own = p.lane = lane;
    p.stage = s0 + S::kRing + (uint32_t)warp * kPatchBytes;
    p.bias = s0 + S::kRing + kEpiWarps * kPatchBytes + (uint32_t)warp * kBiasBytes;
    const bool live = epi && p.row0 + lane < n;
    if (epi && rank == 0u) stage_bias(p, load_bias(a.o, p));
    if (live && rank != 0u) {
#pragma unroll
      for (uint32_t i = 0; i < 32u; ++i) ((uint32_t*)smem)[(set * 32u + i) * kTileM + lane_row] = part[i];
    }
    __syncwarp();
    cluster_sync();
    if (rank == 0u) {
      if (live) {
        for (uint32_t r = 1; r < split; ++r) {
#pragma unroll
          for (uint32_t i = 0; i < 32u; ++i)
            part[i] = __float_as_uint(__uint_as_float(part[i]) +
                                      ld_peer(s0 + ((set * 32u + i) * kTileM + lane_row) * 4u, r));
        }
      }
      __syncwarp();
      if (epi && p.row0 < n && p.col < ((a.o.cout + 63u) & ~63u)) emit32<false, !SPLIT, 8>(a.o, part, p, &out_map);
    }
    __syncwarp();
    cluster_sync();  // nobody leaves while its part is read
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // give copies already issued a bounded time to land before the CTA exits
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 50000ull) {
    }
    __syncthreads();
  }
  __syncwarp();
  if (S::kPair) cluster_sync();  // nobody leaves while its memory is read or its barriers are signed
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free_all<S::kPair>(tmem);
  }
}

template <int FMT, int TN, bool SPLIT>
int launch_linear(const LinearArgs& a, const CUtensorMap& map, const CUtensorMap& out_map, uint32_t tiles, cudaStream_t st) {
  using S = Shape<FMT, TN>;
  static bool attr_done[64] = {};
  int dev = 0;
  SPCONVB_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    SPCONVB_CUDA_TRY(cudaFuncSetAttribute(fp4_linear_kernel<FMT, TN, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          (int)S::kSmem));
    if (dev >= 0 && dev < 64) attr_done[dev] = true;
  }
  const uint32_t ctas = SPLIT ? a.split : S::kCtas;  // of a cluster
  const uint32_t grid = SPLIT ? tiles * ctas : tiles < kSmCount / ctas ? tiles * ctas : (uint32_t)kSmCount;
  SPCONVB_CUDA_TRY(launch_clusters(fp4_linear_kernel<FMT, TN, SPLIT>, grid, ctas, kCtaThreads, S::kSmem, st, a, map,
                                   out_map));
  return SPCONVB_OK;
}

template <int FMT>
int launch_shape(LinearArgs a, const CUtensorMap& map, const CUtensorMap& out_map, uint32_t rows, cudaStream_t st) {
  auto tiles = [&](uint64_t tm, uint64_t tn) { return (rows + tm - 1) / tm * ((a.o.cout + tn - 1) / tn); };
  const uint64_t t = tiles(128, 128);
  a.split = 1;
  if (a.nchunk >= 32u)
    while (a.split < 8u && 2u * a.split * t <= (uint64_t)kSmCount && a.nchunk >= 8u * a.split) a.split *= 2u;
  auto cost = [&](uint64_t n, uint64_t places, uint64_t tile, uint64_t chunk) {
    return (n + places - 1) / places * (tile + chunk * a.nchunk);
  };
  // (Where K is split, even in two, that is ahead of pairs: us, split / pairs, 64 x 57 664 -> 256 20 / 80, 1 000 x 57 664 -> 1 024 43 / 83.)
  if (a.split == 1u && a.o.cout > 128u &&
      cost(tiles(256, 256), kSmCount / 2, 5000, 580) + 1500u < cost(t, kSmCount, 2000, 600))
    return launch_linear<FMT, 256, false>(a, map, out_map, (uint32_t)tiles(256, 256), st);
  return a.split > 1u ? launch_linear<FMT, 128, true>(a, map, out_map, (uint32_t)t, st)
                      : launch_linear<FMT, 128, false>(a, map, out_map, (uint32_t)t, st);
}

}  // namespace
}  // namespace fp4
}  // namespace spconvb

using namespace spconvb;
using namespace spconvb::fp4;

extern "C" int spconvb_fp4_linear(const spconvb_fp4_params* p, const void* codes, const void* scales, const uint32_t* n_ptr,
                                  uint32_t launch_rows, const void* packed, const float* bias, void* out, uint32_t* status,
                                  void* stream) {
  if (!p || !codes || !scales || !n_ptr || !packed || !out || launch_rows < 1 || launch_rows > 0x7fffff00u)
    return SPCONVB_E_ARG;
  if (!format_ok(p->format) || !channels_ok(p->cin) || !channels_ok(p->cout) || p->kvol != 1 || p->res)
    return SPCONVB_E_ARG;
  LinearArgs a{};
  if (((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)packed) & 15u || !make_output(*p, bias, out, a.o)) return SPCONVB_E_ARG;
  if (((uint64_t)launch_rows + kTileM - 1) / kTileM * (((uint64_t)p->cout + 127) / 128) > 0x7fffffffu)
    return SPCONVB_E_RANGE;  // more tiles than a 32-bit number counts
  const uint32_t cp = cpad((uint32_t)p->cin), nchunk = (cp + kChunkK - 1) / kChunkK;
  if (launch_rows <= kFewRows && (uint64_t)launch_rows * (uint32_t)p->cin * (uint32_t)p->cout <= kFewProducts &&
      short_share(p->format, launch_rows, nchunk) && !p->out_fp4 && p->wait_test == 0)
    return linear_few(p->format, codes, scales, (uint32_t)p->cin, n_ptr, launch_rows, packed, a.o, (cudaStream_t)stream);
  a.scales = (const uint8_t*)scales;
  a.spitch = scale_pitch(p->format, (uint32_t)p->cin);
  a.nchunk = nchunk;
  a.last_steps = (cp - (a.nchunk - 1) * kChunkK) / 64u;
  a.n_ptr = n_ptr;
  a.cap = launch_rows;
  a.wpk = (const uint8_t*)packed;
  a.record = 128u * 128u + words_per_chunk(p->format, cp) * kAtomBytes;
  a.status = status;
  a.wait_test = p->wait_test;

  CUtensorMap map;
  if (!encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, cp / 2u, launch_rows, 128, kTileM, CU_TENSOR_MAP_SWIZZLE_128B))
    return encode_tiled() ? SPCONVB_E_ARG : SPCONVB_E_UNSUPPORTED;
  CUtensorMap out_map{};
  a.o.bulk = encode_out(out_map, a.o, launch_rows, 32);
  return p->format == SPCONVB_MXFP4 ? launch_shape<SPCONVB_MXFP4>(a, map, out_map, launch_rows, (cudaStream_t)stream)
                                    : launch_shape<SPCONVB_NVFP4>(a, map, out_map, launch_rows, (cudaStream_t)stream);
}
