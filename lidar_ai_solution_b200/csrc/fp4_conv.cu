// Sparse convolution of 4-bit rows as an implicit GEMM:
//
//   out[o, :] = act(alpha * sum_k W[:, k, :] . in[map[k][o], :] + bias)  (+ residual)
//
// Voxel rows on the M side (a tile is up to 128 of them, one an accumulator lane), output channels on the N side, K in chunks
// of 256 channels: 4, 2 or 1 taps of 64, 128 or 256.  Roles of the warps of a CTA (one an SM, walking over tiles whose height
// deals the rows out evenly):
//
//   0-15   epilogue: a lane owns a row, a warp its quadrant of 32 and 32 channels; with 64 channels two sets of warps take the
//          tiles in turn
//   16     allocates tensor memory, copies a chunk's scales there, issues its MMAs
//   17     one lane: the weights, a bulk copy of codes and scales a chunk, or once where all chunks fit
//   18-25  producers, two groups of four that take the chunks in turn; a warp owns 32 rows, a thread one 16-byte segment of 8
//          of them, and words of scales: cp.async of 16 and of 4 bytes, which arrive on the stage's barrier by
//          themselves.  A missing neighbour has zeros for scales; its codes stay what they were (any sixteen values are numbers, and times
//          an e4m3 scale of 0 they are 0), except in MXFP4, whose smallest scale is not 0
//   26     64 channels: every second stage's copies and MMAs, into accumulators of its own, which the epilogue adds to the others (a sum of
//          two, whichever is which).  One warp's waits, fences and commits for a stage then pass beside the other's MMAs
//
// What bounds it.  A chunk of 128 rows costs the tensor pipe 331 cycles (128 channels) or 267 (64), its 48 copies about 400 in the
// load-store pipe, and shared memory 544 in the wide layer (18 KB of rows and 18 of weights written, 32 read by the MMAs, at 128 bytes a cycle).  In
// the kernel it takes 665 (64: 570-600), counted in the issuing warp from the first full stage to the last MMA.  Of 120 000 rows 128 -> 128 the
// longest CTA walks 7 tiles of 14 chunks: 33.2 us of the 42.0 at 1 965 MHz (the clock under this load; with a residual 1 942); 5 000 cycles,
// 2.5 us, go by from its start to the first full stage, the rest is the launch and the last tile's way out.  Every tile walks all 27 taps: of a
// benchmark frame's (tile, tap) pairs 9 % have no neighbour at 120 000 rows, 21 % at 60 000 and 52 % at 14 000 (tiles of 96), and are walked all
// the same.  120 000 rows, us, MXFP4 / NVFP4: 64 -> 64 24.3 / 23.1 (with one warp for the MMAs 25.2 / 24.3, 4-bit rows out 24.0 / 23.7 and
// 26.1 / 26.4), 128 -> 128 41.1 / 42.0 (twice the scale words), with a residual 25.7 / 24.1 and 44.6 / 45.7; 14 000 rows 64 -> 64 6.6.
// Without the gather of the codes 64 -> 64 takes 19.9, without the scales' 21.0, without the output 20.7: they share the SM's issue slots and
// its load-store pipe.  Zeros for the codes of missing neighbours, too, cost NVFP4 4 %.  Stages of two chunks because every wait,
// fence and commit is paid once a stage (one chunk a stage: 28.7, 55.9).  128 channels with two warps for the MMAs take 45.7 / 46.5: their four
// accumulators leave no room for scales, and a single pair is drained with no MMA beside it.  With a tile on two SMs that share the weights
// they take 41.4 / 43.8, and 14 000 rows 10.4 / 10.9 in place of 9.4 / 10.0.
//
// Rows lie in another order in the operand than in the tile, chosen so that words of scales that the 32 lanes write at the same time lie
// in many banks (kSpread says how); the epilogue puts them back.
#include "fp4_epilogue.cuh"

namespace spconvb {
namespace fp4 {
namespace {

constexpr uint32_t kTileRows = 128;
constexpr int kEpiWarps = 16, kMmaWarp = 16, kWeightWarp = 17, kProdWarp0 = 18;
constexpr uint32_t kGroups = 2;
constexpr uint32_t kPair = 2;
constexpr int kMmaWarp2 = kProdWarp0 + 4 * (int)kGroups;
constexpr int cta_threads(int cout) { return 32 * (kMmaWarp2 + (cout == 64 ? 1 : 0)); }
constexpr uint32_t kRingBytes = 191 * 1024;
constexpr size_t kSmemBytes = kRingBytes + kEpiWarps * (kPatchBytes + kBiasBytes) + 1024 + 512;

static_assert(kSmemBytes <= 232448, "shared memory");

struct ConvArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  const int32_t* map;
  uint32_t cap, in_rows;
  const uint32_t* n_out_ptr;
  const uint8_t* wpk;
  uint32_t* status;
  int kvol;
  Output o;
  int wait_test;
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}

// A copy that is made or not made: nothing is written where it is not.
__device__ __forceinline__ void cp_async16_if(uint32_t make, uint32_t dst, const void* src) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p cp.async.cg.shared.global [%0], [%1], 16;\n\t}" ::"r"(dst),
      "l"(src), "r"(make)
      : "memory");
}

// CP: stored channels of an input row.  COUT: output channels, rounded up to 64 or 128.  RES: with a residual.
template <int FMT, int CP, int COUT, bool RES>
__global__ void __launch_bounds__(cta_threads(COUT), 1) fp4_conv_kernel(const ConvArgs a, const __grid_constant__ CUtensorMap out_map) {
  constexpr int RB = CP / 2;                       // bytes of a row's codes
  constexpr int OPC = 128 / RB, SPO = RB / 16;     // taps a chunk, 16-byte segments a tap
  constexpr uint32_t W = FMT == SPCONVB_MXFP4 && CP != 64 ? 2 : 4;  // scale words a row and chunk
  constexpr uint32_t WPT = W / OPC;                // and tap
  constexpr uint32_t kPitch = 4 * WPT;             // bytes of a row's scales
  // Where row 8 slot + i of a producer warp's 32 lies in the operand: with kSpread at 32 slot + 8 warp + i, so that a warp's copies of the
  // same scale word of its rows are 128 bytes in a row; else at 32 warp + 4 i + slot, eight groups of four banks.  (120 000 rows 128 -> 128
  // with a residual 47.4 us, so 45.8; 64 -> 64 to 4 bits 22.4 and 23.2: a row's indices are read once more for it.)
  constexpr bool kSpread = CP != 64;
  constexpr uint32_t kSteps = 4 / W;               // MMAs a word
  constexpr uint32_t kRecord = 128 * 128 + W * kAtomBytes;          // a chunk in the weights' image
  constexpr uint32_t kWeightBytes = COUT * 128 + W * kAtomBytes;     // and in shared memory
  // a stage is kPair chunks: codes, codes, scales, scales
  constexpr uint32_t kCodes = kTileRows * 128, kSfOff = kPair * kCodes, kRowStage = kSfOff + kPair * W * kAtomBytes;
  constexpr uint32_t kWeightStage = kPair * kWeightBytes;
  constexpr uint32_t kSfCols = kPair * 8 * W;  // of a stage in tensor memory: rows, weights, chunk by chunk
  constexpr uint32_t kDrain = COUT / 32 * 4;   // warps that drain a tile
  constexpr uint32_t kMmas = COUT == 64 ? 2 : 1;   // warps that issue MMAs, each into an accumulator of its own
  constexpr uint32_t kAccCols = 2 * kMmas * COUT;  // accumulators of two tiles
  constexpr uint32_t kDeepest = (kTmemCols - kAccCols) / kSfCols < kMaxStages / kMmas ? (kTmemCols - kAccCols) / kSfCols : kMaxStages / kMmas;

  const int kbytes = a.kvol * RB;
  const int nchunk = (kbytes + 127) / 128;
  const int npair = (nchunk + (int)kPair - 1) / (int)kPair;
  const uint32_t last_steps = (uint32_t)((kbytes - (nchunk - 1) * 128) / 32);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint64_t* bars = (uint64_t*)(smem + kRingBytes + kEpiWarps * (kPatchBytes + kBiasBytes));
  uint32_t* tmem_holder = (uint32_t*)(bars + 4 * kMaxStages + 4);
  volatile uint32_t* abort_flag = tmem_holder + 1;
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * kMaxStages;
  const uint32_t bar_tfull = bar_empty + 8 * kMaxStages, bar_tempty = bar_tfull + 16;
  const uint32_t bar_wfull = bar_tempty + 16, bar_wempty = bar_wfull + 8 * kMaxStages;
  // Warp index, row count and tensor-memory address are made the same for all lanes where the compiler sees it: what is computed from
  // them, and the loops they bound, then stay in uniform registers, which is where the tensor-core instructions take their operands.
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const uint32_t lane = threadIdx.x & 31;

  if (warp == kMmaWarp) {
    tmem_alloc_all<false>(smem_u32(tmem_holder));
  }
  pdl_wait_and_trigger();
  const uint32_t n_out = __shfl_sync(0xffffffffu, min(load_in_order(a.n_out_ptr), a.cap), 0);

  // Tile height: the smallest multiple of 32 with which every CTA gets the same number of tiles.
  const uint32_t per_cta = (n_out + gridDim.x - 1) / gridDim.x;
  const uint32_t rounds = max(1u, (per_cta + kTileRows - 1) / kTileRows);
  const uint32_t tile_rows = max(32u, ((per_cta + rounds - 1) / rounds + 31u) & ~31u);
  const uint32_t t32 = tile_rows >> 5;
  const uint32_t ntiles = (n_out + tile_rows - 1) / tile_rows;
  // Two rings share the buffer, rows with their scales (three stages or more) and weights with theirs.  Weights that fit beside
  // three stages of rows stay.
  const bool resident = npair <= kMaxStages && kRingBytes >= (uint32_t)npair * kWeightStage + 3u * kRowStage;
  const uint32_t nwst = resident ? (uint32_t)npair : min((uint32_t)kMaxStages, (kRingBytes - 3u * kRowStage) / kWeightStage / kMmas * kMmas);
  const uint32_t nst = min(kDeepest, (kRingBytes - nwst * kWeightStage) / kRowStage);
  // A stage has a pair of barriers for each of the MMA warps, used in turn.  The warps take the pairs of chunks in turn too, and so all
  // phases of a barrier are one warp's (and one producer group's), in order: nobody can look at one two phases early, where its parity
  // would say what it said two before.
  const uint32_t nbar = kMmas * nst;
  const uint32_t sW = smem_u32(smem), sR = sW + nwst * kWeightStage;

  if (threadIdx.x < kMaxStages) {
    mbar_init(bar_full + 8 * threadIdx.x, 32u * t32);
    mbar_init(bar_empty + 8 * threadIdx.x, 1);
    mbar_init(bar_wfull + 8 * threadIdx.x, 1);
    mbar_init(bar_wempty + 8 * threadIdx.x, 1);
    if (threadIdx.x < 2) {
      mbar_init(bar_tfull + 8 * threadIdx.x, kMmas);
      mbar_init(bar_tempty + 8 * threadIdx.x, kDrain);
    }
    if (threadIdx.x == 0) *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_holder, 0);

  if (warp == kWeightWarp) {
    // -------------------------------------------------------------- weights
    if (lane == 0) {
      uint32_t ws = 0, ph = 1;
      for (uint32_t tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
        for (int j = 0; j < nchunk; j += kPair) {
          if (!mbar_wait_spin(bar_wempty + 8 * ws, ph, abort_flag, a.status, 36u)) {
            tile = ntiles;  // (the loops end)
            break;
          }
          const uint32_t n = min(kPair, (uint32_t)(nchunk - j)), bar = bar_wfull + 8 * ws;
          const uint8_t* src = a.wpk + (size_t)j * kRecord;
          const uint32_t dst = sW + ws * kWeightStage;
          mbar_expect_tx(bar, n * kWeightBytes);
          if (COUT == 128) {
            bulk_g2s(dst, src, n * kWeightBytes, bar);
          } else {
            for (uint32_t c = 0; c < n; ++c) {
              bulk_g2s(dst + c * kWeightBytes, src + c * kRecord, COUT * 128, bar);
              bulk_g2s(dst + c * kWeightBytes + COUT * 128, src + c * kRecord + 128 * 128, W * kAtomBytes, bar);
            }
          }
          if (++ws == nwst) {
            ws = 0;
            ph ^= 1u;
          }
        }
        if (resident || tile >= ntiles) break;
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp || warp == kMmaWarp2) {
    // ------------------------------------------------------------ MMA issue
    const bool leader = elect_one();
    const uint64_t wdesc0 = make_smem_desc(sW), rdesc0 = make_smem_desc(sR);
    const uint32_t desc_hi = (uint32_t)(wdesc0 >> 32);
    const uint32_t sf_hi = (uint32_t)(scale_desc(sW) >> 32), sfw0 = (uint32_t)scale_desc(sW), sfr0 = (uint32_t)scale_desc(sR);
    bool alive = true;
    uint32_t b = 0, ws = 0, ph = 0, wph = 0, tl = 0;
    const uint32_t which = warp == kMmaWarp ? 0u : 1u;
    uint32_t turn = which;  // 0: the next stage is this warp's
    for (uint32_t tile = blockIdx.x; tile < ntiles; tile += gridDim.x, ++tl) {
      const uint32_t buf = tl & 1u;
      alive = alive && mbar_wait_spin(bar_tempty + 8 * buf, ((tl >> 1) & 1u) ^ 1u, abort_flag, a.status, 32u);
      __syncwarp();
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + (kMmas * buf + which) * COUT;
      uint32_t accumulate = 0u;
#pragma unroll 1
      for (int j = 0; j < nchunk; j += kPair) {
        if (kMmas == 1u || turn == 0u) {
          const uint32_t s = b >= nst ? b - nst : b;
          const uint32_t wp = resident ? 0u : wph;
          if (!resident || tl < 2u)
            alive = alive && (mbar_test_wait(bar_wfull + 8 * ws, wp) ||
                              mbar_wait_spin(bar_wfull + 8 * ws, wp, abort_flag, a.status, 37u));
          alive = alive && (mbar_test_wait(bar_full + 8 * b, ph) ||
                            mbar_wait_spin(bar_full + 8 * b, ph, abort_flag, a.status, 33u));
          __syncwarp();
          const uint32_t issue = leader && alive ? 1u : 0u;
          fence_proxy_async();  // rows come through the generic proxy, MMAs and copies read through the async one
          tc_fence_after();
#pragma unroll
          for (uint32_t c = 0; c < kPair; ++c) {
            if (j + (int)c >= nchunk) break;
            const uint32_t w_at = (ws * kWeightStage + c * kWeightBytes) >> 4, r_at = (s * kRowStage + c * kCodes) >> 4;
            const uint32_t f_at = (s * kRowStage + kSfOff + c * W * kAtomBytes) >> 4;
            // a place for every stage: it is filled again only when the MMAs that read its scales are complete
            const uint32_t sfr = tmem_base + kAccCols + s * kSfCols + c * 8u * W, sfw = sfr + 4u * W;
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) {
              copy_scales_if(issue, sfr + 4u * w, sfr0 + f_at + ((w * kAtomBytes) >> 4), sf_hi);
              copy_scales_if(issue, sfw + 4u * w, sfw0 + w_at + ((COUT * 128u + w * kAtomBytes) >> 4), sf_hi);
            }
            const uint32_t steps = j + (int)c + 1 == nchunk ? last_steps : 4u;
            const uint32_t wd = (uint32_t)wdesc0 + w_at, rd = (uint32_t)rdesc0 + r_at;
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
              const uint32_t w = k / kSteps;
              umma_scaled_if<FMT>(issue && k < steps ? 1u : 0u, d_tmem, rd + 2u * k, wd + 2u * k, desc_hi,
                                  idesc_of<FMT>(COUT, (k % kSteps) * 2u), sfr + 4u * w, sfw + 4u * w,
                                  k == 0 ? accumulate : 1u);
            }
            accumulate = 1u;
          }
          tc_commit_if(issue, bar_empty + 8 * b);
          if (!resident) tc_commit_if(issue, bar_wempty + 8 * ws);
        }
        turn ^= 1u;
        if (++b == nbar) {
          b = 0;
          ph ^= 1u;
        }
        if (++ws == nwst) {
          ws = 0;
          wph ^= 1u;
        }
      }
      tc_commit_if(leader && alive ? 1u : 0u, bar_tfull + 8 * buf);
    }
    __syncwarp();
  } else if (warp >= kProdWarp0) {
    // ------------------------------------------------------------ producers
    const uint32_t pw_all = (uint32_t)(warp - kProdWarp0);
    const uint32_t grp = pw_all >> 2, pw = pw_all & 3u;
    const uint32_t seg = lane & 7u, slot = lane >> 3;
    const uint32_t seg_tap = seg / SPO, seg_in = seg % SPO;
    const uint32_t row_in_tile = pw * 32u + slot * 8u;
    const bool vec_ok = (a.cap & 7u) == 0u && ((uintptr_t)a.map & 15u) == 0u;
    // Scales: with kSpread this thread copies the words of one row, for all taps of a chunk; else its tap's word of every second row.
    static_assert(kSpread || (SPO == 2 && WPT == 1), "two threads share a row's word");
    const uint32_t own_row = row_in_tile + seg;
    const uint32_t sf_dst = kSfOff + (kSpread ? (pw * 8u + seg) * 16u + slot * 4u
                                              : seg_tap * kAtomBytes + pw * 4u + slot * 16u + seg_in * 64u);

    auto load_idx = [&](uint32_t tile, int j, int32_t (&v)[8]) {
      const int k = j * OPC + (int)seg_tap;
      const uint32_t row = tile * tile_rows + row_in_tile;
      const bool live = tile < ntiles && k < a.kvol && row < n_out;
      const int32_t* src = a.map + (size_t)k * a.cap + row;
      if (live && vec_ok && row + 8u <= n_out) {
        const int4 lo = __ldg((const int4*)src), hi = __ldg((const int4*)src + 1);
        v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
        v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = (live && row + i < n_out) ? __ldg(src + i) : -1;
      }
    };
    // j counts pairs of chunks
    auto advance = [&](uint32_t& tile, int& j, int by) {
      j += by;
      while (j >= npair) {
        j -= npair;
        tile += gridDim.x;
      }
    };
    uint32_t tile = pw < t32 ? blockIdx.x : ntiles;  // a warp without rows has no chunks
    int j = 0;
    advance(tile, j, (int)grp);
    uint32_t ntile = tile;
    int nj = j;
    uint32_t it = grp, b = grp, ph = 0u;
    int32_t idx[kPair][8], own[kPair][OPC];
    auto load_pair = [&]() {
#pragma unroll
      for (uint32_t c = 0; c < kPair; ++c) load_idx(ntile, nj * (int)kPair + (int)c, idx[c]);
      if (kSpread) {
        const uint32_t row = ntile * tile_rows + own_row;
        const bool live = ntile < ntiles && row < n_out;
#pragma unroll
        for (uint32_t c = 0; c < kPair; ++c) {
#pragma unroll
          for (int t = 0; t < OPC; ++t) {
            const int k = (nj * (int)kPair + (int)c) * OPC + t;
            own[c][t] = live && k < a.kvol ? __ldg(a.map + (size_t)k * a.cap + row) : -1;
          }
        }
      }
      advance(ntile, nj, kGroups);
    };
    auto step = [&]() -> bool {
      if (tile >= ntiles) return false;
      // the use of the stage before this one, nst pairs ago
      const bool wrap = b < nst;
      const uint32_t s = wrap ? b : b - nst;
      if (!mbar_wait(bar_empty + 8 * (wrap ? b + nbar - nst : b - nst), ph ^ (wrap ? 1u : 0u), abort_flag, a.status, 31u)) return false;
#pragma unroll
      for (uint32_t c = 0; c < kPair; ++c) {
        const int chunk = j * (int)kPair + (int)c;
        if (chunk >= nchunk) break;
        const uint32_t stage = sR + s * kRowStage + c * kCodes;
        // what lies in K steps past the last tap is never read by an MMA
        const bool dead_seg = chunk == nchunk - 1 && (seg >> 1) >= last_steps;
        if (!dead_seg) {
          const uint8_t* src = a.codes + seg_in * 16u;
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i) {
            const int32_t sr = idx[c][i];
            const uint32_t r = kSpread ? i : 4u * (i & 1u) + slot;  // row of its group of 8
            const uint32_t to = stage + (kSpread ? slot * 4u + pw : pw * 4u + (i >> 1)) * 1024u + r * 128u + ((seg ^ r) << 4);
            const bool there = (uint32_t)sr < a.in_rows;
            if (FMT == SPCONVB_NVFP4) cp_async16_if(there, to, src + (int64_t)sr * RB);
            else cp_async16(to, src + (int64_t)sr * RB, there ? 16u : 0u);
          }
        }
        // (taps past the last one have indices -1, and zeros for scales)
        const uint32_t to = sR + s * kRowStage + sf_dst + c * W * kAtomBytes;
        if (kSpread) {
#pragma unroll
          for (int t = 0; t < OPC; ++t) {
            const uint8_t* src = a.scales + (int64_t)own[c][t] * kPitch;
            const uint32_t bytes = (uint32_t)own[c][t] < a.in_rows ? 4u : 0u;
#pragma unroll
            for (uint32_t w = 0; w < WPT; ++w) cp_async4(to + (t * WPT + w) * kAtomBytes, src + 4u * w, bytes);
          }
        } else {
#pragma unroll
          for (uint32_t i = 0; i < 8; i += 2) {
            const int32_t sr = seg_in ? idx[c][i + 1] : idx[c][i];
            cp_async4(to + i * 64u, a.scales + (int64_t)sr * kPitch, (uint32_t)sr < a.in_rows ? 4u : 0u);
          }
        }
      }
      if (!(a.wait_test > 0 && it + 1u >= (uint32_t)a.wait_test)) cp_async_arrive_noinc(bar_full + 8 * b);
      load_pair();
      advance(tile, j, kGroups);
      it += kGroups;
      b += kGroups;
      if (b >= nbar) {
        b -= nbar;
        ph ^= 1u;
      }
      return true;
    };
    // (a second set of indices, loaded one step further ahead, gained nothing: 120 000 rows 64 -> 64 26.0 us, with one 25.3)
    load_pair();
    while (step()) {
    }
    cp_async_wait_all();  // nothing of this thread may still be writing when the CTA exits
    __syncwarp();
  } else {
    // ------------------------------------------------------------- epilogue
    const uint32_t q = (uint32_t)warp & 3u, set = (uint32_t)warp >> 2;
    constexpr uint32_t kTurns = kEpiWarps / kDrain;  // sets of warps that take the tiles in turn
    const uint32_t turn = set / (COUT / 32u);
    Patch p;
    p.col = set % (COUT / 32u) * 32u;
    // (without kSpread lane 4 i + slot of a quadrant is row 8 slot + i of its 32)
    p.own = kSpread ? lane : (lane & 3u) * 8u + (lane >> 2);
    p.lane = lane;
    p.stage = sW + kRingBytes + (uint32_t)warp * kPatchBytes;
    p.bias = sW + kRingBytes + kEpiWarps * kPatchBytes + (uint32_t)warp * kBiasBytes;
    const bool cols = p.col < ((a.o.cout + 63u) & ~63u);
    stage_bias(p, load_bias(a.o, p));
    uint32_t tl = turn;
    for (uint32_t tile = blockIdx.x + turn * gridDim.x; tile < ntiles; tile += kTurns * gridDim.x, tl += kTurns) {
      const uint32_t buf = tl & 1u;
      p.row0 = (uint64_t)tile * tile_rows + (kSpread ? 8u : 32u) * q;
      p.rows = min((uint64_t)n_out, (uint64_t)tile * tile_rows + tile_rows);  // rows of the tile end here
      const bool any = p.row0 < p.rows && cols;
      if (RES && any) prefetch_residual<kSpread, kSpread ? 32 : 8>(a.o, p);
      uint32_t ok = 1u;
      if (lane == 0) ok = mbar_wait(bar_tfull + 8 * buf, (tl >> 1) & 1u, abort_flag, a.status, 34u) ? 1u : 0u;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      uint32_t v[32];
      const uint32_t acc = tmem_base + ((32u * q) << 16) + kMmas * buf * COUT + p.col;
      if (kMmas == 1u || npair == 1) {
        tmem_ld32(acc + (kMmas == 1u ? 0u : (tl & 1u) * COUT), v);
        tmem_ld_wait();
      } else {
        tmem_ld32(acc, v);
#pragma unroll
        for (uint32_t h = 0; h < 32u; h += 16u) {
          uint32_t u[16];
          tmem_ld16(acc + COUT + h, u);
          tmem_ld_wait();
#pragma unroll
          for (uint32_t i = 0; i < 16u; ++i) v[h + i] = __float_as_uint(__uint_as_float(v[h + i]) + __uint_as_float(u[i]));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty + 8 * buf);
      if (any) emit32<RES, kSpread, kSpread ? 32 : 8>(a.o, v, p, &out_map);
    }
    if (kSpread) stores_done(a.o, p);
    if (RES) cp_async_wait_all();  // nothing of this thread may still be writing when the CTA exits
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
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free_all<false>(tmem_base);
  }
}

template <int FMT, int CP, int COUT, bool RES>
int launch_conv(const ConvArgs& a, const CUtensorMap& out_map, uint32_t launch_rows, cudaStream_t st) {
  static bool attr_done[64] = {};
  int dev = 0;
  SPCONVB_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    SPCONVB_CUDA_TRY(cudaFuncSetAttribute(fp4_conv_kernel<FMT, CP, COUT, RES>,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes));
    if (dev >= 0 && dev < 64) attr_done[dev] = true;
  }
  const uint32_t tiles = (launch_rows + 31) / 32;  // the kernel picks the tile height
  const uint32_t grid = tiles < (uint32_t)kSmCount ? (tiles ? tiles : 1u) : (uint32_t)kSmCount;
  SPCONVB_CUDA_TRY(launch_pdl(fp4_conv_kernel<FMT, CP, COUT, RES>, dim3(grid), dim3(cta_threads(COUT)), kSmemBytes, st, a,
                              out_map));
  return SPCONVB_OK;
}
template <int FMT, int CP, int COUT>
int launch_res(const ConvArgs& a, const CUtensorMap& out_map, uint32_t rows, cudaStream_t st) {
  return a.o.res ? launch_conv<FMT, CP, COUT, true>(a, out_map, rows, st) : launch_conv<FMT, CP, COUT, false>(a, out_map, rows, st);
}
template <int FMT, int CP>
int launch_cout(const ConvArgs& a, const CUtensorMap& out_map, uint32_t rows, cudaStream_t st) {
  return a.o.cout <= 64u ? launch_res<FMT, CP, 64>(a, out_map, rows, st) : launch_res<FMT, CP, 128>(a, out_map, rows, st);
}
template <int FMT>
int launch_cin(uint32_t cp, const ConvArgs& a, const CUtensorMap& out_map, uint32_t rows, cudaStream_t st) {
  if (cp == 64u) return launch_cout<FMT, 64>(a, out_map, rows, st);
  return cp == 128u ? launch_cout<FMT, 128>(a, out_map, rows, st) : launch_cout<FMT, 256>(a, out_map, rows, st);
}

}  // namespace
}  // namespace fp4
}  // namespace spconvb

using namespace spconvb;
using namespace spconvb::fp4;

extern "C" {

int spconvb_fp4_conv_supported(int32_t cin, int32_t cout, int32_t kvol) {
  if (cin < 1 || cin > 256 || cout < 1 || cout > 128 || kvol < 1 || kvol > kMaxTaps) return 0;
  return cpad((uint32_t)cin) != 192u ? 1 : 0;
}

int spconvb_fp4_conv(const spconvb_fp4_params* p, const void* codes, const void* scales, const int32_t* map, uint32_t cap,
                     const uint32_t* n_out_ptr, uint32_t launch_rows, const void* packed, const float* bias, void* out,
                     uint32_t* status, void* stream) {
  if (!p || !codes || !scales || !map || !n_out_ptr || !packed || !out || cap < 1 || cap > 0x7fffff00u || p->in_rows < 1 ||
      p->in_rows > 0x80000000u)
    return SPCONVB_E_ARG;
  if (!format_ok(p->format) || !channels_ok(p->cin) || !channels_ok(p->cout) || p->kvol < 1) return SPCONVB_E_ARG;
  ConvArgs a{};
  if (((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)packed) & 15u || (uintptr_t)map & 3u || !make_output(*p, bias, out, a.o))
    return SPCONVB_E_ARG;
  if (!spconvb_fp4_conv_supported(p->cin, p->cout, p->kvol)) return SPCONVB_E_UNSUPPORTED;
  if (launch_rows == 0 || launch_rows > cap) launch_rows = cap;
  a.codes = (const uint8_t*)codes;
  a.scales = (const uint8_t*)scales;
  a.map = map;
  a.cap = cap;
  a.in_rows = p->in_rows;
  a.n_out_ptr = n_out_ptr;
  a.wpk = (const uint8_t*)packed;
  a.status = status;
  a.kvol = p->kvol;
  a.wait_test = p->wait_test;
  const uint32_t cp = cpad((uint32_t)p->cin);
  CUtensorMap out_map{};
  a.o.bulk = cp != 64u && encode_out(out_map, a.o, cap, 8);
  return p->format == SPCONVB_MXFP4 ? launch_cin<SPCONVB_MXFP4>(cp, a, out_map, launch_rows, (cudaStream_t)stream)
                                    : launch_cin<SPCONVB_NVFP4>(cp, a, out_map, launch_rows, (cudaStream_t)stream);
}

}  // extern "C"
