/*
 * spconvb_fp4.h - microscaled 4-bit floating point: rows, weights and their products.
 *
 * The precision below int8: e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with a scale for every
 * 16 or 32 channels of a row, multiplied by the block-scaled tensor-core instructions of sm_100a with fp32
 * accumulators.  The conventions are those of spconvb.h: stream-ordered, row counts in device memory, no allocation,
 * no synchronisation, capturable.  Rows, quantised or not, and the linear layer: rows [0, min(*n_ptr, launch_rows)) are processed, the
 * buffers hold launch_rows rows.  The convolution: rows [0, min(*n_out_ptr, cap)), the buffers hold cap rows, launch_rows only
 * sizes the grid.  Rows behind those are left as they were.  Buffers may not overlap unless a comment says so.
 *
 * Formats
 *   SPCONVB_MXFP4  blocks of 32 channels; scale byte e8m0 = exponent + 127 of 2^(floor(log2 amax) - 2), the
 *                  exponent clamped to -127 (amax = 0 gives byte 0).  No tensor scale: pass 1.
 *   SPCONVB_NVFP4  blocks of 16 channels; scale byte e4m3 = amax / (6 * tensor_scale), rounded to nearest even and
 *                  saturated at 448; tensor_scale is one positive fp32 number a tensor, from 1.2e-38 to 7.5e35.
 *   A block's scale is S = 2^e, or e4m3 * tensor_scale rounded to fp32; its codes are x / S (in fp32, to the last bit, and
 *   exactly on the borders between codes) rounded to nearest even and saturated at 6, all 0 where S is 0 (the sign of a zero is not specified).  A block that holds an infinity or a NaN gets the NaN scale
 *   (0xff, 0x7f) and codes 0, so that it stays visible: it reads as NaN, and so does every product with it.  (Of
 *   weights: its output channel, in every row, also where a convolution's row lacks that neighbour.)
 *
 * Layout of rows (all pointers 16-byte aligned)
 *   codes   uint8 [rows][cpad / 2], cpad = channels rounded up to 64; code = sign << 3 | index of the value, the even
 *           channel in the low four bits.  The codes of padding channels are 0.
 *   scales  uint8 [rows][spconvb_fp4_scale_pitch()]: one byte a block, a multiple of 4 bytes a row.  Padding
 *           blocks and bytes are 0.
 */
#ifndef SPCONVB_FP4_H_
#define SPCONVB_FP4_H_

#include "spconvb.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SPCONVB_MXFP4 0
#define SPCONVB_NVFP4 1

/* one more element kind, for the calls of this header only */
#define SPCONVB_F32 2

/* Most channels of a row. */
#define SPCONVB_FP4_MAX_CHANNELS 65536

/* Bytes of a row's codes and of its scales; 0 for a format or a number of channels that is not offered. */
SPCONVB_API uint32_t spconvb_fp4_code_pitch(int32_t channels);
SPCONVB_API uint32_t spconvb_fp4_scale_pitch(int32_t format, int32_t channels);

/* Rows x [launch_rows][channels] (SPCONVB_F16, SPCONVB_F32, or SPCONVB_I8 times in_scale; in_scale is not used
 * otherwise) to codes and scales.  x needs the alignment of its elements only. */
SPCONVB_API int spconvb_fp4_quantize(int32_t format, const void* x, int32_t kind, float in_scale,
                                     int32_t channels, float tensor_scale, const uint32_t* n_ptr,
                                     uint32_t launch_rows, void* codes, void* scales, void* stream);

/* Codes and scales to rows out [launch_rows][channels] (SPCONVB_F16 or SPCONVB_F32): code * S in fp32, rounded
 * once more for fp16.  out needs the alignment of its elements only. */
SPCONVB_API int spconvb_fp4_dequantize(int32_t format, const void* codes, const void* scales,
                                       int32_t channels, float tensor_scale, int32_t out_kind,
                                       const uint32_t* n_ptr, uint32_t launch_rows, void* out,
                                       void* stream);

/* Weights: [cout][kvol][cin] quantised as cout * kvol rows of cin channels, laid out once for the products below.  kvol 1 in any
 * sizes, for spconvb_fp4_linear; more taps where spconvb_fp4_conv_supported() says 1 (else SPCONVB_E_UNSUPPORTED). */
SPCONVB_API size_t spconvb_fp4_packed_bytes(int32_t format, int32_t cin, int32_t cout, int32_t kvol);
SPCONVB_API int spconvb_fp4_pack_weights(int32_t format, int32_t cin, int32_t cout, int32_t kvol,
                                         const void* codes, const void* scales, void* packed,
                                         void* stream);

typedef struct spconvb_fp4_params {
  int32_t format;         /* of rows and weights */
  int32_t cin, cout, kvol;
  float alpha;            /* tensor scale of the rows times that of the weights; finite */
  int32_t act;            /* SPCONVB_ACT_* */
  /* Output: fp16 [rows][cout], or 4-bit rows of `out_format` and `out_tensor_scale` with their scales in out_scales. */
  int32_t out_fp4;        /* 0: fp16 */
  int32_t out_format;
  float out_tensor_scale;
  void* out_scales;
  /* Residual add (spconvb_fp4_conv only; NULL: none), fp16 [rows][cout]: the result is rounded to fp16 as if it had been
   * stored, then out = relu?(result + res).  It may be `out` itself. */
  const void* res;
  int32_t res_relu;
  int32_t wait_test;      /* 0 in normal use; as in spconvb_conv_params */
  uint32_t in_rows;       /* rows of `codes` and `scales` (spconvb_fp4_conv only), at least 1: what the map says beyond them is missing.
                             (An input without rows is one row of zeros, which add nothing.) */
} spconvb_fp4_params;

/* out[r] = act(alpha * W . x[r] + bias), kvol = 1, any cin and cout up to SPCONVB_FP4_MAX_CHANNELS.  bias: fp32 [cout]
 * or NULL.  status: the status block (SPCONVB_ST_TIMEOUT) or NULL. */
SPCONVB_API int spconvb_fp4_linear(const spconvb_fp4_params* p, const void* codes,
                                   const void* scales, const uint32_t* n_ptr, uint32_t launch_rows,
                                   const void* packed, const float* bias, void* out,
                                   uint32_t* status, void* stream);

/* 1 where spconvb_fp4_conv covers these sizes: cin <= 64, 65..128 or 193..256 (rows of 32, 64 or 128 bytes of
 * codes), cout <= 128, kvol <= 27.  Fewer than 64 channels cost what 64 do. */
SPCONVB_API int spconvb_fp4_conv_supported(int32_t cin, int32_t cout, int32_t kvol);

/* out[o] = act(alpha * sum_k W[:, k, :] . in[map[k * cap + o]] + bias), then the residual, for the min(*n_out_ptr, cap) rows that there
 * are, whatever launch_rows says (it only sizes the grid; 0: cap), as in spconvb_conv_forward: out, out_scales and res
 * hold cap rows.  An entry of the map that is not below in_rows is a missing neighbour. */
SPCONVB_API int spconvb_fp4_conv(const spconvb_fp4_params* p, const void* codes, const void* scales,
                                 const int32_t* map, uint32_t cap, const uint32_t* n_out_ptr,
                                 uint32_t launch_rows, const void* packed, const float* bias,
                                 void* out, uint32_t* status, void* stream);

#ifdef __cplusplus
}
#endif
#endif
