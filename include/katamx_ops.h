/*
 * katamx_ops.h — operators on device buffers, beside the net evaluation of katamx.h: what surrounds the attention of a transformer trunk
 * when its projections run in 8 bits. Each is one layer of the reference's transformer blocks (TransformerRMSNormLayer::apply,
 * eigenbackend.cpp:885-915; the projections of TransformerAttentionBlock / TransformerFFNBlock::apply, :1376-1718; applyRoPE, :1417-1456) in
 * a form of its own: on buffers that the caller owns, on the caller's stream.
 *
 * Conventions (those of katamx.h, and)
 *   - device: the HIP device that the pointers and the stream belong to; the calling thread's current device is left as it was.
 *   - stream: a hipStream_t of that device, NULL = its default stream. A call launches its kernels there and returns; it allocates nothing,
 *     keeps nothing and does not wait, so it may be captured into a graph, and calls on several threads and streams do not
 *     meet. Every call is deterministic: the same inputs give the same bits.
 *   - type: KMX_PREC_FP16, KMX_PREC_BF16 or KMX_PREC_FP32, the type of a tensor's elements. The last dimension is contiguous, the others
 *     have strides in ELEMENTS (of codes: bytes); input strides may be 0 (a broadcast). Offsets are 64-bit. Tensors need the alignment of their
 *     elements only, except where said.
 *   - e4m3: 8-bit floating point, 1 sign, 4 exponent, 3 mantissa bits, largest value 448, no infinities, 0x7f / 0xff are NaN.
 *   - arguments are checked before any device is touched: KMX_ERR_INVALID_ARG, and kmx_last_error() says which. Nothing is
 *     launched then. No rows (or tokens) is a valid call that does nothing.
 */
#ifndef KATAMX_OPS_H_
#define KATAMX_OPS_H_

#include "katamx.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KMX_OPS_VERSION 1
int kmx_ops_version(void);

/* How a row of e4m3 codes is scaled; value = code * scale.
 *   ROW: float[rows], scale = max(amax / 448, 2^-126) of the row, rounded to fp32 once the codes are made; 1 for a row of zeros
 *   MX:  uint8[rows][channels / 32], e8m0: 2^(code - 127) for 32 channels each, the smallest power of two (from 2^-127) that brings them
 *        to at most 448, 1 (code 127) where all are 0. channels is a multiple of 32.
 * A row (a block) that holds an infinity or a NaN has the scale NaN (code 255) and codes 0: it stays NaN in whatever it is multiplied with. */
enum { KMX_SCALES_NONE = 0, KMX_SCALES_ROW = 1, KMX_SCALES_MX = 2 };

/* RMS norm with the residual's addition in front and an 8-bit output behind:
 *   sum = x + residual (rounded to `type`; without a residual: x)
 *   y = sum / sqrt(mean over the channels of sum^2 + epsilon) * weight + beta;  0 on rows whose mask is 0
 *   codes, scales = y in e4m3 (of y before its own rounding to `type`)
 * x, residual, sum, y: [rows][channels]; residual and sum are both given or both NULL. weight, beta: float[channels] or NULL (1 and 0);
 * mask: float[rows] or NULL. y and codes may be NULL, not both; codes and scales are NULL with KMX_SCALES_NONE. sum and y may each be the very
 * tensor x or residual (same pointer and stride); no other output may overlap anything. The mean is good for all
 * finite values of the type, those whose squares leave fp32 included; a row of zeros with epsilon 0 is 0 / 0, NaN. */
typedef struct kmx_rmsnorm_args {
  int32_t type, scale_kind;
  int64_t rows;
  int32_t channels;
  float epsilon;
  const void* x;
  const void* residual;
  void* sum;
  const float* weight;
  const float* beta;
  const float* mask;
  void* y;
  void* codes;
  void* scales; /* contiguous; float* or uint8_t* */
  int64_t x_stride, residual_stride, sum_stride, y_stride, codes_stride;
} kmx_rmsnorm_args;
int kmx_rmsnorm(int device, void* stream, const kmx_rmsnorm_args* args);

/* codes, scales = x in e4m3 (weights once when they are loaded, activations that no norm precedes) */
int kmx_quantize(int device, void* stream, int type, int scale_kind, int64_t rows, int channels, const void* x, int64_t x_stride,
                 void* codes, int64_t codes_stride, void* scales);

/* out[m][n] = sum over k of a[m][k] w[n][k], both e4m3 with scales of one kind (ROW or MX, as the two calls above leave them), + bias[n];
 * a [rows][k], w [n][k], bias float[n] or NULL, out [rows][n] of out_type. k is a multiple of 16 (MX: of 32), a and w and their strides are
 * 16-byte aligned; n, k and the strides are below 2^23. With ROW scales, whatever their size, results leave fp32 on their way only
 * where they leave it themselves.
 * 16-bit outputs are summed on the 8-bit matrix instructions, whose sums of 8 products keep 13 bits below the largest of them: a result is off by up to
 * 7 * 2^-13 of the sum of its products' magnitudes. fp32 outputs are summed in fp32 throughout, MX values code * scale as bf16 numbers: exact for scales
 * from 2^-124 to 2^119 (codes 3 to 246); beyond these a value of 2^128 or more is infinite, one below 2^-133 is lost. */
typedef struct kmx_linear8_args {
  int32_t out_type, scale_kind;
  int64_t rows;
  int32_t n, k;
  const void* a;
  const void* a_scales;
  const void* w;
  const void* w_scales;
  const float* bias;
  void* out;
  int64_t a_stride, w_stride, out_stride;
} kmx_linear8_args;
int kmx_linear8(int device, void* stream, const kmx_linear8_args* args);

/* Rotary positions: for each token and head the pair p of channels - (2p, 2p + 1), or (p, p + pairs) with `half` - turned by
 *   angle = sum over the axes of position[axis] * frequencies[head][axis][p]
 *   (u, v) -> magnitude * (u cos - v sin, u sin + v cos); `inverse` negates the angle (times magnitude^2 = 1 that undoes it; it is also
 *   the turn's transpose: what a gradient goes through)
 * in fp64 up to the angle's fraction of a turn, so positions of millions lose nothing; fp32 tensors turn with sines and cosines good to their last bits,
 * 16-bit ones with such that are off by 2^-22 at most. Channels from 2 pairs on are copied.
 * q and k: [batch][seq][heads][head_dim] each, in and out; k_heads = 0: no k. out may be in itself (same pointer and strides), or a tensor that
 * overlaps nothing. positions: int32 or int64 [batch][seq][axes] by strides (0: the same for every sequence); frequencies: double
 * [freq_heads][axes][pairs], radians per position, contiguous, on the device. freq_heads is 1, or divides q_heads and k_heads: head h of H turns with
 * frequency head h / (H / freq_heads). axes is 1 or 2; 2 * pairs <= head_dim; batch * seq < 2^31. */
typedef struct kmx_rotary_tensor {
  const void* in;
  void* out;
  int64_t in_batch_stride, in_seq_stride, in_head_stride;
  int64_t out_batch_stride, out_seq_stride, out_head_stride;
} kmx_rotary_tensor;
typedef struct kmx_rotary_args {
  int32_t type, half, inverse;
  float magnitude;
  int64_t batch, seq;
  int32_t q_heads, k_heads, head_dim, pairs, axes, freq_heads;
  const double* frequencies;
  const void* positions;
  int32_t positions_are_64bit;
  int64_t pos_batch_stride, pos_seq_stride, pos_axis_stride;
  kmx_rotary_tensor q, k;
} kmx_rotary_args;
int kmx_rotary(int device, void* stream, const kmx_rotary_args* args);

#ifdef __cplusplus
}
#endif
#endif /* KATAMX_OPS_H_ */
