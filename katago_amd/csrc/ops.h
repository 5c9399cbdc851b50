// ops.h — launch interface of the operators on device buffers (ops_api.cpp): RMS norm with the residual's addition and an 8-bit
// output (norm_quant.hip), the product of two 8-bit matrices (linear8.hip) and rotary positions (rotary.hip). Strides are in elements.
// The callers have checked every argument; a launcher only picks a kernel.
#ifndef KMX_OPS_H_
#define KMX_OPS_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kmx {

enum { SCALES_NONE = 0, SCALES_ROW = 1, SCALES_MX = 2 };  // = KMX_SCALES_* of katamx_ops.h
constexpr int MX_BLOCK = 32;                              // channels that share an e8m0 scale
constexpr float E4M3_MAX = 448.0f;

struct NormQuantArgs {
  const void* x;         // T[rows][C]
  const void* residual;  // T[rows][C] or null
  void* sum;             // T[rows][C]: x + residual (with a residual; may be x or residual themselves)
  const float* weight;   // [C] or null (1)
  const float* beta;     // [C] or null (0)
  const float* mask;     // [rows] or null: 0 = the row's results are 0
  void* y;               // T[rows][C] or null (may be x or residual themselves)
  uint8_t* codes;        // e4m3 [rows][C] or null
  void* scales;          // SCALES_ROW: float[rows]; SCALES_MX: e8m0 [rows][C / 32]
  int64_t xStride, residualStride, sumStride, yStride, codesStride;
  int64_t rows;
  int C;
  int scaleKind;
  int normed;  // 0: the 8-bit form of x alone
  float eps;
  double perChannel;  // 1 / C
};
hipError_t launchNormQuant(int dtype, const NormQuantArgs& a, hipStream_t stream);

struct Linear8Args {
  const uint8_t* a;       // e4m3 [rows][K]
  const uint8_t* w;       // e4m3 [N][K]
  const void* aScales;    // SCALES_ROW: float[rows] / float[N]; SCALES_MX: e8m0 [rows][K / 32] / [N][K / 32]
  const void* wScales;
  const float* bias;      // [N] or null
  void* out;              // TO[rows][N]
  int64_t aStride, wStride, outStride;
  int64_t rows;
  int N, K;               // K: a multiple of 16 (SCALES_MX: of 32); strides of a and w multiples of 16, pointers 16-byte aligned
  int scaleKind;
};
hipError_t launchLinear8(int outType, const Linear8Args& a, hipStream_t stream);

struct RotarySide {  // q or k
  const void* in;
  void* out;
  int64_t inBatch, inToken, inHead, outBatch, outToken, outHead;
  int heads;
};
struct RotaryArgs {
  RotarySide side[2];    // q, k (heads = 0: absent)
  const void* positions;  // int32 or int64
  int64_t posBatch, posToken, posAxis;
  int pos64;
  const double* freqs;   // [freqHeads][axes][pairs], radians per position
  int freqHeads, axes, pairs, headDim;
  int seq;
  int64_t tokens;        // batch * seq, below 2^31
  float magnitude;
  int inverse, half;     // half: pair p is channels (p, p + pairs); else (2p, 2p + 1)
};
hipError_t launchRotary(int dtype, const RotaryArgs& a, hipStream_t stream);

}  // namespace kmx
#endif
