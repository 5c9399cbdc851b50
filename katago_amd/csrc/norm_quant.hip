// norm_quant.hip — RMS norm of rows with the residual's addition in front and e4m3 with scales behind (TransformerRMSNormLayer::apply,
// eigenbackend.cpp:885-915, between two sublayers of a transformer trunk whose projections read 8 bits), and the 8-bit form alone.
//
//   h_c = T(x_c + r_c)        rounded to the stream's type, because the stream is what the next sublayer adds to: the norm is of what is stored
//   y_c = h_c * (sum_c h_c^2 / C + eps)^(-1/2) * w_c + beta_c;  0 on rows whose mask is 0
//   SCALES_ROW  s = max(max_c |y_c| / 448, 2^-126), 1 where y is all 0;                  code_c = e4m3(y_c / s)
//   SCALES_MX   s = 2^k with the smallest k >= -127 for which max |y| / s <= 448 over 32 channels, 1 where they are all 0
//   A row (a block of 32) that holds an infinity or a NaN gets the scale NaN and codes 0.
// Everything between the loads and the stores is fp32; the sum of squares is fp64 where fp32's is not good enough. e4m3 rounds to nearest even.
//
// Bound by memory: a row's values stay in registers, so that everything is read once and written once. 92416 rows of 384 channels in fp16 with residual,
// mask and codes 52 us (4.8 TB/s; a large copy reaches 5.1), 8190 of 4096 in bf16 with sum, y and codes for 32 channels each 55 us (5.5), the
// 8-bit form alone of 16383 x 1536 17 us (4.4). A few rows are bound by one trip to memory and a launch: 361 x 384 4.2 us (3.6 in a graph).
// With operands that the last call left in the caches: 92416 x 384 44 us, in fp32 84 (8190 x 4096 in fp32 78), 92416 x 383 57.
#include "ops.h"
#include "ops_device.h"

namespace kmx {

namespace {

// Vectors at element alignment: rows of any length start anywhere. gfx950 serves unaligned 16-byte accesses; aligned ones cost the same as with
// an aligned type (eight sizes, within 0.3 %), rows at odd addresses about a tenth more (92416 x 384 at a stride of 387 48.5 us against 44.3).
typedef _Float16 h16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 b16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef float f32x8u __attribute__((ext_vector_type(8), aligned(4)));
typedef unsigned u32x2u __attribute__((ext_vector_type(2), aligned(1)));
template <class T> struct Unaligned8;
template <> struct Unaligned8<_Float16> { typedef h16x8u V; };
template <> struct Unaligned8<__bf16> { typedef b16x8u V; };
template <> struct Unaligned8<float> { typedef f32x8u V; };

__device__ __forceinline__ unsigned bitsOf(float x) { return __builtin_bit_cast(unsigned, x); }
__device__ __forceinline__ float floatOf(unsigned x) { return __builtin_bit_cast(float, x); }

// 8 elements from c on as fp32; those at or beyond C are 0
template <class TR>
__device__ __forceinline__ void load8(const typename TR::T* p, int c, int C, float (&v)[8]) {
  if(c + 8 <= C) {
    const typename Unaligned8<typename TR::T>::V t = *(const typename Unaligned8<typename TR::T>::V*)(p + c);
#pragma unroll
    for(int i = 0; i < 8; i++) v[i] = TR::toFloat(t[i]);
  }
  else {
#pragma unroll
    for(int i = 0; i < 8; i++) v[i] = c + i < C ? TR::toFloat(p[c + i]) : 0.0f;
  }
}
template <class TR, bool STREAM = false>
__device__ __forceinline__ void store8(typename TR::T* p, int c, int C, const float (&v)[8]) {
  if(c + 8 <= C) {
    typename Unaligned8<typename TR::T>::V t;
#pragma unroll
    for(int i = 0; i < 8; i++) t[i] = TR::fromFloat(v[i]);
    if(STREAM) __builtin_nontemporal_store(t, (typename Unaligned8<typename TR::T>::V*)(p + c));
    else *(typename Unaligned8<typename TR::T>::V*)(p + c) = t;
  }
  else {
#pragma unroll
    for(int i = 0; i < 8; i++)
      if(c + i < C) p[c + i] = TR::fromFloat(v[i]);
  }
}
// What a row's or a block's values are divided by: a power of two (EXACT), whose reciprocal is exact; or largest magnitude / 448 to twice fp32's bits: scale is
// that rounded, rest what is left, inv = 1 / scale. A product with inv alone would be off by up to two roundings, and scale by one more, which puts
// values at the border of two codes on the other side (10700 of 25.2 million bf16 values; with the quotient by scale 1100; so none). A step on what the
// product leaves makes it the formula's quotient, rounded once. (16383 x 1536 15.8 -> 16.4 us, 92416 x 384 43.3 -> 44.3.)
struct Divisor {
  float scale, rest, inv;
};
template <bool EXACT>
__device__ __forceinline__ float dividedBy(float v, Divisor d) {
  const float q = v * d.inv;
  return EXACT ? q : __builtin_fmaf(__builtin_fmaf(-q, d.rest, __builtin_fmaf(-q, d.scale, v)), d.inv, q);
}
// (a quotient may lie a rounding beyond 448)
template <bool EXACT>
__device__ __forceinline__ void storeCodes8(uint8_t* p, int c, int C, const float (&v)[8], Divisor d) {
  float u[8];
#pragma unroll
  for(int i = 0; i < 8; i++) u[i] = __builtin_fminf(__builtin_fmaxf(dividedBy<EXACT>(v[i], d), -E4M3_MAX), E4M3_MAX);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[4], u[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[6], u[7], hi, true);
  if(c + 8 <= C) {
    u32x2u t;
    t[0] = (unsigned)lo;
    t[1] = (unsigned)hi;
    *(u32x2u*)(p + c) = t;
  }
  else {
#pragma unroll
    for(int i = 0; i < 8; i++)
      if(c + i < C) p[c + i] = (uint8_t)((unsigned)(i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}

// |v| as bits: as unsigned numbers they are ordered as the values are, infinities and NaNs above all finite ones
__device__ __forceinline__ unsigned maxBits(const float (&v)[8]) {
  unsigned m = 0;
#pragma unroll
  for(int i = 0; i < 8; i++) {
    const unsigned b = bitsOf(v[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  return m;
}
__device__ __forceinline__ unsigned shflXorBits(unsigned v, int mask) { return bitsOf(__shfl_xor(floatOf(v), mask)); }

// The row's scale and what its values are divided by, from the bits of its largest magnitude (a spoilt row's values are zeros by then: by 1)
__device__ __forceinline__ bool spoilt(unsigned top) { return top >= 0x7f800000u; }
__device__ __forceinline__ void rowScale(unsigned top, float& scale, Divisor& d) {
  float rest = 0.0f;
  scale = 1.0f;
  if(!spoilt(top) && top != 0) {
    scale = floatOf(top) / E4M3_MAX;
    rest = __builtin_fmaf(-scale, E4M3_MAX, floatOf(top)) / E4M3_MAX;
    if(scale < 1.17549435e-38f) {
      scale = 1.17549435e-38f;
      rest = 0.0f;
    }
  }
  d = Divisor{scale, rest, 1.0f / scale};
  if(spoilt(top)) scale = floatOf(0x7fc00000u);
}
// ... and a block's e8m0 code: top = (1 + m) 2^(e - 127), 448 = 1.75 * 2^8, so k = e - 127 - 8, one more where 1 + m > 1.75
__device__ __forceinline__ void mxScale(unsigned top, unsigned& code, float& inv) {
  if(top >= 0x7f800000u) {
    code = 255;
    inv = 0.0f;
  }
  else if(top == 0) {
    code = 127;
    inv = 1.0f;
  }
  else {
    const int k = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);  // + 127
    code = k < 0 ? 0 : (unsigned)k;
    inv = floatOf((254u - code) << 23);  // 2^(127 - code); code <= 247
  }
}
// v with the infinities and NaNs of a spoilt row replaced, so that 0 * v is 0
__device__ __forceinline__ void zeroIf(bool spoilt, float (&v)[8]) {
  if(!spoilt) return;
#pragma unroll
  for(int i = 0; i < 8; i++) v[i] = 0.0f;
}

// Sum / largest over the TPR threads of a row; up to a wave through lane exchanges, beyond it through LDS. The order is fixed: the same
// inputs give the same bits.
__device__ __forceinline__ float laneXor(float v, int mask) { return __shfl_xor(v, mask); }
__device__ __forceinline__ double laneXor(double v, int mask) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)shflXorBits((unsigned)(b >> 32), mask) << 32 | shflXorBits((unsigned)b, mask));
}
template <int TPR, class S>
__device__ __forceinline__ S rowSum(S v, S* part) {
#pragma unroll
  for(int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) v += laneXor(v, o);
  if constexpr(TPR > 64) {
    if((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for(int w = 0; w < TPR / 64; w++) v += part[w];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ unsigned rowMax(unsigned v, unsigned* part) {
#pragma unroll
  for(int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) {
    const unsigned u = shflXorBits(v, o);
    v = u > v ? u : v;
  }
  if constexpr(TPR > 64) {
    if((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for(int w = 0; w < TPR / 64; w++) v = part[w] > v ? part[w] : v;
  }
  return v;
}

__device__ __forceinline__ void addSquares(double& ss, const float (&v)[8]) {
#pragma unroll
  for(int j = 0; j < 8; j++) ss = __builtin_fma((double)v[j], (double)v[j], ss);
}
// The mean of the squares + eps. fp32's sum of squares is good while that is within these bounds: below 2^-96 squares lose bits among the subnormals, above 2^126
// their sum overflows (a NaN is outside).
__device__ __forceinline__ double meanOf(const NormQuantArgs& a, double sum) { return sum * a.perChannel + (double)a.eps; }
__device__ __forceinline__ bool ordinary(double mean) { return mean >= 0x1p-96 && mean <= 0x1p126; }
// mean^(-1/2) in two parts: fp32's own error in it (up to 2^-23) would be the row's in every channel and move codes and scales that lie next to a border.
// One Newton step on what is left of 1 - x r^2. Where the root or its second part would leave fp32, the row's values are multiplied with `pre` first: 2^100
// for means below 2^-96 (a subnormal value is then at least 2^-49), 2^-64 above 2^126 (what loses bits by it is below 2^-125 in the result). A row of zeros
// without eps gives infinity, one with an infinity 0, both without a second part.
struct Factor {
  float hi, lo, pre;
};
__device__ __forceinline__ Factor factorOf(double x) {
  float pre = 1.0f;
  if(x < 0x1p-96) {
    x *= 0x1p200;
    pre = 0x1p100f;
  }
  if(x > 0x1p126) {
    x *= 0x1p-128;
    pre = 0x1p-64f;
  }
  const float xh = (float)x, xl = (float)(x - (double)xh), r = rsqrtf(xh);
  const float t = xh * r, left = __builtin_fmaf(-t, r, 1.0f) - (__builtin_fmaf(xh, r, -t) + xl * r) * r, lo = 0.5f * r * left;
  return Factor{r, __builtin_fabsf(lo) < r * 1e-3f ? lo : 0.0f, pre};
}
// The norm's factor applied to 8 values: v * r * w, rounded once, + beta; 0 on a masked row. (Of 35.5 million codes 8 lie on the other side of a border than
// the formula's in 64 bits; 16 with fp32's root, each product and the scale rounded. 256 boards take 1.3 us longer for it.)
__device__ __forceinline__ void scale8(const NormQuantArgs& a, int c, Factor r, bool on, float (&v)[8]) {
  if(!a.normed) return;
  float w[8];
  if(a.weight != nullptr) load8<TraitsF32>(a.weight, c, a.C, w);
  if(__builtin_expect(r.pre != 1.0f, 0)) {
#pragma unroll
    for(int i = 0; i < 8; i++) v[i] *= r.pre;
  }
#pragma unroll
  for(int i = 0; i < 8; i++) {
    const float p = v[i] * r.hi, e = __builtin_fmaf(v[i], r.lo, __builtin_fmaf(v[i], r.hi, -p));
    v[i] = a.weight != nullptr ? __builtin_fmaf(p, w[i], e * w[i]) : p + e;
  }
  if(a.beta != nullptr) {
    load8<TraitsF32>(a.beta, c, a.C, w);
#pragma unroll
    for(int i = 0; i < 8; i++) v[i] += w[i];
  }
  zeroIf(!on, v);
}
// x + residual of 8 channels, rounded to the stream's type and stored (STREAM: past the caches, which the codes and y, that are read next, then have to
// themselves: 256 boards 56.9 -> 55.6 us, and what multiplies the codes 2 us less)
template <class TR, bool STREAM>
__device__ __forceinline__ void stream8(const NormQuantArgs& a, int64_t row, int c, float (&v)[8]) {
  typedef typename TR::T T;
  load8<TR>((const T*)a.x + row * a.xStride, c, a.C, v);
  if(a.residual == nullptr) return;
  float r[8];
  load8<TR>((const T*)a.residual + row * a.residualStride, c, a.C, r);
#pragma unroll
  for(int i = 0; i < 8; i++) v[i] = TR::toFloat(TR::fromFloat(v[i] + r[i]));
  store8<TR, STREAM>((T*)a.sum + row * a.sumStride, c, a.C, v);
}
// 8-bit output of 8 channels whose block of 32 lies in four neighbouring lanes
__device__ __forceinline__ void mx8(const NormQuantArgs& a, int64_t row, int c, bool in, float (&v)[8]) {
  unsigned top = maxBits(v), u = shflXorBits(top, 1);
  top = u > top ? u : top;
  u = shflXorBits(top, 2);
  top = u > top ? u : top;
  unsigned code;
  Divisor d = {1.0f, 0.0f, 1.0f};
  mxScale(top, code, d.inv);
  zeroIf(code == 255, v);
  if(!in) return;
  storeCodes8<true>(a.codes + row * a.codesStride, c, a.C, v, d);
  if((c & (MX_BLOCK - 1)) == 0) ((uint8_t*)a.scales)[row * (a.C / MX_BLOCK) + c / MX_BLOCK] = (uint8_t)code;
}

// A row on TPR threads, its values in registers: 8 consecutive channels a thread and round, NCH rounds. x and residual are read once, everything
// else is written once. (Of 1024 threads a CU holds two work-groups, if a thread has 64 registers; fp32 has 80 at four pieces.)
template <class TR, int TPR, int NCH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256, TPR == 1024 && sizeof(typename TR::T) == 2 ? 8 : 1) void normQuantKernel(NormQuantArgs a) {
  constexpr int BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
  __shared__ float part[2][TPR > 64 ? TPR / 64 : 1];
  __shared__ double partWide[TPR > 64 ? TPR / 64 : 1];
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  const bool valid = row < a.rows;  // (lanes without a row stay for the exchanges)
  float v[NCH][8];
  float ss = 0.0f;
#pragma unroll
  for(int i = 0; i < NCH; i++) {
    const int c = (t + i * TPR) * 8;
    if(valid && c < a.C) stream8<TR, (NCH > 1)>(a, row, c, v[i]);
    else zeroIf(true, v[i]);
#pragma unroll
    for(int j = 0; j < 8; j++) ss += v[i][j] * v[i][j];
  }
  Factor r = {1.0f, 0.0f, 1.0f};
  if(a.normed) {
    double mean = meanOf(a, rowSum<TPR>(ss, part[0]));
    if(__builtin_expect(anyLane(!ordinary(mean)), 0)) {  // such rows again in fp64 (for every row 92416 of 384 channels take 4.6 us longer)
      double wide = 0.0;
#pragma unroll
      for(int i = 0; i < NCH; i++) addSquares(wide, v[i]);
      wide = rowSum<TPR>(wide, partWide);  // (rows of more than a wave: one to a work-group, all of it is here)
      if(!ordinary(mean)) mean = meanOf(a, wide);
    }
    r = factorOf(mean);
  }
  const bool on = a.mask == nullptr || !valid || a.mask[row] != 0.0f;
  unsigned top = 0;
#pragma unroll
  for(int i = 0; i < NCH; i++) {
    const int c = (t + i * TPR) * 8;
    if(valid && c < a.C) {
      scale8(a, c, r, on, v[i]);
      if(a.y != nullptr) store8<TR>((typename TR::T*)a.y + row * a.yStride, c, a.C, v[i]);
    }
    if(a.scaleKind == SCALES_ROW) {
      const unsigned m = maxBits(v[i]);
      top = m > top ? m : top;
    }
  }
  if(a.scaleKind == SCALES_ROW) {
    top = rowMax<TPR>(top, (unsigned*)part[1]);
    float scale;
    Divisor d;
    rowScale(top, scale, d);
#pragma unroll
    for(int i = 0; i < NCH; i++) {
      const int c = (t + i * TPR) * 8;
      if(!valid || c >= a.C) continue;
      zeroIf(spoilt(top), v[i]);
      storeCodes8<false>(a.codes + row * a.codesStride, c, a.C, v[i], d);
    }
    if(valid && t == 0) ((float*)a.scales)[row] = scale;
  }
  else if(a.scaleKind == SCALES_MX) {
#pragma unroll
    for(int i = 0; i < NCH; i++) {
      const int c = (t + i * TPR) * 8;
      mx8(a, row, c, valid && c < a.C, v[i]);
    }
  }
}

// Rows longer than the registers hold: a work-group of 1024 walks the row up to three times (sum of squares, largest magnitude, outputs); after the
// first walk it reads what it wrote itself. Rows are long enough here that later walks mostly hit the caches.
template <class TR>
__global__ __launch_bounds__(1024) void normQuantLongKernel(NormQuantArgs a) {
  typedef typename TR::T T;
  constexpr int TPR = 1024;
  __shared__ double part[TPR / 64];
  __shared__ unsigned partTop[TPR / 64];
  const int64_t row = blockIdx.x;
  const T* const h = a.residual != nullptr ? (const T*)a.sum + row * a.sumStride : (const T*)a.x + row * a.xStride;
  float v[8];
  Factor r = {1.0f, 0.0f, 1.0f};
  if(a.normed) {
    double ss = 0.0;  // (a lane's terms are many: in fp32 2^24 channels of one value are 920 roundings off)
    for(int c = threadIdx.x * 8; c < a.C; c += TPR * 8) {
      stream8<TR, false>(a, row, c, v);
      addSquares(ss, v);
    }
    r = factorOf(meanOf(a, rowSum<TPR>(ss, part)));
  }
  const bool on = a.mask == nullptr || a.mask[row] != 0.0f;
  Divisor d = {1.0f, 0.0f, 1.0f};
  unsigned top = 0;
  if(a.scaleKind == SCALES_ROW) {
    for(int c = threadIdx.x * 8; c < a.C; c += TPR * 8) {
      load8<TR>(h, c, a.C, v);
      scale8(a, c, r, on, v);
      const unsigned m = maxBits(v);
      top = m > top ? m : top;
    }
    top = rowMax<TPR>(top, partTop);
    float scale;
    rowScale(top, scale, d);
    if(threadIdx.x == 0) ((float*)a.scales)[row] = scale;
  }
  for(int c0 = 0; c0 < a.C; c0 += TPR * 8) {  // (all lanes take part in a block's exchanges)
    const int c = c0 + threadIdx.x * 8;
    const bool in = c < a.C;
    zeroIf(true, v);
    if(in) {
      load8<TR>(h, c, a.C, v);
      scale8(a, c, r, on, v);
      if(a.y != nullptr) store8<TR>((T*)a.y + row * a.yStride, c, a.C, v);
    }
    if(a.scaleKind == SCALES_ROW && in) {
      zeroIf(spoilt(top), v);
      storeCodes8<false>(a.codes + row * a.codesStride, c, a.C, v, d);
    }
    else if(a.scaleKind == SCALES_MX) mx8(a, row, c, in, v);
  }
}

// A launch's threads are counted in 32 bits: more rows than that go in several launches
template <class TR>
NormQuantArgs rowsFrom(const NormQuantArgs& a, int64_t first, int64_t most) {
  typedef typename TR::T T;
  NormQuantArgs b = a;
  b.rows = a.rows - first < most ? a.rows - first : most;
  b.x = (const T*)a.x + first * a.xStride;
  if(a.residual != nullptr) b.residual = (const T*)a.residual + first * a.residualStride;
  if(a.sum != nullptr) b.sum = (T*)a.sum + first * a.sumStride;
  if(a.y != nullptr) b.y = (T*)a.y + first * a.yStride;
  if(a.mask != nullptr) b.mask = a.mask + first;
  if(a.codes != nullptr) b.codes = a.codes + first * a.codesStride;
  if(a.scaleKind == SCALES_ROW) b.scales = (float*)a.scales + first;
  if(a.scaleKind == SCALES_MX) b.scales = (uint8_t*)a.scales + first * (a.C / MX_BLOCK);
  return b;
}
template <class TR, int TPR, int NCH>
hipError_t launchRows(const NormQuantArgs& a, hipStream_t stream) {
  constexpr int BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
  constexpr int64_t MOST = (int64_t)0x7fffffff / BLOCK * RPB;
  for(int64_t first = 0; first < a.rows; first += MOST) {
    const NormQuantArgs b = rowsFrom<TR>(a, first, MOST);
    hipError_t e;
    if constexpr(NCH > 0) e = launchKernel(normQuantKernel<TR, TPR, NCH>, dim3((unsigned)((b.rows + RPB - 1) / RPB)), dim3(BLOCK), 0, stream, b);
    else e = launchKernel(normQuantLongKernel<TR>, dim3((unsigned)b.rows), dim3(BLOCK), 0, stream, b);
    if(e != hipSuccess) return e;
  }
  return hipSuccess;
}
template <class TR>
hipError_t launchOne(const NormQuantArgs& a, hipStream_t stream) {
  const int pieces = (a.C + 7) / 8;
  // While the chip has a lane for every piece (1024 to a CU), each lane takes one: the call is one trip to memory and the row's exchanges, and
  // a lane's rounds would only add to it (361 rows of 384 channels 5.2 -> 3.3 us, of 2048 6.3 -> 3.8, one row of 8192 5.9 -> 3.9). More rows are
  // faster on fewer lanes with several pieces each in flight (92416 rows of 384 42.7 us against 52, operands in the caches).
  auto laneEach = [&](int lanes) { return a.rows * lanes <= 256 * 1024; };
  if(pieces <= 16) return launchRows<TR, 16, 1>(a, stream);
  if(pieces <= 64 && laneEach(64)) return launchRows<TR, 64, 1>(a, stream);
  if(pieces <= 32) return launchRows<TR, 16, 2>(a, stream);
  if(pieces <= 64) return launchRows<TR, 16, 4>(a, stream);
  if(pieces <= 128) return launchRows<TR, 64, 2>(a, stream);
  if(pieces <= 256) return laneEach(256) ? launchRows<TR, 256, 1>(a, stream) : launchRows<TR, 64, 4>(a, stream);
  if(pieces <= 512) return laneEach(512) ? launchRows<TR, 512, 1>(a, stream) : launchRows<TR, 256, 2>(a, stream);
  if(pieces <= 1024) return laneEach(1024) ? launchRows<TR, 1024, 1>(a, stream) : launchRows<TR, 256, 4>(a, stream);
  if(pieces <= 4096) return launchRows<TR, 1024, 4>(a, stream);
  return launchRows<TR, 1024, 0>(a, stream);  // (0: any length)
}

}  // namespace

hipError_t launchNormQuant(int dtype, const NormQuantArgs& a, hipStream_t stream) {
  if(a.rows == 0) return hipSuccess;
  if(dtype == DT_F16) return launchOne<TraitsF16>(a, stream);
  if(dtype == DT_BF16) return launchOne<TraitsBF16>(a, stream);
  if(dtype == DT_F32) return launchOne<TraitsF32>(a, stream);
  return hipErrorInvalidValue;
}

}  // namespace kmx
