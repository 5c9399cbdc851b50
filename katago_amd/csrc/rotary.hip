// rotary.hip — rotary positions on device buffers (applyRoPE, eigenbackend.cpp:1417-1456, whose tables desc.cpp:1300-1363 builds for one board
// size): for pair p of a head at a token with position(s) m_a
//   angle = sum_a m_a f[head][a][p];   (u, v) -> magnitude (u cos - v sin, u sin + v cos), the sine negated for the inverse
// where (u, v) are channels (2p, 2p + 1) or (p, p + pairs); channels beyond 2 pairs are copied. Query head h turns with the frequencies of the key
// head it reads.
//
// Angles are formed in fp64 and as turns (1 = 2 pi): a position of a million times a frequency near 1 has no correct bit left of its phase in
// fp32; the turns' fraction is exact, and only then rounded. The rotation itself is fp32, rounded once.
//
// Bound by memory: 4 x 8191 tokens of 32 + 8 heads of 128 in bf16 123 us (5.4 TB/s; a large copy reaches 5.1), 256 boards of 12 + 6 heads of 32 in fp16
// with learned frequencies 44 us (4.8). Eight tokens take 3.7 us (3.0 in a graph), a launch and two trips to memory. Pairs that are no multiple of 4
// go one to a thread, in pieces of 2 bytes: the same long sequences with 46 pairs of 64 take 213 us.
#include "ops.h"
#include "ops_device.h"

namespace kmx {

namespace {

typedef _Float16 h16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 h16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 b16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 b16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x8u __attribute__((ext_vector_type(8), aligned(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
template <class T, int N> struct UnalignedV;
template <> struct UnalignedV<_Float16, 8> { typedef h16x8u V; };
template <> struct UnalignedV<_Float16, 4> { typedef h16x4u V; };
template <> struct UnalignedV<__bf16, 8> { typedef b16x8u V; };
template <> struct UnalignedV<__bf16, 4> { typedef b16x4u V; };
template <> struct UnalignedV<float, 8> { typedef f32x8u V; };
template <> struct UnalignedV<float, 4> { typedef f32x4u V; };

template <class T> struct UnalignedV<T, 1> { typedef T V __attribute__((ext_vector_type(1))); };

// Sine and cosine of 2 pi t, |t| <= 1/2.
// For 16-bit tensors by the instructions that take turns: over 2^27 values of t neither is off by more than 2.1 * 2^-24, and t's rounding moves the angle by
// 1.6 * 2^-24 at most: 2^-22 of a pair's size, a quarter of an fp16 rounding of a result 2^-9 of it.
__device__ __forceinline__ void sinCosOfTurnFast(float t, float* s, float* c) {
#if defined(__AMDGCN__)
  *s = __builtin_amdgcn_sinf(t);
  *c = __builtin_amdgcn_cosf(t);
#else
  *s = sinf(6.28318530717958647692f * t);
  *c = cosf(6.28318530717958647692f * t);
#endif
}
// For fp32 tensors each good to its last bits, next to 0 and to pi (where a sine is small beside t) as anywhere: what is left of t beyond whole quarters of a
// turn is at most pi / 4, exact in fp64 and rounded to fp32 there. The series end where the next term is below 2^-25 of the sum. (For every type: 8 tokens
// 3.05 -> 3.35 us, 256 boards with learned frequencies 35.4 -> 36.7; 4 x 8191 x 9 heads of 64 in fp32 24.0 -> 24.1.)
__device__ __forceinline__ void sinCosOfTurn(double t, float* s, float* c) {
  const double n = __builtin_rint(4.0 * t);
  const float x = (float)((t - 0.25 * n) * 6.28318530717958647692), z = x * x;
  const float sp = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f), z, 8.3333333e-3f), z, -1.6666667e-1f);
  const float cp = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f), z, -1.3888889e-3f), z, 4.1666667e-2f), z, -0.5f);
  const float sx = __builtin_fmaf(x * z, sp, x), cx = __builtin_fmaf(z, cp, 1.0f);
  const int q = (int)n;  // -2 .. 2
  const float a = q & 1 ? cx : sx, b = q & 1 ? sx : cx;
  *s = q & 2 ? -a : a;
  *c = (q + 1) & 2 ? -b : b;
}

struct RotaryLaunch {
  RotaryArgs a;
  int perFreq[2];          // heads of q and of k that turn with one set of frequencies
  int hpt, chunks;         // heads of one thread; such chunks of the perFreq[0] + perFreq[1] heads of a set
  int rotItems, copyItems; // pieces of a head: PV pairs each / 2 PV untouched channels each
  unsigned token0;
  unsigned threads;
};

// A thread owns PV pairs of a token in up to hpt heads of q and k that turn with the same frequencies: it forms their sines and cosines once and turns
// head after head, HB at a time so that several heads' loads are in flight. Channels that are only copied are pieces of the same size, of the same
// code (a lane's rotation is thrown away there). Threads of neighbouring pieces are neighbours: a head's row is read in consecutive pieces of 16
// bytes (16-bit types, PV = 8).
template <class TR, int PV, bool HALF>
__global__ __launch_bounds__(256) void rotaryKernel(RotaryLaunch r) {
  typedef typename TR::T T;
  constexpr int HB = 4;
  const RotaryArgs& a = r.a;
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  if(idx >= r.threads) return;
  const unsigned items = (unsigned)(r.rotItems + r.copyItems), groups = (unsigned)(a.freqHeads * r.chunks);
  const unsigned item = idx % items, rest = idx / items;
  const unsigned group = rest % groups, token = rest / groups + r.token0;
  const unsigned b = token / (unsigned)a.seq, s = token % (unsigned)a.seq;
  const int fh = (int)(group / (unsigned)r.chunks), first = (int)(group % (unsigned)r.chunks) * r.hpt;
  const int all = r.perFreq[0] + r.perFreq[1], end = first + r.hpt < all ? first + r.hpt : all;  // of this set's heads: q's, then k's
  const T* const in[2] = {(const T*)a.side[0].in + b * a.side[0].inBatch + s * a.side[0].inToken + (int64_t)fh * r.perFreq[0] * a.side[0].inHead,
                          (const T*)a.side[1].in + b * a.side[1].inBatch + s * a.side[1].inToken + (int64_t)fh * r.perFreq[1] * a.side[1].inHead};
  T* const out[2] = {(T*)a.side[0].out + b * a.side[0].outBatch + s * a.side[0].outToken + (int64_t)fh * r.perFreq[0] * a.side[0].outHead,
                     (T*)a.side[1].out + b * a.side[1].outBatch + s * a.side[1].outToken + (int64_t)fh * r.perFreq[1] * a.side[1].outHead};
  auto inOf = [&](int h) { return h < r.perFreq[0] ? in[0] + h * a.side[0].inHead : in[1] + (h - r.perFreq[0]) * a.side[1].inHead; };
  auto outOf = [&](int h) { return h < r.perFreq[0] ? out[0] + h * a.side[0].outHead : out[1] + (h - r.perFreq[0]) * a.side[1].outHead; };

  const bool copied = item >= (unsigned)r.rotItems;
  const int c = 2 * a.pairs + (int)(item - (unsigned)r.rotItems) * 2 * PV;  // of a copied piece
  if(copied && c + 2 * PV > a.headDim) {  // the last channels of a head, fewer than a piece
    for(int h = first; h < end; h++) {
      const T* const ip = inOf(h);
      T* const op = outOf(h);
      for(int i = c; i < a.headDim; i++) op[i] = ip[i];
    }
    return;
  }
  const int p0 = copied ? 0 : (int)item * PV;  // pairs is a multiple of PV
  const int at0 = copied ? c : HALF ? p0 : 2 * p0, at1 = copied || !HALF ? at0 + PV : p0 + a.pairs;

  typedef typename UnalignedV<T, PV>::V V;
  V u[HB], v[HB];  // channels at0 + [0, PV) and at1 + [0, PV) of a head
  auto fetch = [&](int hb) {
#pragma unroll
    for(int j = 0; j < HB; j++) {
      if(hb + j >= end) break;
      const T* const ip = inOf(hb + j);
      u[j] = *(const V*)(ip + at0);
      v[j] = *(const V*)(ip + at1);
    }
  };
  double pos[2] = {0.0, 0.0};
  for(int ax = 0; ax < a.axes; ax++) {
    const int64_t at = b * a.posBatch + s * a.posToken + ax * a.posAxis;
    pos[ax] = a.pos64 ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
  }
  const double* const f = a.freqs + (size_t)fh * a.axes * a.pairs + p0;
  // Positions and frequencies are requested ahead of the heads: a wave's loads return in order, so the sines are formed while the heads are
  // still on their way (behind them: 92416 tokens with learned frequencies 62 us, 49 so)
  double f0[PV], f1[PV];
#pragma unroll
  for(int i = 0; i < PV; i++) f0[i] = f[i];
  if(a.axes == 2) {
#pragma unroll
    for(int i = 0; i < PV; i++) f1[i] = f[a.pairs + i];
  }
  __builtin_amdgcn_sched_barrier(0);
  fetch(first);
  __builtin_amdgcn_sched_barrier(0);
  float cs[PV], sn[PV];
#pragma unroll
  for(int i = 0; i < PV; i++) {
    double t = pos[0] * f0[i];
    if(a.axes == 2) t += pos[1] * f1[i];
    t *= 0.15915494309189533577;  // 1 / 2 pi
    t -= __builtin_rint(t);
    float sv, cv;
    if constexpr(sizeof(T) == 4) sinCosOfTurn(t, &sv, &cv);
    else sinCosOfTurnFast((float)t, &sv, &cv);
    cs[i] = cv * a.magnitude;
    sn[i] = (a.inverse ? -sv : sv) * a.magnitude;
  }

  for(int hb = first; hb < end; hb += HB) {
    if(hb != first) fetch(hb);
#pragma unroll
    for(int j = 0; j < HB; j++) {
      if(hb + j >= end) break;
      V x, y;
#pragma unroll
      for(int i = 0; i < PV; i++) {  // pair i: HALF (u[i], v[i]), else neighbours of u and v in a row
        const float m = TR::toFloat(HALF ? u[j][i] : 2 * i < PV ? u[j][(2 * i) % PV] : v[j][(2 * i) % PV]);
        const float n = TR::toFloat(HALF ? v[j][i] : 2 * i + 1 < PV ? u[j][(2 * i + 1) % PV] : v[j][(2 * i + 1) % PV]);
        const T p = TR::fromFloat(m * cs[i] - n * sn[i]), q = TR::fromFloat(m * sn[i] + n * cs[i]);
        if(HALF) {
          x[i] = p;
          y[i] = q;
        }
        else {
          if(2 * i < PV) x[(2 * i) % PV] = p;
          else y[(2 * i) % PV] = p;
          if(2 * i + 1 < PV) x[(2 * i + 1) % PV] = q;
          else y[(2 * i + 1) % PV] = q;
        }
      }
      T* const op = outOf(hb + j);
      *(V*)(op + at0) = copied ? u[j] : x;
      *(V*)(op + at1) = copied ? v[j] : y;
    }
  }
}

template <class TR, int PV, bool HALF>
hipError_t launchPieces(const RotaryArgs& a, hipStream_t stream) {
  RotaryLaunch r;
  r.a = a;
  for(int i = 0; i < 2; i++) r.perFreq[i] = a.side[i].heads / a.freqHeads;
  r.rotItems = a.pairs / PV;
  const bool copies = a.side[0].in != a.side[0].out || (a.side[1].heads > 0 && a.side[1].in != a.side[1].out);
  r.copyItems = copies ? (a.headDim - 2 * a.pairs + 2 * PV - 1) / (2 * PV) : 0;
  const int items = r.rotItems + r.copyItems, all = r.perFreq[0] + r.perFreq[1];
  // Few tokens: one head a thread, all loads of the call in flight at once (8 tokens, 32 + 8 heads of 128: 5.6 us with 8 heads a thread). Many: 8
  // heads share a thread's sines and cosines, once there are threads enough to fill the chip.
  r.hpt = 8;
  while(r.hpt > 1 && a.tokens * items * a.freqHeads * ((all + r.hpt - 1) / r.hpt) < 256 * 1024) r.hpt /= 2;
  r.chunks = (all + r.hpt - 1) / r.hpt;
  r.hpt = (all + r.chunks - 1) / r.chunks;  // evenly
  const int64_t perToken = (int64_t)items * a.freqHeads * r.chunks;
  const int64_t most = (int64_t)0x7fffffff / perToken;  // tokens of one launch: its threads are counted in 31 bits
  for(int64_t t0 = 0; t0 < a.tokens; t0 += most) {
    const int64_t n = a.tokens - t0 < most ? a.tokens - t0 : most;
    r.token0 = (unsigned)t0;
    r.threads = (unsigned)(n * perToken);
    const hipError_t e = launchKernel(rotaryKernel<TR, PV, HALF>, dim3((r.threads + 255) / 256), dim3(256), 0, stream, r);
    if(e != hipSuccess) return e;
  }
  return hipSuccess;
}
template <class TR>
hipError_t launchType(const RotaryArgs& a, hipStream_t stream) {
  // pieces of 16 bytes: 8 pairs of a 16-bit type, 4 of fp32 (8 of fp32 take 184 registers: 4 x 8191 x 9 heads of 64 in 34 us against 28)
  if constexpr(sizeof(typename TR::T) == 2)
    if(a.pairs % 8 == 0) return a.half ? launchPieces<TR, 8, true>(a, stream) : launchPieces<TR, 8, false>(a, stream);
  if(a.pairs % 4 == 0) return a.half ? launchPieces<TR, 4, true>(a, stream) : launchPieces<TR, 4, false>(a, stream);
  return a.half ? launchPieces<TR, 1, true>(a, stream) : launchPieces<TR, 1, false>(a, stream);
}

}  // namespace

hipError_t launchRotary(int dtype, const RotaryArgs& a, hipStream_t stream) {
  if(a.tokens == 0) return hipSuccess;
  if(dtype == DT_F16) return launchType<TraitsF16>(a, stream);
  if(dtype == DT_BF16) return launchType<TraitsBF16>(a, stream);
  if(dtype == DT_F32) return launchType<TraitsF32>(a, stream);
  return hipErrorInvalidValue;
}

}  // namespace kmx
