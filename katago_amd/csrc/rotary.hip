// rotary.hip — rotary positions on device buffers (applyRoPE, eigenbackend.cpp:1417-1456, whose tables desc.cpp:1300-1363 builds for one board
// size): for pair p of a head at a token with position(s) m_a
//   angle = sum_a m_a f[head][a][p];   (u, v) -> magnitude (u cos - v sin, u sin + v cos), the sine negated for the inverse
// where (u, v) are channels (2p, 2p + 1) or (p, p + pairs); channels beyond 2 pairs are copied. Query head h turns with the frequencies of the key
// head it reads.
//
// Angles are formed in fp64 and as turns (1 = 2 pi): a position of a million times a frequency near 1 has no correct bit left of its phase in
// fp32; the turns' fraction is exact, and only then rounded to fp32. The rotation itself is fp32, rounded once.
#include "device_common.h"
#include "ops.h"

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

template <class TR, int N>
__device__ __forceinline__ void loadN(const typename TR::T* p, float* v) {
  if constexpr(N == 1) v[0] = TR::toFloat(p[0]);
  else {
    const typename UnalignedV<typename TR::T, N>::V t = *(const typename UnalignedV<typename TR::T, N>::V*)p;
#pragma unroll
    for(int i = 0; i < N; i++) v[i] = TR::toFloat(t[i]);
  }
}
template <class TR, int N>
__device__ __forceinline__ void storeN(typename TR::T* p, const float* v) {
  if constexpr(N == 1) p[0] = TR::fromFloat(v[0]);
  else {
    typename UnalignedV<typename TR::T, N>::V t;
#pragma unroll
    for(int i = 0; i < N; i++) t[i] = TR::fromFloat(v[i]);
    *(typename UnalignedV<typename TR::T, N>::V*)p = t;
  }
}

// sine and cosine of 2 pi t, |t| <= 1/2
__device__ __forceinline__ void sinCosOfTurn(float t, float* s, float* c) {
#if defined(__AMDGCN__)
  sincospif(2.0f * t, s, c);
#else
  *s = sinf(6.28318530717958647692f * t);
  *c = cosf(6.28318530717958647692f * t);
#endif
}

struct RotaryLaunch {
  RotaryArgs a;
  int hpt;                 // heads of one thread
  int groups[2];           // ceil(heads / hpt) of q and k
  int rotItems, copyItems; // pieces of a head: PV pairs each / PV untouched channels each
  unsigned token0;
  unsigned threads;
};

// A thread owns PV pairs (or PV channels to copy) of a token in hpt heads: it forms their sines and cosines once and turns head after head, HB at a
// time so that several heads' loads are in flight. Threads of neighbouring pieces are neighbours: a head's row is read in consecutive pieces of
// 16 bytes (16-bit types, PV = 8).
template <class TR, int PV, bool HALF>
__global__ __launch_bounds__(256) void rotaryKernel(RotaryLaunch r) {
  typedef typename TR::T T;
  constexpr int HB = 4;
  const RotaryArgs& a = r.a;
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  if(idx >= r.threads) return;
  const unsigned items = (unsigned)(r.rotItems + r.copyItems), groups = (unsigned)(r.groups[0] + r.groups[1]);
  const unsigned item = idx % items, rest = idx / items;
  const unsigned group = rest % groups, token = rest / groups + r.token0;
  const unsigned b = token / (unsigned)a.seq, s = token % (unsigned)a.seq;
  const int which = group < (unsigned)r.groups[0] ? 0 : 1;
  const RotarySide& side = a.side[which];
  const int h0 = (int)(which ? group - (unsigned)r.groups[0] : group) * r.hpt;
  const int h1 = h0 + r.hpt < side.heads ? h0 + r.hpt : side.heads;
  const T* const in = (const T*)side.in + b * side.inBatch + s * side.inToken;
  T* const out = (T*)side.out + b * side.outBatch + s * side.outToken;

  if(item >= (unsigned)r.rotItems) {  // channels that are not turned (only where out is another buffer)
    const int c = 2 * a.pairs + (int)(item - (unsigned)r.rotItems) * PV;
    for(int h = h0; h < h1; h++) {
      const T* const ip = in + h * side.inHead + c;
      T* const op = out + h * side.outHead + c;
      if(c + PV <= a.headDim) {
        float v[PV];
        loadN<TR, PV>(ip, v);
        storeN<TR, PV>(op, v);
      }
      else
        for(int i = 0; c + i < a.headDim; i++) op[i] = ip[i];
    }
    return;
  }

  const int p0 = (int)item * PV;  // pairs is a multiple of PV
  double pos[2] = {0.0, 0.0};
  for(int ax = 0; ax < a.axes; ax++) {
    const int64_t at = b * a.posBatch + s * a.posToken + ax * a.posAxis;
    pos[ax] = a.pos64 ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
  }
  float cs[PV], sn[PV];
  int turned = -1;  // the frequencies' head that cs / sn belong to
  const int perFreq = side.heads / a.freqHeads;
  for(int hb = h0; hb < h1; hb += HB) {
    float u[HB][PV], v[HB][PV];
#pragma unroll
    for(int j = 0; j < HB; j++) {
      if(hb + j >= h1) break;
      const T* const ip = in + (hb + j) * side.inHead;
      if(HALF) {
        loadN<TR, PV>(ip + p0, u[j]);
        loadN<TR, PV>(ip + a.pairs + p0, v[j]);
      }
      else {
        float w[2 * PV];
        if constexpr(PV == 1) {
          w[0] = TR::toFloat(ip[2 * p0]);
          w[1] = TR::toFloat(ip[2 * p0 + 1]);
        }
        else {
          loadN<TR, PV>(ip + 2 * p0, w);
          loadN<TR, PV>(ip + 2 * p0 + PV, w + PV);
        }
#pragma unroll
        for(int i = 0; i < PV; i++) {
          u[j][i] = w[2 * i];
          v[j][i] = w[2 * i + 1];
        }
      }
    }
#pragma unroll
    for(int j = 0; j < HB; j++) {
      if(hb + j >= h1) break;
      const int fh = (hb + j) / perFreq;
      if(fh != turned) {
        turned = fh;
        const double* const f = a.freqs + (size_t)fh * a.axes * a.pairs + p0;
#pragma unroll
        for(int i = 0; i < PV; i++) {
          double t = pos[0] * f[i];
          if(a.axes == 2) t += pos[1] * f[a.pairs + i];
          t *= 0.15915494309189533577;  // 1 / 2 pi
          float sv, cv;
          sinCosOfTurn((float)(t - __builtin_rint(t)), &sv, &cv);
          cs[i] = cv * a.magnitude;
          sn[i] = (a.inverse ? -sv : sv) * a.magnitude;
        }
      }
      float x[PV], y[PV];
#pragma unroll
      for(int i = 0; i < PV; i++) {
        x[i] = u[j][i] * cs[i] - v[j][i] * sn[i];
        y[i] = u[j][i] * sn[i] + v[j][i] * cs[i];
      }
      T* const op = out + (hb + j) * side.outHead;
      if(HALF) {
        storeN<TR, PV>(op + p0, x);
        storeN<TR, PV>(op + a.pairs + p0, y);
      }
      else {
        float w[2 * PV];
#pragma unroll
        for(int i = 0; i < PV; i++) {
          w[2 * i] = x[i];
          w[2 * i + 1] = y[i];
        }
        if constexpr(PV == 1) {
          op[2 * p0] = TR::fromFloat(w[0]);
          op[2 * p0 + 1] = TR::fromFloat(w[1]);
        }
        else {
          storeN<TR, PV>(op + 2 * p0, w);
          storeN<TR, PV>(op + 2 * p0 + PV, w + PV);
        }
      }
    }
  }
}

template <class TR, int PV, bool HALF>
hipError_t launchPieces(const RotaryArgs& a, hipStream_t stream) {
  RotaryLaunch r;
  r.a = a;
  r.rotItems = a.pairs / PV;
  const bool copies = (a.side[0].heads > 0 && a.side[0].in != a.side[0].out) || (a.side[1].heads > 0 && a.side[1].in != a.side[1].out);
  r.copyItems = copies ? (a.headDim - 2 * a.pairs + PV - 1) / PV : 0;
  const int items = r.rotItems + r.copyItems;
  r.hpt = 8;
  r.groups[0] = (a.side[0].heads + r.hpt - 1) / r.hpt;
  r.groups[1] = (a.side[1].heads + r.hpt - 1) / r.hpt;
  const int64_t perToken = (int64_t)items * (r.groups[0] + r.groups[1]);
  const int64_t most = (int64_t)0x7fffffff / perToken;  // tokens of one launch: its threads are counted in 31 bits
  for(int64_t t0 = 0; t0 < a.tokens; t0 += most) {
    const int64_t n = a.tokens - t0 < most ? a.tokens - t0 : most;
    r.token0 = (unsigned)t0;
    r.threads = (unsigned)(n * perToken);
    auto kern = rotaryKernel<TR, PV, HALF>;
    hipLaunchKernelGGL(kern, dim3((r.threads + 255) / 256), dim3(256), 0, stream, r);
    const hipError_t e = hipGetLastError();
    if(e != hipSuccess) return e;
  }
  return hipSuccess;
}
template <class TR>
hipError_t launchType(const RotaryArgs& a, hipStream_t stream) {
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
