// linear8.hip — the product of two e4m3 matrices with scales:  out[m][n] = (sum_k a[m][k] sa * w[n][k] sw) + bias[n],  in fp16, bf16 or fp32.
// SCALES_ROW: one fp32 scale for each row of a and of w, applied to the finished sum; SCALES_MX: one e8m0 scale for each 32 consecutive k.
//
// Two ways to multiply, by the output's type:
//   16-bit outputs  v_mfma_scale_f32_32x32x64_f8f6f4 on the codes (2048 flop a cycle and SIMD; e8m0 scales are its operands). Its adder
//                   brings 8 products at a time to the largest one's exponent and keeps 13 bits below it, then adds those sums in fp32 (measured
//                   with a product of 2^16 beside one of 2^e: 2^3 still counts, 2^2 does not). Over a row that is 1.4e-5 of the result (7e-5 with
//                   a few channels 400 times the others): 1/3 of an fp16 rounding at worst.
//   fp32 outputs    the codes, times their e8m0 scale, are exact bf16 numbers (4 significant bits): v_mfma_f32_32x32x16_bf16, all sums in
//                   fp32, at half the rate.
#include <atomic>

#include "device_common.h"
#include "ops.h"

namespace kmx {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef b16x8 Bf8;
typedef u32x4 u32x4u __attribute__((aligned(2)));
typedef f32x4 f32x4u __attribute__((aligned(4)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));

constexpr int KSTEP = 128;  // k of one step: a row of 128 bytes in LDS, eight pieces of 16
constexpr int KPIECES = 8;

__device__ __attribute__((aligned(16))) unsigned linear8Zeros[4];  // what pieces beyond K are fetched from

#ifdef KMX_EMULATED_HIP
inline unsigned ldsAddress(void* p) { return (unsigned)(size_t)p; }
inline void dma16(const void* src, unsigned dst) { emu::globalLoadLds((size_t)src, (size_t)dst, 16, 0, 0); }
inline u32x4 ldsRead16(unsigned at) { return *(const u32x4*)(size_t)at; }
inline void waitLoads0() { emu::waitVm(0); }
#else
__device__ __forceinline__ unsigned ldsAddress(void* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) char*)p; }
__device__ __forceinline__ void dma16(const void* src, unsigned dst) {  // lane l's 16 bytes land at dst + 16 l; dst is uniform
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)(size_t)dst, 16, 0, 0);
}
__device__ __forceinline__ u32x4 ldsRead16(unsigned at) { return *(const __attribute__((address_space(3))) u32x4*)(size_t)at; }
__device__ __forceinline__ void waitLoads0() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
#endif

template <int OUT> struct OutTraits;
template <> struct OutTraits<DT_F16> { typedef TraitsF16 TR; };
template <> struct OutTraits<DT_BF16> { typedef TraitsBF16 TR; };
template <> struct OutTraits<DT_F32> { typedef TraitsF32 TR; };

// 8 codes times a power of two as bf16
__device__ __forceinline__ Bf8 bf16Of(unsigned lo, unsigned hi, float scale) {
  Bf8 v;
  const b16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const b16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
  return v;
}
__device__ __forceinline__ float ofE8m0(unsigned code) {  // 2^(code - 127); 0 is a denormal fp32, 255 a NaN
  return __builtin_bit_cast(float, code == 0 ? 0x00400000u : code == 255 ? 0x7fc00000u : code << 23);
}

// One BM x BN tile of the output on WM x WN waves. Steps of 128 k: the rows of a and w lie in LDS as they lie in memory, 128 bytes each, the eight
// pieces of row r at piece ^ ((r >> 1) & 7): the 16 lanes that a ds_read_b128 serves at a time then touch all 64 banks. The pieces are brought
// by LDS-DMA in that order (the lanes of a request take their pieces' addresses), two stages, the next step's requests behind the barrier that opens
// this step. The weights are the matrix instruction's A operand: a lane ends with consecutive output channels of one row of a and stores 16 bytes.
template <int BM, int BN, int WM, int WN, bool MX, int OUT>
__global__ __launch_bounds__(64 * WM * WN) void linear8Kernel(Linear8Args g) {
  typedef typename OutTraits<OUT>::TR TR;
  typedef typename TR::T TO;
  constexpr bool EXACT = OUT == DT_F32;
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
  constexpr int REQ_A = BM / 8 / NW, REQ_W = BN / 8 / NW;  // requests of a wave and step, 8 rows each
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && TM % 32 == 0 && TN % 32 == 0, "tile");
  constexpr unsigned STAGE = (unsigned)(BM + BN) * KSTEP;
  HIP_DYNAMIC_SHARED(f32x4, smemLinear8)
  const unsigned lds = ldsAddress(smemLinear8);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hh = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  const unsigned nTiles = (unsigned)(g.N + BN - 1) / BN;
  const int64_t m0 = (int64_t)(blockIdx.x / nTiles) * BM;
  const int n0 = (int)(blockIdx.x % nTiles) * BN;
  const int steps = (g.K + KSTEP - 1) / KSTEP, pieces = g.K / 16;
  const int mLast = (int)(g.rows - m0 < BM ? g.rows - m0 : BM) - 1, nLast = (g.N - n0 < BN ? g.N - n0 : BN) - 1;  // of this tile

  // rows beyond the matrix are fetched from its last row: their products end in rows / channels that are not stored
  const uint8_t* const aTile = g.a + m0 * g.aStride;
  const uint8_t* const wTile = g.w + (int64_t)n0 * g.wStride;
  unsigned off[REQ_A + REQ_W], piece[REQ_A + REQ_W];
#pragma unroll
  for(int j = 0; j < REQ_A + REQ_W; j++) {
    const int r = (wave + NW * (j < REQ_A ? j : j - REQ_A)) * 8 + (lane >> 3), last = j < REQ_A ? mLast : nLast;
    piece[j] = (unsigned)((lane & 7) ^ ((r >> 1) & 7));
    off[j] = (unsigned)(r < last ? r : last) * (unsigned)(j < REQ_A ? g.aStride : g.wStride) + piece[j] * 16;
  }
  auto issue = [&](int step) {
    const unsigned stage = lds + (unsigned)(step & 1) * STAGE;
    const bool whole = (step + 1) * KPIECES <= pieces;
#pragma unroll
    for(int j = 0; j < REQ_A + REQ_W; j++) {
      const uint8_t* src = (j < REQ_A ? aTile : wTile) + (size_t)step * KSTEP + off[j];
      if(!whole && step * KPIECES + (int)piece[j] >= pieces) src = (const uint8_t*)linear8Zeros;
      dma16(src, stage + (unsigned)((j < REQ_A ? 0 : BM) + (wave + NW * (j < REQ_A ? j : j - REQ_A)) * 8) * KSTEP);
    }
  };

  // a step's four e8m0 codes of this lane's rows, one byte for each 32 k
  const int blocks = MX ? g.K / MX_BLOCK : 0;
  unsigned aCodes[MX ? MI : 1], wCodes[MX ? NI : 1];
  auto fourCodes = [&](const void* scales, int64_t row, int step) {
    const uint8_t* const p = (const uint8_t*)scales + row * blocks;
    unsigned v = 0;
#pragma unroll
    for(int q = 0; q < 4; q++) {
      const int blk = step * 4 + q;
      v |= (blk < blocks ? (unsigned)p[blk] : 127u) << (8 * q);
    }
    return v;
  };
  auto loadCodes = [&](int step) {
    if constexpr(MX) {
#pragma unroll
      for(int mi = 0; mi < MI; mi++) {
        const int r = wm * TM + mi * 32 + col;
        aCodes[mi] = fourCodes(g.aScales, m0 + (r < mLast ? r : mLast), step);
      }
#pragma unroll
      for(int ni = 0; ni < NI; ni++) {
        const int r = wn * TN + ni * 32 + col;
        wCodes[ni] = fourCodes(g.wScales, n0 + (r < nLast ? r : nLast), step);
      }
    }
  };

  f32x16 acc[NI][MI];
#pragma unroll
  for(int ni = 0; ni < NI; ni++)
#pragma unroll
    for(int mi = 0; mi < MI; mi++)
#pragma unroll
      for(int v = 0; v < 16; v++) acc[ni][mi][v] = 0.0f;

  const unsigned swz = (unsigned)(col >> 1) & 7u;
  issue(0);
  for(int step = 0; step < steps; step++) {
    loadCodes(step);
    waitLoads0();
    __builtin_amdgcn_s_barrier();  // this step's pieces are there, and nobody reads the other stage any more
    if(step + 1 < steps) issue(step + 1);
    const unsigned stage = lds + (unsigned)(step & 1) * STAGE;
    const unsigned aRows = stage + (unsigned)(wm * TM + col) * KSTEP, wRows = stage + (unsigned)(BM + wn * TN + col) * KSTEP;
#pragma unroll
    for(int s = 0; s < 2; s++) {  // 64 k: pieces 4 s + hh (k 0..31 of them) and 4 s + 2 + hh (k 32..63)
      const unsigned c0 = ((unsigned)(4 * s + hh) ^ swz) * 16, c1 = ((unsigned)(4 * s + 2 + hh) ^ swz) * 16;
      u32x4 fa[MI][2], fw[NI][2];
#pragma unroll
      for(int mi = 0; mi < MI; mi++) {
        fa[mi][0] = ldsRead16(aRows + mi * 32 * KSTEP + c0);
        fa[mi][1] = ldsRead16(aRows + mi * 32 * KSTEP + c1);
      }
#pragma unroll
      for(int ni = 0; ni < NI; ni++) {
        fw[ni][0] = ldsRead16(wRows + ni * 32 * KSTEP + c0);
        fw[ni][1] = ldsRead16(wRows + ni * 32 * KSTEP + c1);
      }
      if constexpr(EXACT) {
#pragma unroll
        for(int q = 0; q < 4; q++) {  // 16 k: 8 codes of each half wave
          const int blk = 2 * s + (q >> 1);
          Bf8 ba[MI], bw[NI];
#pragma unroll
          for(int mi = 0; mi < MI; mi++)
            ba[mi] = bf16Of(fa[mi][q >> 1][2 * (q & 1)], fa[mi][q >> 1][2 * (q & 1) + 1], MX ? ofE8m0(aCodes[mi] >> (8 * blk) & 255u) : 1.0f);
#pragma unroll
          for(int ni = 0; ni < NI; ni++)
            bw[ni] = bf16Of(fw[ni][q >> 1][2 * (q & 1)], fw[ni][q >> 1][2 * (q & 1) + 1], MX ? ofE8m0(wCodes[ni] >> (8 * blk) & 255u) : 1.0f);
#pragma unroll
          for(int ni = 0; ni < NI; ni++)
#pragma unroll
            for(int mi = 0; mi < MI; mi++) acc[ni][mi] = TraitsBF16::mfma(bw[ni], ba[mi], acc[ni][mi]);
        }
      }
      else {
        // the instruction takes the scale of k 0..31 from lanes 0..31 and that of k 32..63 from lanes 32..63: byte hh of the pair of blocks
        constexpr int UNIT = 0x7f7f7f7f;
        i32x8 xa[MI], xw[NI];
#pragma unroll
        for(int mi = 0; mi < MI; mi++)
#pragma unroll
          for(int i = 0; i < 8; i++) xa[mi][i] = (int)fa[mi][i >> 2][i & 3];
#pragma unroll
        for(int ni = 0; ni < NI; ni++)
#pragma unroll
          for(int i = 0; i < 8; i++) xw[ni][i] = (int)fw[ni][i >> 2][i & 3];
#pragma unroll
        for(int ni = 0; ni < NI; ni++)
#pragma unroll
          for(int mi = 0; mi < MI; mi++)
            acc[ni][mi] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xw[ni], xa[mi], acc[ni][mi], 0, 0, 0,
                                                                          MX ? (int)(wCodes[ni] >> (16 * s + 8 * hh)) : UNIT, 0,
                                                                          MX ? (int)(aCodes[mi] >> (16 * s + 8 * hh)) : UNIT);
      }
    }
  }

  // element v of a lane: channel 8 (v / 4) + 4 hh + v % 4 of the 32, row `col`
#pragma unroll
  for(int mi = 0; mi < MI; mi++) {
    const int r = wm * TM + mi * 32 + col;
    const bool rowIn = r <= mLast;
    const float sa = MX ? 1.0f : ((const float*)g.aScales)[m0 + (rowIn ? r : mLast)];
    TO* const row = (TO*)g.out + (m0 + r) * g.outStride + n0;
#pragma unroll
    for(int ni = 0; ni < NI; ni++) {
      const int c0 = wn * TN + ni * 32;
      u32x2 pk[4];
#pragma unroll
      for(int q = 0; q < 4; q++) {
        const int c = c0 + 8 * q + 4 * hh;
        float o[4];
#pragma unroll
        for(int i = 0; i < 4; i++) {
          const int n = n0 + (c + i < nLast ? c + i : nLast);
          float x = acc[ni][mi][4 * q + i] * sa;
          if(!MX) x *= ((const float*)g.wScales)[n];
          if(g.bias != nullptr) x += g.bias[n];
          o[i] = x;
        }
        if constexpr(OUT == DT_F32) {
          if(rowIn && c + 3 <= nLast) {
            f32x4 t;
#pragma unroll
            for(int i = 0; i < 4; i++) t[i] = o[i];
            *(f32x4u*)(row + c) = t;
          }
          else if(rowIn)
            for(int i = 0; i < 4 && c + i <= nLast; i++) row[c + i] = o[i];
        }
        else {
          typename TR::V4 t;
#pragma unroll
          for(int i = 0; i < 4; i++) t[i] = TR::fromFloat(o[i]);
          pk[q] = __builtin_bit_cast(u32x2, t);
        }
      }
      if constexpr(OUT != DT_F32) {
        u32x4 whole[2];
        pairUp(pk, whole);  // whole[j]: channels 16 j + 8 hh + [0, 8)
#pragma unroll
        for(int j = 0; j < 2; j++) {
          const int c = c0 + 16 * j + 8 * hh;
          if(rowIn && c + 7 <= nLast) *(u32x4u*)(row + c) = whole[j];
          else if(rowIn) {
            const typename TR::V8 t = __builtin_bit_cast(typename TR::V8, whole[j]);
#pragma unroll
            for(int i = 0; i < 8; i++)
              if(c + i <= nLast) row[c + i] = t[i];
          }
        }
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, bool MX, int OUT>
hipError_t launchTile(const Linear8Args& g, hipStream_t stream) {
  const int64_t tiles = (g.rows + BM - 1) / BM * ((g.N + BN - 1) / BN);
  if(tiles > 0x7fffffff) return hipErrorInvalidValue;
  auto kern = linear8Kernel<BM, BN, WM, WN, MX, OUT>;
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(64 * WM * WN), 2 * (BM + BN) * KSTEP, stream, g);
  return hipGetLastError();
}
template <bool MX, int OUT>
hipError_t launchShape(const Linear8Args& g, hipStream_t stream) {
  const int64_t tiles128 = (g.rows + 127) / 128 * ((g.N + 127) / 128);
  if(tiles128 >= 256) return launchTile<128, 128, 2, 2, MX, OUT>(g, stream);
  return launchTile<64, 64, 2, 2, MX, OUT>(g, stream);
}
template <int OUT>
hipError_t launchScales(const Linear8Args& g, hipStream_t stream) {
  return g.scaleKind == SCALES_MX ? launchShape<true, OUT>(g, stream) : launchShape<false, OUT>(g, stream);
}

}  // namespace

hipError_t launchLinear8(int outType, const Linear8Args& g, hipStream_t stream) {
  if(g.rows == 0) return hipSuccess;
  if(outType == DT_F16) return launchScales<DT_F16>(g, stream);
  if(outType == DT_BF16) return launchScales<DT_BF16>(g, stream);
  if(outType == DT_F32) return launchScales<DT_F32>(g, stream);
  return hipErrorInvalidValue;
}

}  // namespace kmx
