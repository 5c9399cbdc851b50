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
typedef u32x4 Out16 __attribute__((aligned(2)));  // 16 bytes of an output row, which starts at any element
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));

constexpr int KSTEP = 128;  // k of one step: a row of 128 bytes in LDS, eight pieces of 16
constexpr int KPIECES = 8;

#ifdef KMX_EMULATED_HIP
inline unsigned ldsAddress(void* p) { return (unsigned)(size_t)p; }
typedef const char* Rsrc;
inline Rsrc bufferOf(const void* p) { return (const char*)p; }
inline void dma16(Rsrc b, unsigned off, unsigned step, unsigned dst) { emu::globalLoadLds((size_t)b + off + step, (size_t)dst, 16, 0, 0); }
inline void ldsWrite16(unsigned at, u32x4 v) { *(u32x4*)(size_t)at = v; }
inline u32x4 ldsRead16(unsigned at) { return *(const u32x4*)(size_t)at; }
template <int N> inline void waitLoads() { emu::waitVm(N); }
inline void waitReads0() {}
inline void waveBarrier() { __syncthreads(); }
#else
__device__ __forceinline__ unsigned ldsAddress(void* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) char*)p; }
// LDS-DMA: the 16 bytes at off (a lane's own) + step (uniform) of a buffer land at dst (uniform) + 16 lane. (As a buffer and not by pointers: no 64-bit
// address for each request and lane, which took more registers than there are.)
typedef __amdgpu_buffer_rsrc_t Rsrc;
__device__ __forceinline__ Rsrc bufferOf(const void* p) {  // p is uniform; said again, because a request on a descriptor in vector registers is a loop over lanes
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)(size_t)p), hi = __builtin_amdgcn_readfirstlane((unsigned)((size_t)p >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)((size_t)hi << 32 | lo), 0, 0xffffffff, 0x00027000);
}
__device__ __forceinline__ void dma16(Rsrc b, unsigned off, unsigned step, unsigned dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void*)(size_t)dst, 16, off, step, 0, 0);
}
__device__ __forceinline__ u32x4 ldsRead16(unsigned at) { return *(const __attribute__((address_space(3))) u32x4*)(size_t)at; }
__device__ __forceinline__ void ldsWrite16(unsigned at, u32x4 v) { *(__attribute__((address_space(3))) u32x4*)(size_t)at = v; }
template <int N>
__device__ __forceinline__ void waitLoads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void waitReads0() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void waveBarrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
#endif

template <int I> struct Index { static constexpr int value = I; };

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

typedef unsigned u32u __attribute__((aligned(1)));
// A row's e8m0 codes of one step, a byte for each 32 k; beyond the row's end 0 (their weights are zeros). The word is fetched in one piece - so that
// the main loop stays one block, in whose order the products and the barrier stay where they are written - and shifted when it is used.
__device__ __forceinline__ int codesAt(int blocks, int step) { return step * 4 < blocks - 4 ? step * 4 : blocks - 4; }
__device__ __forceinline__ unsigned fetchCodes(const uint8_t* p, int blocks, int step) { return *(const u32u*)(p + codesAt(blocks, step)); }
__device__ __forceinline__ unsigned shiftedCodes(unsigned word, int blocks, int step) { return word >> (8 * (step * 4 - codesAt(blocks, step))); }

// One BM x BN tile of the output on WM x WN waves. Steps of 128 k: the rows of a and w lie in LDS as they lie in memory, 128 bytes each, the eight
// pieces of row r at piece ^ ((r >> 1) & 7): the 16 lanes that a ds_read_b128 serves at a time then touch all 64 banks. The pieces are brought
// by LDS-DMA in that order (the lanes of a request take their pieces' addresses), two stages. A step multiplies two halves of 64 k: a row tile's fragments
// are replaced by the next half's as soon as they are used up, the weights' have two sets; the barrier stands behind the second half's first
// products, when the stage has been read out - it is requested anew there, a whole step ahead of its use. The weights are the matrix instruction's A
// operand: a lane ends with consecutive output channels of one row of a and stores 16 bytes.
template <int BM, int BN, int WM, int WN, bool MX, int OUT>
__global__ __launch_bounds__(64 * WM * WN) void linear8Kernel(Linear8Args g) {
  typedef typename OutTraits<OUT>::TR TR;
  typedef typename TR::T TO;
  constexpr bool EXACT = OUT == DT_F32;
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
  constexpr int REQ_A = BM / 8 / NW, REQ_W = BN / 8 / NW;  // requests of a wave and step, 8 rows each
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && TM % 32 == 0 && TN % 32 == 0 && BM + BN <= 64 * NW, "tile");
  constexpr unsigned STAGE = (unsigned)(BM + BN) * KSTEP;
  HIP_DYNAMIC_SHARED(f32x4, smemLinear8)
  const unsigned lds = ldsAddress(smemLinear8);
  unsigned* const codesOf = (unsigned*)((char*)smemLinear8 + 2 * STAGE);  // [2][BM + BN]: a step's e8m0 codes of each row of a and of w
  float* const scalesOf = (float*)codesOf;                                  // ... or [BM + BN] the rows' scales; behind either
  float* const biasOf = (float*)codesOf + 2 * (BM + BN);                    // [BN]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hh = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;

  // Work-groups go round the 8 XCDs one by one: each XCD takes a contiguous eighth of the tiles, in strips of 8 tiles of rows, so that what runs at
  // a time on an XCD shares rows of a and of w in its L2
  const unsigned mTiles = (unsigned)((g.rows + BM - 1) / BM), nTiles = (unsigned)(g.N + BN - 1) / BN;
  unsigned tile = blockIdx.x;
  {
    const unsigned all = mTiles * nTiles, xcd = tile & 7, each = all >> 3, more = all & 7;
    tile = xcd * each + (xcd < more ? xcd : more) + (tile >> 3);
  }
  const unsigned strip = tile / (8 * nTiles), in = tile % (8 * nTiles), tall = mTiles - strip * 8 < 8 ? mTiles - strip * 8 : 8;
  const int64_t m0 = (int64_t)(strip * 8 + in % tall) * BM;
  const int n0 = (int)(in / tall) * BN;
  const int steps = (g.K + KSTEP - 1) / KSTEP, pieces = g.K / 16;
  const int mLast = (int)(g.rows - m0 < BM ? g.rows - m0 : BM) - 1, nLast = (g.N - n0 < BN ? g.N - n0 : BN) - 1;  // of this tile

  // rows beyond the matrix are fetched from its last row: their products end in rows / channels that are not stored
  const uint8_t* const aTile = g.a + m0 * g.aStride;
  const uint8_t* const wTile = g.w + (int64_t)n0 * g.wStride;
  unsigned off[REQ_A + REQ_W];
  auto pieceOf = [&](int r) { return (lane & 7) ^ ((r >> 1) & 7); };
  auto rowOf = [&](int j) { return (wave + NW * (j < REQ_A ? j : j - REQ_A)) * 8 + (lane >> 3); };
#pragma unroll
  for(int j = 0; j < REQ_A + REQ_W; j++) {
    const int r = rowOf(j), last = j < REQ_A ? mLast : nLast;
    off[j] = (unsigned)(r < last ? r : last) * (unsigned)(j < REQ_A ? g.aStride : g.wStride) + (unsigned)pieceOf(r) * 16;
  }
  const Rsrc aRsrc = bufferOf(aTile), wRsrc = bufferOf(wTile);
  // CUT: the step that holds the end of K. Pieces beyond it are fetched as the row's last one; the weights' are zeroed before they are multiplied
  auto issue = [&](int step, auto cutTag) {
    const unsigned stage = lds + (unsigned)(step & 1) * STAGE;
#pragma unroll
    for(int j = 0; j < REQ_A + REQ_W; j++) {
      const unsigned dst = stage + (unsigned)((j < REQ_A ? 0 : BM) + (wave + NW * (j < REQ_A ? j : j - REQ_A)) * 8) * KSTEP;
      unsigned from = off[j];
      if constexpr(decltype(cutTag)::value != 0) {
        const int over = step * KPIECES + pieceOf(rowOf(j)) - (pieces - 1);
        from -= over > 0 ? (unsigned)over * 16 : 0;
      }
      dma16(j < REQ_A ? aRsrc : wRsrc, from, (unsigned)step * KSTEP, dst);
    }
  };

  // e8m0 codes: a thread fetches one row's of a step and puts them into LDS half a step later
  const int blocks = MX ? g.K / MX_BLOCK : 0;
  const int codeRow = (int)threadIdx.x < BM + BN ? (int)threadIdx.x : BM + BN - 1;
  const bool ofA = codeRow < BM;
  const int64_t scaleRow = ofA ? m0 + (codeRow < mLast ? codeRow : mLast) : n0 + (codeRow - BM < nLast ? codeRow - BM : nLast);
  const uint8_t* const myCodes = (const uint8_t*)(ofA ? g.aScales : g.wScales) + scaleRow * blocks;
  unsigned fetched = 0;
  auto putCodes = [&](int step) {
    if constexpr(MX) codesOf[(step & 1) * (BM + BN) + codeRow] = shiftedCodes(fetched, blocks, step);
  };

  f32x16 acc[NI][MI];
#pragma unroll
  for(int ni = 0; ni < NI; ni++)
#pragma unroll
    for(int mi = 0; mi < MI; mi++)
#pragma unroll
      for(int v = 0; v < 16; v++) acc[ni][mi][v] = 0.0f;

  const unsigned swz = (unsigned)(col >> 1) & 7u;
  // a step is two halves of 64 k; s = 0, 1: pieces 4 s + hh (k 0..31 of the half) and 4 s + 2 + hh (k 32..63)
  u32x4 fa[MI][2], fw[2][NI][2];
  auto rowsOf = [&](int step, int base) { return lds + (unsigned)(step & 1) * STAGE + (unsigned)(base + col) * KSTEP; };
  auto pieceAt = [&](int p) { return ((unsigned)(p + hh) ^ swz) * 16; };
  auto readA = [&](int step, int s, int mi) {
    const unsigned rows = rowsOf(step, wm * TM) + mi * 32 * KSTEP;
    fa[mi][0] = ldsRead16(rows + pieceAt(4 * s));
    fa[mi][1] = ldsRead16(rows + pieceAt(4 * s + 2));
  };
  auto readW = [&](int step, int s) {
    const unsigned rows = rowsOf(step, BM + wn * TN);
#pragma unroll
    for(int ni = 0; ni < NI; ni++) {
      fw[s][ni][0] = ldsRead16(rows + ni * 32 * KSTEP + pieceAt(4 * s));
      fw[s][ni][1] = ldsRead16(rows + ni * 32 * KSTEP + pieceAt(4 * s + 2));
    }
  };
  // The instruction takes the scale of k 0..31 from lanes 0..31 and that of k 32..63 from lanes 32..63: its byte 2 s of a step's four, shifted by hh
  // here. (The bf16 way needs both of a half's in every lane.)
  unsigned aCodes[MX ? MI : 1], wCodes[MX ? NI : 1], aNext[MX ? MI : 1], wNext[MX ? NI : 1];
  auto readCodes = [&](int step) {
    if constexpr(MX) {
      const unsigned* const c = codesOf + (step & 1) * (BM + BN);
#pragma unroll
      for(int mi = 0; mi < MI; mi++) aNext[mi] = c[wm * TM + mi * 32 + col] >> (EXACT ? 0 : 8 * hh);
#pragma unroll
      for(int ni = 0; ni < NI; ni++) wNext[ni] = c[BM + wn * TN + ni * 32 + col] >> (EXACT ? 0 : 8 * hh);
    }
  };
  auto takeCodes = [&]() {
    if constexpr(MX) {
#pragma unroll
      for(int mi = 0; mi < MI; mi++) aCodes[mi] = aNext[mi];
#pragma unroll
      for(int ni = 0; ni < NI; ni++) wCodes[ni] = wNext[ni];
    }
  };
  auto multiply = [&](auto sTag, int mi) {
    constexpr int s = decltype(sTag)::value;
    if constexpr(EXACT) {
#pragma unroll
      for(int q = 0; q < 4; q++) {  // 16 k: 8 codes of each half wave
        const int blk = 2 * s + (q >> 1), e = 2 * (q & 1);
        const Bf8 ba = bf16Of(fa[mi][q >> 1][e], fa[mi][q >> 1][e + 1], MX ? ofE8m0(aCodes[MX ? mi : 0] >> (8 * blk) & 255u) : 1.0f);
#pragma unroll
        for(int ni = 0; ni < NI; ni++)
          acc[ni][mi] = TraitsBF16::mfma(bf16Of(fw[s][ni][q >> 1][e], fw[s][ni][q >> 1][e + 1], MX ? ofE8m0(wCodes[MX ? ni : 0] >> (8 * blk) & 255u) : 1.0f), ba,
                                         acc[ni][mi]);
      }
    }
    else {
      constexpr int UNIT = 0x7f7f7f7f;
      i32x8 xa;
#pragma unroll
      for(int i = 0; i < 8; i++) xa[i] = (int)fa[mi][i >> 2][i & 3];
#pragma unroll
      for(int ni = 0; ni < NI; ni++) {
        i32x8 xw;
#pragma unroll
        for(int i = 0; i < 8; i++) xw[i] = (int)fw[s][ni][i >> 2][i & 3];
        acc[ni][mi] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xw, xa, acc[ni][mi], 0, 0, 2 * s, MX ? (int)wCodes[MX ? ni : 0] : UNIT, 2 * s,
                                                                      MX ? (int)aCodes[MX ? mi : 0] : UNIT);
      }
    }
  };

  const int wholeSteps = pieces / KPIECES;  // steps or steps - 1
  auto issueAny = [&](int step) {
    if(step < wholeSteps) issue(step, Index<0>());
    else issue(step, Index<1>());
  };
  auto zeroBeyond = [&](int step, int s) {  // (whatever the rows of a hold there: finite, or a NaN that the row has anyway)
#pragma unroll
    for(int b = 0; b < 2; b++)
      if(step * KPIECES + 4 * s + 2 * b + hh >= pieces) {
#pragma unroll
        for(int ni = 0; ni < NI; ni++)
#pragma unroll
          for(int i = 0; i < 4; i++) fw[s][ni][b][i] = 0;
      }
  };
  constexpr int NOTHING = 0, WHOLE = 1, CUT = 2;  // what a step requests for two steps on
  auto body = [&](int step, auto moreTag, auto requestTag) {
    constexpr bool MORE = decltype(moreTag)::value != 0;
    constexpr int REQUEST = decltype(requestTag)::value;
    takeCodes();
    readW(step, 1);
    if constexpr(!MORE)
      if(wholeSteps < steps) {
        zeroBeyond(step, 0);
        zeroBeyond(step, 1);
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for(int mi = 0; mi < MI; mi++) {
      multiply(Index<0>(), mi);
      __builtin_amdgcn_sched_barrier(0);  // (the fragment's registers are free now)
      readA(step, 1, mi);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr(MORE) putCodes(step + 1);
    multiply(Index<1>(), 0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr(MORE) {
      waitLoads<0>();   // the next stage is there,
      waitReads0();   // this one has been read out by this wave,
      waveBarrier();  // by all of them
      if constexpr(REQUEST != NOTHING) {
        if constexpr(MX) fetched = fetchCodes(myCodes, blocks, step + 2);
        issue(step + 2, Index<REQUEST == CUT ? 1 : 0>());
      }
      readCodes(step + 1);
      readW(step + 1, 0);
      readA(step + 1, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for(int mi = 1; mi < MI; mi++) {
      multiply(Index<1>(), mi);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr(MORE) readA(step + 1, 0, mi);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // both stages are requested at once; what the epilogue needs and the codes come in front of them
  const float myScale = MX ? 0.0f : ((const float*)(ofA ? g.aScales : g.wScales))[scaleRow];
  const float myBias = ofA || g.bias == nullptr ? 0.0f : g.bias[scaleRow];
  unsigned firstCodes = 0;
  if constexpr(MX) {
    if(blocks >= 4) firstCodes = fetchCodes(myCodes, blocks, 0);
    else
      for(int q = 0; q < blocks; q++) firstCodes |= (unsigned)myCodes[q] << (8 * (q + 4 - blocks));  // (as the shifted word)
    if(steps > 1) fetched = fetchCodes(myCodes, blocks, 1);
  }
  issueAny(0);
  if(steps > 1) issueAny(1);
  if constexpr(!MX) scalesOf[codeRow] = myScale;
  else codesOf[codeRow] = shiftedCodes(firstCodes, blocks, 0);
  if(!ofA) biasOf[codeRow - BM] = myBias;
  if(steps > 1) waitLoads<REQ_A + REQ_W>();
  else waitLoads<0>();
  waitReads0();
  waveBarrier();
  readCodes(0);
  readW(0, 0);
#pragma unroll
  for(int mi = 0; mi < MI; mi++) readA(0, 0, mi);
  int step = 0;
  for(; step + 2 < wholeSteps; step++) body(step, Index<1>(), Index<WHOLE>());
  if(step + 2 < steps) body(step++, Index<1>(), Index<CUT>());
  if(step + 1 < steps) body(step++, Index<1>(), Index<NOTHING>());
  body(step, Index<0>(), Index<NOTHING>());

  // The tile goes through LDS, so that a store instruction covers whole lines of consecutive rows. Element v of a lane: channel 8 (v / 4) + 4 hh + v % 4
  // of the 32, row `col`; piece p of 16 bytes of row r lies at p ^ (r & 15).
  constexpr int PER = 16 / (int)sizeof(TO), P = BN / PER;  // elements of a piece, pieces of a row
  static_assert(BM * P * 16 <= 2 * (int)STAGE && P >= 8 && (P & (P - 1)) == 0, "the tile fits the stages");
  constexpr int SWZ = P < 16 ? P - 1 : 15;
  auto place = [&](int r, int p) { return lds + (unsigned)(r * P + (p ^ (r & SWZ))) * 16; };
  waveBarrier();  // nobody reads the last stage any more
#pragma unroll
  for(int ni = 0; ni < NI; ni++) {
    const int c0 = wn * TN + ni * 32;
    f32x4 sw[4], bias[4];
#pragma unroll
    for(int q = 0; q < 4; q++) {
      if(!MX) sw[q] = *(const f32x4*)(scalesOf + BM + c0 + 8 * q + 4 * hh);
      bias[q] = *(const f32x4*)(biasOf + c0 + 8 * q + 4 * hh);
    }
#pragma unroll
    for(int mi = 0; mi < MI; mi++) {
      const int r = wm * TM + mi * 32 + col;
      const float sa = MX ? 1.0f : scalesOf[r];
      u32x2 pk[4];
#pragma unroll
      for(int q = 0; q < 4; q++) {
        f32x4 o;
#pragma unroll
        for(int i = 0; i < 4; i++) o[i] = (MX ? acc[ni][mi][4 * q + i] : acc[ni][mi][4 * q + i] * sa * sw[q][i]) + bias[q][i];
        if constexpr(OUT == DT_F32) ldsWrite16(place(r, (c0 + 8 * q + 4 * hh) / 4), __builtin_bit_cast(u32x4, o));
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
        for(int j = 0; j < 2; j++) ldsWrite16(place(r, (c0 + 16 * j + 8 * hh) / 8), whole[j]);
      }
    }
  }
  waitReads0();
  waveBarrier();
#pragma unroll 4
  for(int at = (int)threadIdx.x; at < BM * P; at += 64 * NW) {
    const int r = at / P, c = at % P * PER;
    if(r > mLast || c > nLast) continue;
    const u32x4 v = ldsRead16(place(r, at % P));
    TO* const out = (TO*)g.out + (m0 + r) * g.outStride + n0 + c;
    if(c + PER - 1 <= nLast) *(Out16*)out = v;
    else {
      struct Elements { TO e[PER]; };
      const Elements t = __builtin_bit_cast(Elements, v);
#pragma unroll
      for(int i = 0; i < PER; i++)
        if(c + i <= nLast) out[i] = t.e[i];
    }
  }
}

// Few rows: the time is the weights' way from memory, so they go straight into registers, every byte requested at once. A work-group owns 16 output
// channels and up to 16 MT rows; its 8 waves take every eighth step of 128 k (v_mfma_scale_f32_16x16x128_f8f6f4, or four of 16x16x32_bf16) and add their
// sums in LDS, in the order of the waves. Lane (r = l % 16, part = l / 16) holds k 16 part + [0, 16) and 64 + 16 part + [0, 16) of row r: 128
// consecutive bytes of each weight row a step; the e8m0 code of block b comes from the lanes of part b.
template <int MT, bool MX, int OUT>
__global__ __launch_bounds__(512) void linear8FewKernel(Linear8Args g) {
  typedef typename OutTraits<OUT>::TR TR;
  typedef typename TR::T TO;
  constexpr bool EXACT = OUT == DT_F32;
  constexpr int NW = 8, DEPTH = MT == 1 ? 4 : 2;  // waves; steps whose requests are in flight
  __shared__ float sums[NW][16][MT * 16 + 4];     // [wave][channel][row]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, part = lane >> 4;
  const int n0 = (int)blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const int nLast = (g.N - n0 < 16 ? g.N - n0 : 16) - 1, mLast = (int)(g.rows - m0 < 16 * MT ? g.rows - m0 : 16 * MT) - 1;
  const int pieces = g.K / 16, steps = (g.K + KSTEP - 1) / KSTEP, blocks = MX ? g.K / MX_BLOCK : 0;
  const int wRow = n0 + (col < nLast ? col : nLast);
  const uint8_t* const wp = g.w + (int64_t)wRow * g.wStride;
  const uint8_t* const wc = MX ? (const uint8_t*)g.wScales + (int64_t)wRow * blocks : nullptr;
  const uint8_t* ap[MT];
  const uint8_t* ac[MT];
#pragma unroll
  for(int mt = 0; mt < MT; mt++) {
    const int64_t row = m0 + (mt * 16 + col < mLast ? mt * 16 + col : mLast);
    ap[mt] = g.a + row * g.aStride;
    ac[mt] = MX ? (const uint8_t*)g.aScales + row * blocks : nullptr;
  }
  f32x4 acc[MT];
#pragma unroll
  for(int mt = 0; mt < MT; mt++)
#pragma unroll
    for(int v = 0; v < 4; v++) acc[mt][v] = 0.0f;

  for(int s0 = wave; s0 < steps; s0 += NW * DEPTH) {
    u32x4 fw[DEPTH][2], fa[DEPTH][MT][2];
    unsigned cw[DEPTH], ca[DEPTH][MT];
#pragma unroll
    for(int d = 0; d < DEPTH; d++) {  // steps beyond the last: its pieces again, not multiplied
      const int step = s0 + d * NW < steps ? s0 + d * NW : steps - 1;
#pragma unroll
      for(int b = 0; b < 2; b++) {  // pieces beyond K: the row's last one, the weights' then zeroed
        const int want = step * KPIECES + 4 * b + part, piece = want < pieces ? want : pieces - 1;
        fw[d][b] = *(const u32x4*)(wp + (size_t)piece * 16);
#pragma unroll
        for(int mt = 0; mt < MT; mt++) fa[d][mt][b] = *(const u32x4*)(ap[mt] + (size_t)piece * 16);
      }
      if constexpr(MX) {
        if(blocks >= 4) {
          cw[d] = fetchCodes(wc, blocks, step);
#pragma unroll
          for(int mt = 0; mt < MT; mt++) ca[d][mt] = fetchCodes(ac[mt], blocks, step);
        }
        else {  // (as the words that shiftedCodes takes; one step)
          cw[d] = 0;
#pragma unroll
          for(int mt = 0; mt < MT; mt++) ca[d][mt] = 0;
          for(int q = 0; q < blocks; q++) {
            cw[d] |= (unsigned)wc[q] << (8 * (q + 4 - blocks));
#pragma unroll
            for(int mt = 0; mt < MT; mt++) ca[d][mt] |= (unsigned)ac[mt][q] << (8 * (q + 4 - blocks));
          }
        }
      }
    }
#pragma unroll
    for(int d = 0; d < DEPTH; d++) {
      const int step = s0 + d * NW;
      if(step >= steps) break;
#pragma unroll
      for(int b = 0; b < 2; b++)
        if(step * KPIECES + 4 * b + part >= pieces) {
#pragma unroll
          for(int i = 0; i < 4; i++) fw[d][b][i] = 0;
        }
      if constexpr(MX) {
        cw[d] = shiftedCodes(cw[d], blocks, step);
#pragma unroll
        for(int mt = 0; mt < MT; mt++) ca[d][mt] = shiftedCodes(ca[d][mt], blocks, step);
      }
#pragma unroll
      for(int mt = 0; mt < MT; mt++) {
        if constexpr(EXACT) {
#pragma unroll
          for(int q = 0; q < 4; q++) {  // 8 codes of each lane
            const int b = q >> 1, e = 2 * (q & 1), shift = 8 * (2 * b + (part >> 1));
            acc[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16Of(fw[d][b][e], fw[d][b][e + 1], MX ? ofE8m0(cw[d] >> shift & 255u) : 1.0f),
                                                              bf16Of(fa[d][mt][b][e], fa[d][mt][b][e + 1], MX ? ofE8m0(ca[d][mt] >> shift & 255u) : 1.0f), acc[mt], 0, 0, 0);
          }
        }
        else {
          i32x8 xw, xa;
#pragma unroll
          for(int i = 0; i < 8; i++) {
            xw[i] = (int)fw[d][i >> 2][i & 3];
            xa[i] = (int)fa[d][mt][i >> 2][i & 3];
          }
          constexpr int UNIT = 0x7f7f7f7f;
          acc[mt] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xw, xa, acc[mt], 0, 0, 0, MX ? (int)(cw[d] >> (8 * part)) : UNIT, 0,
                                                                     MX ? (int)(ca[d][mt] >> (8 * part)) : UNIT);
        }
      }
    }
  }
#pragma unroll
  for(int mt = 0; mt < MT; mt++)  // element v of a lane: channel 4 part + v, row `col`
#pragma unroll
    for(int v = 0; v < 4; v++) sums[wave][4 * part + v][mt * 16 + col] = acc[mt][v];
  __syncthreads();
  for(int at = (int)threadIdx.x; at < MT * 16 * 16; at += 64 * NW) {
    const int c = at & 15, r = at >> 4;
    if(r > mLast || c > nLast) continue;
    float x = 0.0f;
#pragma unroll
    for(int w = 0; w < NW; w++) x += sums[w][c][r];
    if(!MX) x = x * ((const float*)g.aScales)[m0 + r] * ((const float*)g.wScales)[n0 + c];
    if(g.bias != nullptr) x += g.bias[n0 + c];
    ((TO*)g.out)[(m0 + r) * g.outStride + n0 + c] = TR::fromFloat(x);
  }
}

template <int MT, bool MX, int OUT>
hipError_t launchFew(const Linear8Args& g, hipStream_t stream) {
  auto kern = linear8FewKernel<MT, MX, OUT>;
  hipLaunchKernelGGL(kern, dim3((unsigned)((g.N + 15) / 16), (unsigned)((g.rows + 16 * MT - 1) / (16 * MT))), dim3(512), 0, stream, g);
  return hipGetLastError();
}
template <int BM, int BN, int WM, int WN, bool MX, int OUT>
hipError_t launchTile(const Linear8Args& g, hipStream_t stream) {
  const int64_t tiles = (g.rows + BM - 1) / BM * ((g.N + BN - 1) / BN);
  if(tiles > 0x7fffffff) return hipErrorInvalidValue;
  constexpr int LDS = 2 * (BM + BN) * (KSTEP + 4) + BN * 4;
  auto kern = linear8Kernel<BM, BN, WM, WN, MX, OUT>;
  if(LDS > 64 * 1024) {  // opt in to the large LDS window, once per instantiation and device
    constexpr int MAX_DEVICES = 64;
    static std::atomic<bool> attrSet[MAX_DEVICES];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if(e != hipSuccess) return e;
    if(dev < 0 || dev >= MAX_DEVICES) return hipErrorInvalidDevice;
    if(!attrSet[dev].load(std::memory_order_acquire)) {
      e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
      if(e != hipSuccess) return e;
      attrSet[dev].store(true, std::memory_order_release);
    }
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(64 * WM * WN), LDS, stream, g);
  return hipGetLastError();
}
template <bool MX, int OUT>
hipError_t launchShape(const Linear8Args& g, hipStream_t stream) {
  if(g.rows <= 16) return launchFew<1, MX, OUT>(g, stream);
  if(g.rows <= 32) return launchFew<2, MX, OUT>(g, stream);
  if(g.rows <= 64) return launchFew<4, MX, OUT>(g, stream);
  auto tiles = [&](int bm, int bn) { return (g.rows + bm - 1) / bm * ((g.N + bn - 1) / bn); };
  if constexpr(OUT != DT_F32)
    if(tiles(256, 256) >= 256) return launchTile<256, 256, 2, 4, MX, OUT>(g, stream);
  if(tiles(128, 128) >= 256) return launchTile<128, 128, 2, 2, MX, OUT>(g, stream);
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
