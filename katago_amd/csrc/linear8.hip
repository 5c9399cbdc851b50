// linear8.hip — the product of two e4m3 matrices with scales:  out[m][n] = (sum_k a[m][k] sa * w[n][k] sw) + bias[n],  in fp16, bf16 or fp32.
// SCALES_ROW: one fp32 scale for each row of a and of w, applied to the finished sum; SCALES_MX: one e8m0 scale for each 32 consecutive k.
//
// Two ways to multiply, by the output's type:
//   16-bit outputs  v_mfma_scale_f32_32x32x64_f8f6f4 on the codes (2048 flop a cycle and SIMD; e8m0 scales are its operands). Its adder
//                   brings 8 products at a time to the largest one's exponent and keeps 13 bits below it, then adds those sums in fp32 (measured
//                   with a product of 2^16 beside one of 2^e: 2^3 still counts, 2^2 does not): a result is off by up to 7 * 2^-13 of the sum of its
//                   products' magnitudes, relative to itself by more where they cancel. Over random rows it was 1.4e-5 of the results' norm
//                   (7e-5 with a few channels 400 times the others), where an fp16 rounding is 2.8e-4.
//   fp32 outputs    the codes, times their e8m0 scale, as bf16 numbers: v_mfma_f32_32x32x16_bf16, all sums in fp32, at half the rate. 4
//                   significant bits are exact there with scales from 2^-124 (bf16 reaches down to 2^-133, the smallest code is 2^-9) to 2^119
//                   (448 * 2^119 < 2^128). An e8m0 scale beyond these belongs to values that fp32 itself does not hold, or barely.
//
// Long k is bound by the matrix cores and the LDS that feeds them: 8192^3 with row scales 380 to 395 us (2780 to 2890 TFLOP/s; a large library product in
// 8 bits reaches 2330 with scales by row, 2810 with one for all), 8190 x 11008 x 4096 with scales for 32 k each 330 to 340 us (2170 to 2240), the same into fp32
// 740 to 770 us (960 to 1000), 8191 x 11007 x 4096 with row scales 312 (2370). Short k is bound by what surrounds the products, whose steps overlap in
// part: 92416 x 1152 x 384 62 us (4.0 TB/s; bytes alone: 49). Few rows are bound by the weights' way in: 1 x 4096 x 4096 5.0 us (3.4 TB/s), x 11008 10.1 (4.5).
#include <atomic>

#include "ops.h"
#include "ops_device.h"

namespace kmx {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef b16x8 Bf8;
typedef u32x4 Out16 __attribute__((aligned(2)));  // 16 bytes of an output row, which starts at any element
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));

// Whole lines of results go past the caches: in them they would push out a's rows, which several work-groups read, before all have read them
// (92416 x 1152 x 384 79 -> 68 us, x 2048 138 -> 99, 8190 x 11008 x 4096 348 -> 327)
__device__ __forceinline__ void streamOut(void* to, u32x4 v) { __builtin_nontemporal_store(v, (Out16*)to); }

constexpr int KSTEP = 128;  // k of one step: a row of 128 bytes in LDS, eight pieces of 16
constexpr int KPIECES = 8;

#ifdef KMX_EMULATED_HIP
inline unsigned ldsAddress(void* p) { return (unsigned)(size_t)p; }
typedef const char* Rsrc;
inline Rsrc bufferOf(const void* p) { return (const char*)p; }
inline void dma16(Rsrc b, unsigned off, unsigned step, unsigned dst) { emu::globalLoadLds((size_t)b + off + step, (size_t)dst, 16, 0, 0); }
inline void ldsWrite16(unsigned at, u32x4 v) { *(u32x4*)(size_t)at = v; }
inline void waveFence() { emu::waveSync(); }
inline u32x4 ldsRead16(unsigned at) { return *(const u32x4*)(size_t)at; }
template <int N> inline void waitLoads() { emu::waitVm(N); }
inline void waitReads0() {}
inline void waveBarrier() { __syncthreads(); }
inline int anew(int x) { return x; }
inline void countedStore() { emu::vmNote(); }
template <class V> inline void computed(V&) {}
inline hipError_t computeUnits(int, int* n) {
  *n = 8;  // (few: work-groups go round more than once)
  return hipSuccess;
}
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
// Lanes of a wave hand data to one another through LDS, whose instructions a wave has carried out in order: only the compiler, which sees one lane's
// addresses, must not exchange them
__device__ __forceinline__ void waveFence() { asm volatile("" ::: "memory"); }
template <int N>
__device__ __forceinline__ void waitLoads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void waitReads0() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void waveBarrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// v is computed by here: products do not move behind the barriers and branches that follow
template <class V>
__device__ __forceinline__ void computed(V& v) {
  asm volatile("" : "+v"(v));
}
// A store instruction that a later wait's count includes (the emulation enters it into the wave's queue)
__device__ __forceinline__ void countedStore() {}
// x, as far as the compiler can tell a new value each time: what is computed from it is not kept in registers around a loop
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
hipError_t computeUnits(int device, int* n) { return hipDeviceGetAttribute(n, hipDeviceAttributeMultiprocessorCount, device); }
#endif

constexpr int CUS = 256;  // of the chip: what the choice of a kernel was measured on
#ifdef KMX_EMULATED_HIP
constexpr int PER_XCD = 2, SHORT_TILES = 2;  // (few rows are many)
inline int chosenFor() {  // (few tiles are more than such a chip holds: the large ones are chosen, and go round)
  const char* const e = getenv("KMX_EMU_CUS");
  return e != nullptr ? atoi(e) : CUS;
}
#else
constexpr int chosenFor() { return CUS; }
constexpr int PER_XCD = CUS / 8 * 2, SHORT_TILES = 10;  // linear8ShortKernel: work-groups of an XCD, tiles of each at least
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

// A sum of products of codes is 0 or between 2^-18 (the smallest product) and 2^41 (448^2 over 2^23 channels): scales between 2^-40 and 2^40 may be
// applied one after the other and nothing leaves fp32 on the way. Of any others the mantissas are multiplied and the exponents added, so that a result
// is infinite or below the smallest number only where the formula's is. (The choice is made once a wave and tile; 361 x 1152 x 384 take 0.15 us longer for
// the second way's code, large products nothing.)
__device__ __forceinline__ bool mild(float scale) { return scale >= 0x1p-40f && scale <= 0x1p40f; }
__device__ __forceinline__ float scaledByAny(float sum, float sa, float sw) {
  int ea, ew;
  const float ma = frexpf(sa, &ea), mw = frexpf(sw, &ew);
  return ldexpf(sum * ma * mw, ea + ew);
}

typedef unsigned u32u __attribute__((aligned(1)));
// A row's e8m0 codes of one step, a byte for each 32 k; beyond the row's end 0 (their weights are zeros). The word is fetched in one piece - so that
// the main loop stays one block, in whose order the products and the barrier stay where they are written - and shifted when it is used.
__device__ __forceinline__ int codesAt(int blocks, int step) { return step * 4 < blocks - 4 ? step * 4 : blocks - 4; }  // (below 0: fetched byte by byte)
__device__ __forceinline__ unsigned fetchCodes(const uint8_t* p, int blocks, int step) { return *(const u32u*)(p + codesAt(blocks, step)); }
__device__ __forceinline__ unsigned shiftedCodes(unsigned word, int blocks, int step) {
  const int by = 8 * (step * 4 - codesAt(blocks, step));
  return by < 32 ? word >> by : 0u;
}

// BM x BN tiles of the output on WM x WN waves, the work-groups stay and take tile after tile. Steps of 128 k: the rows of a and w lie in LDS as they lie
// in memory, 128 bytes each, the eight pieces of row r at piece ^ ((r >> 1) & 7): the 16 lanes that a ds_read_b128 serves at a time then touch all 64
// banks. The pieces are brought by LDS-DMA in that order (the lanes of a request take their pieces' addresses), two stages (or four). A step multiplies two
// halves of 64 k: a row tile's fragments are replaced by the next half's as soon as they are used up, the weights' have two sets; the barrier stands
// behind the second half's first products, when the stage has been read out - it is requested anew there, a whole step ahead of its use. The last two
// steps of a tile request the first two of the next: a tile's results are scaled and stored while the next one's operands are on their way. The
// weights are the matrix instruction's A operand: a lane ends with consecutive output channels of one row of a.
template <int BM, int BN, int WM, int WN, int STAGES, bool MX, int OUT>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear8Kernel(Linear8Args g) {
  typedef typename OutTraits<OUT>::TR TR;
  typedef typename TR::T TO;
  constexpr bool EXACT = OUT == DT_F32;
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
  constexpr int REQ_A = BM / 8 / NW, REQ_W = BN / 8 / NW;  // requests of a wave and step, 8 rows each
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && TM % 32 == 0 && TN % 32 == 0 && BM + BN <= 64 * NW, "tile");
  constexpr unsigned STAGE = (unsigned)(BM + BN) * KSTEP;
  HIP_DYNAMIC_SHARED(f32x4, smemLinear8)
  const unsigned lds = ldsAddress(smemLinear8);
  static_assert(STAGES == 2 || STAGES == 4, "ring");
  unsigned* const codesOf = (unsigned*)((char*)smemLinear8 + STAGES * STAGE);  // [2][BM + BN]: the e8m0 codes of each row, by step;
  float* const scalesOf = (float*)codesOf;                                // ... or the rows' scales, by tile
  float* const biasOf = (float*)codesOf + 2 * (BM + BN);                  // [2][BN], by tile
  const unsigned patch = lds + STAGES * STAGE + (2 * (BM + BN) + 2 * BN) * 4;  // 2 KB of each wave: what is being stored
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hh = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  const int pieces = g.K / 16, blocks = MX ? g.K / MX_BLOCK : 0;
  // at least one more than there are stages: whatever lies beyond K has weights of zero
  const int steps = g.K > STAGES * KSTEP ? (g.K + KSTEP - 1) / KSTEP : STAGES + 1;

  // Work-groups go round the 8 XCDs one by one: each XCD takes a contiguous eighth of the tiles, in strips of 8 tiles of rows, so that what runs at
  // a time on an XCD shares rows of a and of w in its L2
  const unsigned mTiles = (unsigned)((g.rows + BM - 1) / BM), nTiles = (unsigned)(g.N + BN - 1) / BN, allTiles = mTiles * nTiles;
  struct Tile {
    int64_t m0;
    int n0, mLast, nLast;  // the last row and channel of it that exist
  };
  auto tileAt = [&](unsigned id) {
    const unsigned xcd = id & 7, each = allTiles >> 3, more = allTiles & 7;
    const unsigned at = xcd * each + (xcd < more ? xcd : more) + (id >> 3);
    const unsigned strip = at / (8 * nTiles), in = at % (8 * nTiles), tall = mTiles - strip * 8 < 8 ? mTiles - strip * 8 : 8;
    Tile t;
    t.m0 = (int64_t)(strip * 8 + in % tall) * BM;
    t.n0 = (int)(in / tall) * BN;
    t.mLast = (int)(g.rows - t.m0 < BM ? g.rows - t.m0 : BM) - 1;
    t.nLast = (g.N - t.n0 < BN ? g.N - t.n0 : BN) - 1;
    return t;
  };

  // What is requested: rows beyond the matrix are fetched from its last row (their products end in rows / channels that are not stored), pieces beyond
  // K as the row's last one (the weights' are zeroed before they are multiplied; a's are finite, or a NaN that the row has anyway).
  unsigned off[REQ_A + REQ_W];
  Rsrc aRsrc = bufferOf(g.a), wRsrc = bufferOf(g.w);
  auto pieceOf = [&](int r, int lane) { return (lane & 7) ^ ((r >> 1) & 7); };
  auto rowOf = [&](int j, int lane) { return (wave + NW * (j < REQ_A ? j : j - REQ_A)) * 8 + (lane >> 3); };
  auto aim = [&](const Tile& t) {
    const int ln = anew(lane);
    aRsrc = bufferOf(g.a + t.m0 * g.aStride);
    wRsrc = bufferOf(g.w + (int64_t)t.n0 * g.wStride);
    const unsigned piece = (unsigned)pieceOf(rowOf(0, ln), ln) * 16;  // (rows of one lane differ by multiples of 16: one place of the eight)
    static_assert(NW % 2 == 0, "pieces");
    if(t.mLast == BM - 1 && t.nLast == BN - 1) {
      off[0] = (unsigned)rowOf(0, ln) * (unsigned)g.aStride + piece;
      off[REQ_A] = (unsigned)rowOf(REQ_A, ln) * (unsigned)g.wStride + piece;
#pragma unroll
      for(int j = 1; j < REQ_A; j++) off[j] = off[0] + (unsigned)(j * NW * 8) * (unsigned)g.aStride;
#pragma unroll
      for(int j = 1; j < REQ_W; j++) off[REQ_A + j] = off[REQ_A] + (unsigned)(j * NW * 8) * (unsigned)g.wStride;
    }
    else {
#pragma unroll
      for(int j = 0; j < REQ_A + REQ_W; j++) {
        const int r = rowOf(j, ln), last = j < REQ_A ? t.mLast : t.nLast;
        off[j] = (unsigned)(r < last ? r : last) * (unsigned)(j < REQ_A ? g.aStride : g.wStride) + piece;
      }
    }
  };
  auto issueOne = [&](int j, int step, int stage, auto cutTag, int ln) {  // CUT: pieces of this step may lie beyond K
    const unsigned dst = lds + (unsigned)stage * STAGE + (unsigned)((j < REQ_A ? 0 : BM) + (wave + NW * (j < REQ_A ? j : j - REQ_A)) * 8) * KSTEP;
    if constexpr(decltype(cutTag)::value != 0) {
      const int over = step * KPIECES + pieceOf(rowOf(j, ln), ln) - (pieces - 1);
      dma16(j < REQ_A ? aRsrc : wRsrc, off[j] + (unsigned)step * KSTEP - (over > 0 ? (unsigned)over * 16 : 0), 0, dst);
    }
    else dma16(j < REQ_A ? aRsrc : wRsrc, off[j], (unsigned)step * KSTEP, dst);
  };
  auto issue = [&](int step, int stage) {
    const int ln = anew(lane);
#pragma unroll
    for(int j = 0; j < REQ_A + REQ_W; j++) issueOne(j, step, stage, Index<1>(), ln);
  };

  // A thread fetches one row's e8m0 codes of a step and puts them into LDS a step later; or one row's scale of a tile, and the bias
  const int codeRow = (int)threadIdx.x < BM + BN ? (int)threadIdx.x : BM + BN - 1;
  const bool ofA = codeRow < BM;
  auto scaleRow = [&](const Tile& t) {
    return ofA ? t.m0 + (codeRow < t.mLast ? codeRow : t.mLast) : t.n0 + (codeRow - BM < t.nLast ? codeRow - BM : t.nLast);
  };
  const uint8_t* myCodes = nullptr;
  unsigned fetched = 0;
  auto putCodes = [&](int step, int parity) {
    if constexpr(MX) codesOf[parity * (BM + BN) + codeRow] = shiftedCodes(fetched, blocks, step);
  };
  auto fetchAny = [&](int step) {
    if(blocks >= 4) return fetchCodes(myCodes, blocks, step);
    unsigned v = 0;
    for(int q = 0; q < blocks; q++) v |= (unsigned)myCodes[q] << (8 * (q + 4 - blocks));  // (as the word that is shifted)
    return v;
  };
  float myScale = 0.0f, myBias = 0.0f;
  auto fetchScales = [&](const Tile& t) {
    const int64_t row = scaleRow(t);
    if constexpr(!MX) myScale = ((const float*)(ofA ? g.aScales : g.wScales))[row];
    if(g.bias != nullptr) myBias = g.bias[ofA ? 0 : row];
  };
  auto putScales = [&](int parity) {
    if constexpr(!MX) scalesOf[parity * (BM + BN) + codeRow] = myScale;
    if(!ofA) biasOf[parity * BN + codeRow - BM] = myBias;
  };

  f32x16 acc[NI][MI];
  const unsigned swz = (unsigned)(col >> 1) & 7u;
  // a step is two halves of 64 k; s = 0, 1: pieces 4 s + hh (k 0..31 of the half) and 4 s + 2 + hh (k 32..63)
  u32x4 fa[MI][2], fw[2][NI][2];
  auto rowsOf = [&](int stage, int base) { return lds + (unsigned)stage * STAGE + (unsigned)(base + col) * KSTEP; };
  auto pieceAt = [&](int p) { return ((unsigned)(p + hh) ^ swz) * 16; };
  auto readA = [&](int stage, int s, int mi) {
    const unsigned rows = rowsOf(stage, wm * TM) + mi * 32 * KSTEP;
    fa[mi][0] = ldsRead16(rows + pieceAt(4 * s));
    fa[mi][1] = ldsRead16(rows + pieceAt(4 * s + 2));
  };
  auto readW = [&](int stage, int s) {
    const unsigned rows = rowsOf(stage, BM + wn * TN);
#pragma unroll
    for(int ni = 0; ni < NI; ni++) {
      fw[s][ni][0] = ldsRead16(rows + ni * 32 * KSTEP + pieceAt(4 * s));
      fw[s][ni][1] = ldsRead16(rows + ni * 32 * KSTEP + pieceAt(4 * s + 2));
    }
  };
  // The instruction takes the scale of k 0..31 from lanes 0..31 and that of k 32..63 from lanes 32..63: its byte 2 s of a step's four, shifted by hh
  // here. (The bf16 way needs both of a half's in every lane.)
  unsigned aCodes[MX ? MI : 1], wCodes[MX ? NI : 1], aNext[MX ? MI : 1], wNext[MX ? NI : 1];
  auto readCodes = [&](int parity) {
    if constexpr(MX) {
      const unsigned* const c = codesOf + parity * (BM + BN);
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
  auto multiply = [&](auto sTag, int mi, int ni) {
    constexpr int s = decltype(sTag)::value;
    if constexpr(EXACT) {
#pragma unroll
      for(int q = 0; q < 4; q++) {  // 16 k: 8 codes of each half wave
        const int blk = 2 * s + (q >> 1), e = 2 * (q & 1);
        const Bf8 ba = bf16Of(fa[mi][q >> 1][e], fa[mi][q >> 1][e + 1], MX ? ofE8m0(aCodes[MX ? mi : 0] >> (8 * blk) & 255u) : 1.0f);
        const Bf8 bw = bf16Of(fw[s][ni][q >> 1][e], fw[s][ni][q >> 1][e + 1], MX ? ofE8m0(wCodes[MX ? ni : 0] >> (8 * blk) & 255u) : 1.0f);
        acc[ni][mi] = TraitsBF16::mfma(bw, ba, acc[ni][mi]);
      }
    }
    else {
      constexpr int UNIT = 0x7f7f7f7f;
      i32x8 xa, xw;
#pragma unroll
      for(int i = 0; i < 8; i++) {
        xa[i] = (int)fa[mi][i >> 2][i & 3];
        xw[i] = (int)fw[s][ni][i >> 2][i & 3];
      }
      acc[ni][mi] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xw, xa, acc[ni][mi], 0, 0, 2 * s, MX ? (int)wCodes[MX ? ni : 0] : UNIT, 2 * s,
                                                                    MX ? (int)aCodes[MX ? mi : 0] : UNIT);
    }
  };
  auto zeroBeyond = [&](int step, int s) {
#pragma unroll
    for(int b = 0; b < 2; b++) {
      const unsigned keep = step * KPIECES + 4 * s + 2 * b + hh < pieces ? 0xffffffffu : 0u;
#pragma unroll
      for(int ni = 0; ni < NI; ni++)
#pragma unroll
        for(int i = 0; i < 4; i++) fw[s][ni][b][i] &= keep;
    }
  };
  auto pin = [&]() {
#pragma unroll
    for(int ni = 0; ni < NI; ni++)
#pragma unroll
      for(int mi = 0; mi < MI; mi++) computed(acc[ni][mi]);
  };

  // One step: the at-th of this work-group (its stage and codes by that), `step` of its tile. The stage is requested anew, with step `want` of the tile that
  // is aimed at; a request holds a wave's issue for as long as
  // a product takes, so they are spread among the products behind the barrier. Products and barrier stay in this order because there is no branch
  // between them. youngerTag: how many memory
  // instructions younger than the next stage's requests may be under way at the barrier.
  constexpr int INSIDE = 0, END = 1;  // END: one of a tile's last steps - K may end in it, and what it requests
  constexpr int AHEAD = (STAGES - 2) * (REQ_A + REQ_W);  // requests of the stages behind the next
  auto body = [&](int at, int step, int want, int codesPut, int codesFetch, auto kindTag, auto youngerTag) {
    constexpr int KIND = decltype(kindTag)::value;
    const int stage = at & (STAGES - 1), after = (at + 1) & (STAGES - 1);
    takeCodes();
    readW(stage, 1);
    if constexpr(KIND == END)
      if((step + 1) * KPIECES > pieces) {
        zeroBeyond(step, 0);
        zeroBeyond(step, 1);
      }
    unsigned next = 0;
    if constexpr(MX && KIND == END) next = fetchAny(codesFetch);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for(int mi = 0; mi < MI; mi++) {
#pragma unroll
      for(int ni = 0; ni < NI; ni++) multiply(Index<0>(), mi, ni);
      __builtin_amdgcn_sched_barrier(0);  // (the fragment's registers are free now)
      readA(stage, 1, mi);
      __builtin_amdgcn_sched_barrier(0);
    }
    putCodes(codesPut, (at + 1) & 1);
#pragma unroll
    for(int ni = 0; ni < NI; ni++) multiply(Index<1>(), 0, ni);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr(KIND == END) pin();
    waitLoads<AHEAD + decltype(youngerTag)::value>();  // the next stage is there,
    waitReads0();                                      // this one has been read out by this wave,
    waveBarrier();                                     // by all of them
    if constexpr(MX) fetched = KIND == END ? next : fetchCodes(myCodes, blocks, codesFetch);
    readCodes((at + 1) & 1);
    readW(after, 0);
    readA(after, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    constexpr int REQ = REQ_A + REQ_W, SLOTS = MI > 1 ? (MI - 1) * NI : 1;
    const int ln = KIND == END ? anew(lane) : 0;
    auto requestsOf = [&](int slot) {
#pragma unroll
      for(int j = 0; j < REQ; j++)
        if(j * SLOTS / REQ == slot) issueOne(j, want, stage, Index<KIND>(), ln);
    };
    if constexpr(MI == 1) requestsOf(0);
#pragma unroll
    for(int mi = 1; mi < MI; mi++) {
#pragma unroll
      for(int ni = 0; ni < NI; ni++) {
        requestsOf((mi - 1) * NI + ni);
        __builtin_amdgcn_sched_barrier(0);
        multiply(Index<1>(), mi, ni);
        __builtin_amdgcn_sched_barrier(0);
      }
      readA(after, 0, mi);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr(KIND == END) pin();
  };

  // Scales, bias, the output's type, and the way to memory: some rows at a time through 2 KB of the wave's own, so that a store instruction covers whole
  // lines (16 bytes a lane straight from the accumulators' layout: 4 % slower at 92416 x 1152 x 384). Element v of a lane: channel
  // 8 (v / 4) + 4 hh + v % 4 of the 32, row `col`; piece p of 16 bytes of a row lies at p ^ (row & SWZ). A tile that is whole has no branch here.
  // anyTag: scales of any size.
  auto store = [&](const Tile& t, int parity, auto wholeTag, auto anyTag) {
    constexpr bool WHOLE = decltype(wholeTag)::value != 0, ANY = decltype(anyTag)::value != 0;
    constexpr int PER = 16 / (int)sizeof(TO), P = TN / PER, ROWS = 2048 / (P * 16);  // elements of a piece, pieces of a row, rows of a patch
    constexpr int SWZ = (P < ROWS / 2 ? P : ROWS / 2) - 1 < 7 ? (P < ROWS / 2 ? P : ROWS / 2) - 1 : 7;
    static_assert(ROWS >= 8 && ROWS <= 32 && (P & (P - 1)) == 0, "patch");
    static_assert(64 / P == ROWS / 2 && ((ROWS / 2) & SWZ) == 0, "a lane reads and stores a piece of row lane / P, and the same ROWS / 2 rows on");
    const unsigned mine = patch + (unsigned)wave * 2048;
    const int ln = anew(lane), col = ln & 31, hh = ln >> 5;
    const float* const sc = scalesOf + parity * (BM + BN);
    const float* const bi = biasOf + parity * BN + wn * TN;
    TO* const corner = (TO*)g.out + (t.m0 + wm * TM) * g.outStride + t.n0 + wn * TN;
    const int rowsLeft = t.mLast - wm * TM, colsLeft = t.nLast - wn * TN;  // last row / channel of this wave's part
    const unsigned from = mine + (unsigned)(ln / P * P + (ln % P ^ (ln / P & SWZ))) * 16;
    const unsigned mineTo = (unsigned)(ln / P) * (unsigned)g.outStride * (unsigned)sizeof(TO) + (unsigned)(ln % P) * 16;
    auto put = [&](int row0, u32x4 v) {
      if(WHOLE) countedStore();
      TO* const to = (TO*)((char*)(corner + (int64_t)row0 * g.outStride) + mineTo);
      if(WHOLE && BM > 64) streamOut(to, v);
      else if(WHOLE) *(Out16*)to = v;  // (few rows: whatever reads them next finds them in the caches)
      else if(row0 + ln / P <= rowsLeft) {
        const int c = ln % P * PER;
        if(c + PER - 1 <= colsLeft) *(Out16*)to = v;
        else {
          struct Elements { TO e[PER]; };
          const Elements e = __builtin_bit_cast(Elements, v);
#pragma unroll
          for(int k = 0; k < PER; k++)
            if(c + k <= colsLeft) to[k] = e.e[k];
        }
      }
    };
#pragma unroll
    for(int mi = 0; mi < MI; mi++) {
      const float sa = MX ? 1.0f : sc[wm * TM + mi * 32 + col];
      u32x4 out[NI][OUT == DT_F32 ? 4 : 2];  // fp32: pieces of channels 8 q + 4 hh + [0, 4); 16 bits: 16 j + 8 hh + [0, 8)
#pragma unroll
      for(int ni = 0; ni < NI; ni++) {
        u32x2 pk[4];
#pragma unroll
        for(int q = 0; q < 4; q++) {
          const f32x4 bias = *(const f32x4*)(bi + ni * 32 + 8 * q + 4 * hh);
          f32x4 sw = bias, o;
          if(!MX) sw = *(const f32x4*)(sc + BM + wn * TN + ni * 32 + 8 * q + 4 * hh);
#pragma unroll
          for(int i = 0; i < 4; i++) {
            const float sum = acc[ni][mi][4 * q + i];
            o[i] = (MX ? sum : ANY ? scaledByAny(sum, sa, sw[i]) : sum * sa * sw[i]) + bias[i];
          }
          if constexpr(OUT == DT_F32) out[ni][q] = __builtin_bit_cast(u32x4, o);
          else {
            typename TR::V4 h;
#pragma unroll
            for(int i = 0; i < 4; i++) h[i] = TR::fromFloat(o[i]);
            pk[q] = __builtin_bit_cast(u32x2, h);
          }
        }
        if constexpr(OUT != DT_F32) {
          u32x4 two[2];
          pairUp(pk, two);
          out[ni][0] = two[0];
          out[ni][1] = two[1];
        }
      }
#pragma unroll
      for(int r0 = 0; r0 < 32; r0 += ROWS) {
        if(ROWS == 32 || (col >= r0 && col < r0 + ROWS)) {
          const int r = col - r0;
#pragma unroll
          for(int ni = 0; ni < NI; ni++)
#pragma unroll
            for(int j = 0; j < (OUT == DT_F32 ? 4 : 2); j++) {
              const int p = ni * (32 / PER) + 2 * j + hh;
              ldsWrite16(mine + (unsigned)(r * P + (p ^ (r & SWZ))) * 16, out[ni][j]);
            }
        }
        waveFence();  // (a wave's LDS instructions are carried out in order)
        const u32x4 v0 = ldsRead16(from), v1 = ldsRead16(from + 1024);
        waveFence();
        put(mi * 32 + r0, v0);
        put(mi * 32 + r0 + ROWS / 2, v1);
      }
    }
  };
  constexpr int STORES = MI * TN * 32 * (int)sizeof(TO) / 1024;  // a wave's store instructions of a whole tile
  static_assert(STORES <= 63, "vmcnt");
  auto allMild = [&](int parity) {  // of the scales that this wave's part is multiplied with
    if(MX) return true;
    const float* const sc = scalesOf + parity * (BM + BN);
    bool ok = true;
#pragma unroll
    for(int r = 0; r < TM; r += 64) ok = (r + lane >= TM || mild(sc[wm * TM + r + lane])) && ok;
#pragma unroll
    for(int c = 0; c < TN; c += 64) ok = (c + lane >= TN || mild(sc[BM + wn * TN + c + lane])) && ok;
    return !anyLane(!ok);
  };

  unsigned id = blockIdx.x;
  Tile tile = tileAt(id);
  aim(tile);
  if constexpr(MX) myCodes = (const uint8_t*)(ofA ? g.aScales : g.wScales) + scaleRow(tile) * blocks;
  fetchScales(tile);
  unsigned firstCodes = 0;
  if constexpr(MX) {
    firstCodes = fetchAny(0);
    fetched = fetchAny(1);
  }
#pragma unroll
  for(int k = 0; k < STAGES; k++) issue(k, k);
  putScales(0);
  if constexpr(MX) codesOf[codeRow] = shiftedCodes(firstCodes, blocks, 0);
  waitLoads<AHEAD>();
  waitReads0();
  waveBarrier();
  readCodes(0);
  readW(0, 0);
#pragma unroll
  for(int mi = 0; mi < MI; mi++) readA(0, 0, mi);
  int at = 0, tileParity = 0;
  for(;;) {
#pragma unroll
    for(int ni = 0; ni < NI; ni++)
#pragma unroll
      for(int mi = 0; mi < MI; mi++)
#pragma unroll
        for(int v = 0; v < 16; v++) acc[ni][mi][v] = 0.0f;
    // the stores of the tile before may still be under way at the first barrier: what it waits for was requested in front of them
    body(at++, 0, STAGES, 1, 2, Index<END>(), Index<STORES>());
    int step = 1;
    for(; step + STAGES + 1 < steps; step++) body(at++, step, step + STAGES, step + 1, step + 2, Index<INSIDE>(), Index<0>());
    pin();
    if(step + STAGES < steps) {
      body(at++, step, step + STAGES, step + 1, step + 2, Index<END>(), Index<0>());
      step++;
    }
    // the next tile is requested from here on (this one again where there is none: requested, not used)
    const bool last = id + gridDim.x >= allTiles;
    const Tile next = last ? tile : tileAt(id + gridDim.x);
    aim(next);
    if constexpr(STAGES > 2)
#pragma unroll 1
      for(int want = 0; want < STAGES - 2; want++, step++) body(at++, step, want, step + 1, step + 2, Index<END>(), Index<0>());
    if constexpr(MX) myCodes = (const uint8_t*)(ofA ? g.aScales : g.wScales) + scaleRow(next) * blocks;
    fetchScales(next);
    body(at++, step, STAGES - 2, step + 1, 0, Index<END>(), Index<0>());
    putScales(tileParity ^ 1);
    body(at++, step + 1, STAGES - 1, 0, 1, Index<END>(), Index<0>());
    const bool plain = __builtin_expect(allMild(tileParity), 1);
    if(__builtin_expect(plain && tile.mLast == BM - 1 && tile.nLast == BN - 1, 1)) store(tile, tileParity, Index<1>(), Index<0>());
    else {
      if(__builtin_expect(plain, 1)) store(tile, tileParity, Index<0>(), Index<0>());
      else store(tile, tileParity, Index<0>(), Index<1>());
      waitLoads<0>();  // (who knows how many of its lanes had something to store)
    }
    if(last) break;
    id += gridDim.x;
    tile = next;
    tileParity ^= 1;
  }
  waitLoads<0>();  // (nothing may land in LDS that is another work-group's by then)
}

// Short k, many rows: a work-group keeps 128 output channels, whose weights stay in its waves' registers (64 channels of up to 384 k each), and goes down its
// rows 128 at a time: only a's rows pass through LDS, in steps of 128 k, three of them on their way while one is multiplied. One barrier a step: behind
// it the stage before has been read out by all and is requested anew. Two work-groups share a CU, so that one's products run beside the other's
// results on their way out. The layouts are those of linear8Kernel; what lies beyond K has weights of zero. 92416 x 1152 x 384: 62 us (77 with linear8Kernel,
// which fetches the weights anew for every tile), of which products alone take 39, the results' way through LDS 20; k = 128: 41 us, 5.4 TB/s. k of 384 takes 236
// to 248 of the 256 registers that two work-groups to a CU leave a thread; 512 would need 64 more.
template <int KS, bool MX, int OUT>
__global__ __launch_bounds__(256, 2) void linear8ShortKernel(Linear8Args g, int groups) {
  typedef typename OutTraits<OUT>::TR TR;
  typedef typename TR::T TO;
  constexpr int BM = 128, BN = 128, NW = 4, MI = 2, NI = 2, REQ = BM / 8 / NW, STAGES = 4;
  constexpr unsigned STAGE = BM * KSTEP;
  HIP_DYNAMIC_SHARED(f32x4, smemLinear8)
  const unsigned lds = ldsAddress(smemLinear8);
  float* const scalesOf = (float*)((char*)smemLinear8 + STAGES * STAGE);  // [BN]
  float* const biasOf = scalesOf + BN;                                    // [BN]
  const unsigned patch = lds + STAGES * STAGE + 2 * BN * 4;               // 2 KB of each wave: what is being stored
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hh = lane >> 5;
  const int wm = wave >> 1, wn = wave & 1;
  const int pieces = g.K / 16, blocks = MX ? g.K / MX_BLOCK : 0;

  // Work-groups go round the 8 XCDs one by one: those of an XCD that follow each other share their rows and differ in their channels, so that a's
  // rows come from memory once
  const unsigned mTiles = (unsigned)((g.rows + BM - 1) / BM), nTiles = (unsigned)(g.N + BN - 1) / BN;
  const unsigned xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
  if(local >= groups * nTiles) return;
  const int n0 = (int)(local % nTiles) * BN;
  const unsigned group = xcd * groups + local / nTiles, allGroups = 8 * groups;
  const unsigned first = (unsigned)((uint64_t)mTiles * group / allGroups), end = (unsigned)((uint64_t)mTiles * (group + 1) / allGroups);
  if(first == end) return;
  const int nLast = (g.N - n0 < BN ? g.N - n0 : BN) - 1;
  auto lastRowOf = [&](unsigned tile) { return (int)(g.rows - (int64_t)tile * BM < BM ? g.rows - (int64_t)tile * BM : BM) - 1; };

  // weights, their codes, channel scales and biases
  u32x4 fw[KS][2][NI][2];
  unsigned wCodes[MX ? KS : 1][NI];
#pragma unroll
  for(int ni = 0; ni < NI; ni++) {
    const int c = wn * 64 + ni * 32 + col, row = n0 + (c < nLast ? c : nLast);
    const uint8_t* const wp = g.w + (int64_t)row * g.wStride;
#pragma unroll
    for(int k = 0; k < KS; k++) {
#pragma unroll
      for(int s = 0; s < 2; s++)
#pragma unroll
        for(int b = 0; b < 2; b++) {
          const int piece = k * KPIECES + 4 * s + 2 * b + hh;
          fw[k][s][ni][b] = *(const u32x4*)(wp + (size_t)(piece < pieces ? piece : pieces - 1) * 16);
          if(piece >= pieces) {
#pragma unroll
            for(int i = 0; i < 4; i++) fw[k][s][ni][b][i] = 0;
          }
        }
      if constexpr(MX) wCodes[k][ni] = *(const u32u*)((const uint8_t*)g.wScales + (int64_t)row * blocks + k * 4) >> (8 * hh);
    }
  }
  if(threadIdx.x < BN) {
    const int c = (int)threadIdx.x, n = n0 + (c < nLast ? c : nLast);
    scalesOf[c] = MX ? 1.0f : ((const float*)g.wScales)[n];
    biasOf[c] = g.bias != nullptr ? g.bias[n] : 0.0f;
  }

  const unsigned piece = (unsigned)((lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7));  // ((r >> 1) & 7 of every row that this lane requests)
  struct Request {
    Rsrc a;
    unsigned in, dst;
    int last;
  };
  auto requestOf = [&](unsigned at) {  // of step `at` of this work-group; beyond its last: that tile again, not used
    const unsigned tile = first + at / KS < end ? first + at / KS : end - 1;
    const int k = (int)(at % KS), over = k * KPIECES + (int)piece - (pieces - 1);
    Request r;
    r.a = bufferOf(g.a + (int64_t)tile * BM * g.aStride);
    r.in = (unsigned)k * KSTEP + piece * 16 - (over > 0 ? (unsigned)over * 16 : 0u);
    r.dst = lds + (at & (STAGES - 1)) * STAGE + (unsigned)wave * 8 * KSTEP;
    r.last = lastRowOf(tile);
    return r;
  };
  auto issue = [&](const Request& q, int j) {
    const int r = (wave + NW * j) * 8 + (lane >> 3);
    dma16(q.a, (unsigned)(r < q.last ? r : q.last) * (unsigned)g.aStride + q.in, 0, q.dst + (unsigned)(NW * j) * 8 * KSTEP);
  };
  constexpr int STORES = MI * 32 * 64 * (int)sizeof(TO) / 1024;  // a wave's store instructions of a whole tile
  auto store = [&](f32x16 (&acc)[NI][MI], const float (&sa)[MI], unsigned tile, auto wholeTag, auto anyTag) {
    constexpr bool WHOLE = decltype(wholeTag)::value != 0, ANY = decltype(anyTag)::value != 0;
    constexpr int PER = 8, P = 8, ROWS = 16;
    const unsigned mine = patch + (unsigned)wave * 2048;
    const int ln = anew(lane), col = ln & 31, hh = ln >> 5;
    const float* const sc = scalesOf + wn * 64;
    const float* const bi = biasOf + wn * 64;
    TO* const corner = (TO*)g.out + ((int64_t)tile * BM + wm * 64) * g.outStride + n0 + wn * 64;
    const int rowsLeft = lastRowOf(tile) - wm * 64, colsLeft = nLast - wn * 64;
    const unsigned from = mine + (unsigned)(ln / P * P + (ln % P ^ (ln / P & 7))) * 16;
    const unsigned mineTo = (unsigned)(ln / P) * (unsigned)g.outStride * (unsigned)sizeof(TO) + (unsigned)(ln % P) * 16;
    auto put = [&](int row0, u32x4 v) {
      if(WHOLE) countedStore();
      TO* const to = (TO*)((char*)(corner + (int64_t)row0 * g.outStride) + mineTo);
      if(WHOLE && KS > 1) streamOut(to, v);
      else if(WHOLE) *(Out16*)to = v;  // (k of 128: writing is all there is, and 92416 x 1152 take 41 us so, 47 past the caches)
      else if(row0 + ln / P <= rowsLeft) {
        const int c = ln % P * PER;
        if(c + PER - 1 <= colsLeft) *(Out16*)to = v;
        else {
          struct Elements { TO e[PER]; };
          const Elements e = __builtin_bit_cast(Elements, v);
#pragma unroll
          for(int k = 0; k < PER; k++)
            if(c + k <= colsLeft) to[k] = e.e[k];
        }
      }
    };
    u32x4 out[MI][NI][2];  // pieces of channels 16 j + 8 hh + [0, 8)
#pragma unroll
    for(int ni = 0; ni < NI; ni++) {
      u32x2 pk[MI][4];
#pragma unroll
      for(int q = 0; q < 4; q++) {
        const f32x4 bias = *(const f32x4*)(bi + ni * 32 + 8 * q + 4 * hh);
        f32x4 sw = bias;
        if(!MX) sw = *(const f32x4*)(sc + ni * 32 + 8 * q + 4 * hh);
#pragma unroll
        for(int mi = 0; mi < MI; mi++) {
          typename TR::V4 h;
#pragma unroll
          for(int i = 0; i < 4; i++) {
            const float sum = acc[ni][mi][4 * q + i];
            h[i] = TR::fromFloat((MX ? sum : ANY ? scaledByAny(sum, sa[mi], sw[i]) : sum * sa[mi] * sw[i]) + bias[i]);
          }
          pk[mi][q] = __builtin_bit_cast(u32x2, h);
        }
      }
#pragma unroll
      for(int mi = 0; mi < MI; mi++) pairUp(pk[mi], out[mi][ni]);
    }
#pragma unroll
    for(int r0 = 0; r0 < 32 * MI; r0 += ROWS) {
      if(col >= r0 % 32 && col < r0 % 32 + ROWS) {
        const int r = col - r0 % 32;
#pragma unroll
        for(int ni = 0; ni < NI; ni++)
#pragma unroll
          for(int j = 0; j < 2; j++) {
            const int p = ni * 4 + 2 * j + hh;
            ldsWrite16(mine + (unsigned)(r * P + (p ^ (r & 7))) * 16, out[r0 / 32][ni][j]);
          }
      }
      waveFence();  // (a wave's LDS instructions are carried out in order)
      const u32x4 v0 = ldsRead16(from), v1 = ldsRead16(from + 1024);
      waveFence();
      put(r0, v0);
      put(r0 + ROWS / 2, v1);
    }
  };

#pragma unroll
  for(unsigned k = 0; k < 3; k++) {
    const Request q = requestOf(k);
#pragma unroll
    for(int j = 0; j < REQ; j++) issue(q, j);
  }
  waitLoads<0>();
  const unsigned swz = (unsigned)(col >> 1) & 7u;
  unsigned at = 0;
  // a's scales (or codes) are fetched a tile ahead: in front of the stores of the tile before, which a load has to wait for
  float saNext[MI];
  unsigned codesNext[MX ? KS : 1][MI];
  auto fetchScales = [&](unsigned tile) {
    const int last = lastRowOf(tile);
#pragma unroll
    for(int mi = 0; mi < MI; mi++) {
      const int r = wm * 64 + mi * 32 + col;
      const int64_t row = (int64_t)tile * BM + (r < last ? r : last);
      saNext[mi] = MX ? 1.0f : ((const float*)g.aScales)[row];
      if constexpr(MX) {
#pragma unroll
        for(int k = 0; k < KS; k++) codesNext[k][mi] = *(const u32u*)((const uint8_t*)g.aScales + row * blocks + k * 4);
      }
    }
  };
  fetchScales(first);
  for(unsigned tile = first; tile < end; tile++) {
    float sa[MI];
    unsigned aCodes[MX ? KS : 1][MI];
#pragma unroll
    for(int mi = 0; mi < MI; mi++) {
      sa[mi] = saNext[mi];
      if constexpr(MX) {
#pragma unroll
        for(int k = 0; k < KS; k++) aCodes[k][mi] = codesNext[k][mi] >> (8 * hh);
      }
    }
    f32x16 acc[NI][MI];
#pragma unroll
    for(int ni = 0; ni < NI; ni++)
#pragma unroll
      for(int mi = 0; mi < MI; mi++)
#pragma unroll
        for(int v = 0; v < 16; v++) acc[ni][mi][v] = 0.0f;
    auto step = [&](auto kTag) {
      constexpr int k = decltype(kTag)::value;
      // Younger than what this step multiplies are the requests of the next two and the stores of the tiles in between: a tile whose stores cannot be
      // counted waits for all of them
      constexpr int TILES = KS == 1 ? 3 : KS == 2 ? 2 - k : 1;
      waitLoads<2 * REQ + TILES * STORES>();
      waitReads0();
      waveBarrier();
      if constexpr(k == 0) fetchScales(tile + 1 < end ? tile + 1 : tile);
      const Request q = requestOf(at + 3);
      const unsigned rows = lds + (at & (STAGES - 1)) * STAGE + (unsigned)(wm * 64 + col) * KSTEP;
      u32x4 fa[MI][2][2];
#pragma unroll
      for(int mi = 0; mi < MI; mi++)
#pragma unroll
        for(int s = 0; s < 2; s++)
#pragma unroll
          for(int b = 0; b < 2; b++) fa[mi][s][b] = ldsRead16(rows + mi * 32 * KSTEP + (((unsigned)(4 * s + 2 * b + hh)) ^ swz) * 16);
#pragma unroll
      for(int mi = 0; mi < MI; mi++)
#pragma unroll
        for(int s = 0; s < 2; s++)
#pragma unroll
          for(int ni = 0; ni < NI; ni++) {
            constexpr int UNIT = 0x7f7f7f7f;
            i32x8 xa, xw;
#pragma unroll
            for(int i = 0; i < 8; i++) {
              xa[i] = (int)fa[mi][s][i >> 2][i & 3];
              xw[i] = (int)fw[k][s][ni][i >> 2][i & 3];
            }
            if(s == 0)
              acc[ni][mi] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xw, xa, acc[ni][mi], 0, 0, 0, MX ? (int)wCodes[MX ? k : 0][ni] : UNIT, 0,
                                                                            MX ? (int)aCodes[MX ? k : 0][mi] : UNIT);
            else
              acc[ni][mi] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xw, xa, acc[ni][mi], 0, 0, 2, MX ? (int)wCodes[MX ? k : 0][ni] : UNIT, 2,
                                                                            MX ? (int)aCodes[MX ? k : 0][mi] : UNIT);
            if(ni == NI - 1) {  // (requests hold a wave's issue for as long as a product takes: one after two of them)
              __builtin_amdgcn_sched_barrier(0);
              issue(q, mi * 2 + s);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
      static_assert(REQ == 2 * MI, "a request to each half's products");
#pragma unroll
      for(int ni = 0; ni < NI; ni++)
#pragma unroll
        for(int mi = 0; mi < MI; mi++) computed(acc[ni][mi]);
      at++;
    };
    step(Index<0>());
    if constexpr(KS > 1) step(Index<1>());
    if constexpr(KS > 2) step(Index<2>());
    bool plain = true;
    if constexpr(!MX) {
      bool ok = mild(scalesOf[wn * 64 + lane]);
#pragma unroll
      for(int mi = 0; mi < MI; mi++) ok = mild(sa[mi]) && ok;
      plain = !anyLane(!ok);
    }
    if(plain && lastRowOf(tile) == BM - 1 && nLast == BN - 1) store(acc, sa, tile, Index<1>(), Index<0>());
    else {
      if(plain) store(acc, sa, tile, Index<0>(), Index<0>());
      else store(acc, sa, tile, Index<0>(), Index<1>());
      waitLoads<0>();
    }
  }
  waitLoads<0>();  // (nothing may land in LDS that is another work-group's by then)
}

// Few rows: the time is the weights' way from memory, so they go straight into registers, a wave's share of DEPTH steps in one round of requests. (With e8m0 scales
// all of a round's requests are out before its first product; with row scales the compiler moves some behind it: 12 of 16 are out ahead for 16 rows, 6 of 12
// for 32, 6 of 20 for 64. A second round is requested when the first has been multiplied.) A work-group owns 16 output
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
    if(!MX) x = scaledByAny(x, ((const float*)g.aScales)[m0 + r], ((const float*)g.wScales)[n0 + c]);
    if(g.bias != nullptr) x += g.bias[n0 + c];
    ((TO*)g.out)[(m0 + r) * g.outStride + n0 + c] = TR::fromFloat(x);
  }
}

template <int MT, bool MX, int OUT>
hipError_t launchFew(const Linear8Args& g, hipStream_t stream) {
  return launchKernel(linear8FewKernel<MT, MX, OUT>, dim3((unsigned)((g.N + 15) / 16), (unsigned)((g.rows + 16 * MT - 1) / (16 * MT))), dim3(512), 0, stream, g);
}
// The current device's compute units, asked for once per instantiation and device (cus: 0 until then); a kernel's large LDS window is opted in to there
constexpr int MAX_DEVICES = 64;
template <class K>
hipError_t prepared(K kern, int lds, std::atomic<int>* cus, int* n) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if(e != hipSuccess) return e;
  if(dev < 0 || dev >= MAX_DEVICES) return hipErrorInvalidDevice;
  *n = cus[dev].load(std::memory_order_acquire);
  if(*n != 0) return hipSuccess;
  if(lds > 64 * 1024) {
    e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if(e != hipSuccess) return e;
  }
  e = computeUnits(dev, n);
  if(e != hipSuccess) return e;
  cus[dev].store(*n, std::memory_order_release);
  return hipSuccess;
}
template <int BM, int BN, int WM, int WN, int STAGES, bool MX, int OUT>
hipError_t launchTile(const Linear8Args& g, hipStream_t stream) {
  const int64_t tiles = (g.rows + BM - 1) / BM * ((g.N + BN - 1) / BN);
  if(tiles > 0x7fffffff) return hipErrorInvalidValue;
  constexpr int LDS = STAGES * (BM + BN) * KSTEP + (2 * (BM + BN) + 2 * BN) * 4 + WM * WN * 2048, ALL_LDS = 160 * 1024;
  constexpr int PER_CU = ALL_LDS / LDS < 4 ? ALL_LDS / LDS : 4;  // work-groups of a CU
  static_assert(PER_CU >= 1, "LDS");
  auto kern = linear8Kernel<BM, BN, WM, WN, STAGES, MX, OUT>;
  static std::atomic<int> cus[MAX_DEVICES];
  int n = 0;
  const hipError_t e = prepared(kern, LDS, cus, &n);
  if(e != hipSuccess) return e;
  const int64_t most = (int64_t)n * PER_CU / 8 * 8;  // (a multiple of the XCDs: a work-group's tiles stay on its XCD's part)
  return launchKernel(kern, dim3((unsigned)(tiles < most ? tiles : most)), dim3(64 * WM * WN), LDS, stream, g);
}
template <int KS, bool MX, int OUT>
hipError_t launchShort(const Linear8Args& g, int groups, hipStream_t stream) {
  constexpr int LDS = 4 * 128 * KSTEP + 2 * 128 * 4 + 4 * 2048;
  auto kern = linear8ShortKernel<KS, MX, OUT>;
  static std::atomic<int> cus[MAX_DEVICES];
  int n = 0;
  const hipError_t e = prepared(kern, LDS, cus, &n);
  if(e != hipSuccess) return e;
  return launchKernel(kern, dim3((unsigned)(8 * groups * ((g.N + 127) / 128))), dim3(256), LDS, stream, g, groups);
}
template <bool MX, int OUT>
hipError_t launchShape(const Linear8Args& g, hipStream_t stream) {
  // Few rows: up to 32 on the kernel without LDS (32 x 4096 x 4096 8.1 us; 64 rows 11.7 against 10.0 on 64 x 64 tiles with four stages), up to 64 where k
  // is too short for those to get going (64 x 1152 x 384 3.0 us against 3.8).
  const bool longK = g.K >= 8 * KSTEP;
  // k that fits the registers, and rows enough: ten tiles of 128 rows to a work-group (12.9 of them, 92416 x 1152 x 384: 68 us against 77 when the rule was
  // made; 11.3, n = 1024: equal; 4.3, n = 384: 28 against 26.7; two, 14500 x 1152: 18.7 against 15.4). About 512 work-groups share the chip, so that is 84
  // million results and more.
  if constexpr(OUT != DT_F32) {
    const int64_t groups = PER_XCD / ((g.N + 127) / 128);  // of work-groups that share their rows, on an XCD
    if(g.K <= 3 * KSTEP && (!MX || g.K % KSTEP == 0) && groups >= 1 && (g.rows + 127) / 128 >= SHORT_TILES * 8 * groups) {
      if(g.K <= KSTEP) return launchShort<1, MX, OUT>(g, (int)groups, stream);
      if(g.K <= 2 * KSTEP) return launchShort<2, MX, OUT>(g, (int)groups, stream);
      return launchShort<3, MX, OUT>(g, (int)groups, stream);
    }
  }
  if(g.rows <= 16) return launchFew<1, MX, OUT>(g, stream);
  if(g.rows <= 32) return launchFew<2, MX, OUT>(g, stream);
  if(g.rows <= 64 && !longK) return launchFew<4, MX, OUT>(g, stream);
  // A CU holds one work-group of the 256 x 256 tile or two of the 128 x 128: rounds of such sets until all tiles are done, a round of the large
  // tile measured at 1.6 of a small one's (8192^3: 105 us and 66). The large tile where it needs less time and its edges waste little (92416 rows,
  // k = 384: n = 1152 in 84 us against 89, but n = 384, half of its second tile empty, in 34 against 28); the small one while there is a
  // round of it - with one work-group to a CU four stages, which hide a request's time better (1000 x 4096 x 4096 27.1 -> 24.0 us);
  // below that 64 x 64, with four stages where k is long (128 x 4096 x 4096 16.8 -> 10.0 us, 361 x 1152 x 384 3.8 -> 4.9).
  const int64_t cus = chosenFor();
  auto tiles = [&](int b) { return (g.rows + b - 1) / b * ((g.N + b - 1) / b); };
  const int64_t large = tiles(256), small = tiles(128);
  if constexpr(OUT != DT_F32)
    if((large + cus - 1) / cus * 8 < (small + 2 * cus - 1) / (2 * cus) * 5 && large * 4 * 20 < small * 23)
      return launchTile<256, 256, 2, 4, 2, MX, OUT>(g, stream);
  if(small > cus) return launchTile<128, 128, 2, 2, 2, MX, OUT>(g, stream);
  if(!longK) return launchTile<64, 64, 2, 2, 2, MX, OUT>(g, stream);
  if(small * 8 > cus * 5) return launchTile<128, 128, 2, 2, 4, MX, OUT>(g, stream);
  return launchTile<64, 64, 2, 2, 4, MX, OUT>(g, stream);
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
