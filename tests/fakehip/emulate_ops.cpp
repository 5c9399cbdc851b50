// TEST INFRASTRUCTURE: the operators of include/katamx_ops.h - norm_quant.hip, linear8.hip, rotary.hip and ops_api.cpp - compiled for the host and
// executed on the CPU (see emul/hip/hip_runtime.h), behind their own C entry points: "device" pointers are host pointers here.
// tests/test_ops_emulated.py compares them with plain formulas in 64 bits: indexing, masks, tails, refusals, before a GPU sees them. Nothing in the
// product links or loads this file.
#include <hip/hip_runtime.h>  // the stand-in (-I tests/fakehip/emul)

#include <stdexcept>

// Three devices, of which a thread has a current one; a launch notes which that was
namespace emu {
inline thread_local int currentDevice = 0, launchedOn = -1;
inline hipError_t countDevices(int* n) {
  *n = 3;
  return hipSuccess;
}
inline hipError_t getDevice(int* d) {
  *d = currentDevice;
  return hipSuccess;
}
inline hipError_t setDevice(int d) {
  if(d < 0 || d >= 3) return hipErrorInvalidDevice;
  currentDevice = d;
  return hipSuccess;
}
}  // namespace emu
#define hipGetDeviceCount emu::countDevices
#define hipGetDevice emu::getDevice
#define hipSetDevice emu::setDevice
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(kern, grid, block, lds, stream, ...) (emu::launchedOn = emu::currentDevice, emu::launchImpl(grid, block, [&] { kern(__VA_ARGS__); }))
extern "C" int emu_launched_on(void) { return emu::launchedOn; }
extern "C" int emu_current_device(void) { return emu::currentDevice; }
extern "C" void emu_make_current(int device) { emu::currentDevice = device; }

namespace emu {
inline float decodeE4m3(unsigned v) {
  const unsigned e = (v >> 3) & 15, m = v & 7;
  float r = e ? ldexpf(1.0f + m / 8.0f, (int)e - 7) : ldexpf((float)m, -9);
  if(e == 15 && m == 7) r = NAN;
  return v & 0x80 ? -r : r;
}
inline unsigned encodeE4m3(float x) {  // nearest even; beyond 464 and NaN: NaN
  const unsigned sign = std::signbit(x) ? 0x80u : 0u;
  const float a = fabsf(x);
  if(!(a < 464.0f)) return a == 464.0f ? sign | 0x7e : sign | 0x7f;
  int e;
  frexpf(a, &e);  // a = m 2^e, m in [1/2, 1)
  e = a == 0.0f || e - 1 < -6 ? -6 : e - 1;
  int q = (int)nearbyintf(ldexpf(a, 3 - e));  // in steps of 2^(e - 3)
  if(e == -6 && q < 8) return sign | (unsigned)q;
  if(q == 16) {
    q = 8;
    e++;
  }
  return sign | (unsigned)((e + 7) << 3) | (unsigned)(q - 8);
}
inline int cvtPkFp8(float a, float b, int old, bool hi) {
  const unsigned v = encodeE4m3(a) | encodeE4m3(b) << 8;
  return hi ? (int)(((unsigned)old & 0xffffu) | v << 16) : (int)(((unsigned)old & 0xffff0000u) | v);
}
typedef __bf16 Bf2 __attribute__((ext_vector_type(2)));
inline Bf2 cvtBf16Fp8(unsigned src, float scale, bool hi) {
  Bf2 r;
  r[0] = (__bf16)(decodeE4m3(src >> (hi ? 16 : 0) & 255) * scale);
  r[1] = (__bf16)(decodeE4m3(src >> (hi ? 24 : 8) & 255) * scale);
  return r;
}
inline float ofE8m0(int code) { return (code & 255) == 255 ? NAN : ldexpf(1.0f, (code & 255) - 127); }
// v_mfma_scale_f32_32x32x64_f8f6f4 on e4m3: lane (row or column l % 32, part l / 32) holds k = 16 part + [0, 16) in its first 16 bytes and 32 + 16
// part + [0, 16) in the others; the scale of k 0..31 is that of the lane with part 0, of k 32..63 that of part 1 (byte 0 of the operand).
template <class I8, class F16>
inline F16 mfmaScale(I8 a, I8 b, F16 c, int sa, int sb) {
  Wave& w = cur->waves[tIdx.x >> 6];
  const unsigned lane = tIdx.x & 63;
  uint8_t av[64][32], bv[64][32];
  int as[64], bs[64];
  {
    const unsigned set = waveOp++ & 1;
    memcpy(&w.opA[set][lane][0], &a, 32);
    memcpy(&w.opB[set][lane][0], &b, 32);
    w.bar->arrive_and_wait();
    memcpy(av, w.opA[set], sizeof(av));
    memcpy(bv, w.opB[set], sizeof(bv));
  }
  {
    const unsigned set = waveOp++ & 1;
    memcpy(&w.opA[set][lane][0], &sa, 4);
    memcpy(&w.opB[set][lane][0], &sb, 4);
    w.bar->arrive_and_wait();
    for(int l = 0; l < 64; l++) {
      memcpy(&as[l], &w.opA[set][l][0], 4);
      memcpy(&bs[l], &w.opB[set][l][0], 4);
    }
  }
  const unsigned col = lane & 31, half = lane >> 5;
  for(int v = 0; v < 16; v++) {
    const unsigned row = (v / 4) * 8 + half * 4 + (v % 4);
    double sum = 0;
    for(int blk = 0; blk < 2; blk++) {
      double part = 0;
      for(int p = 0; p < 2; p++)
        for(int i = 0; i < 16; i++) part += (double)decodeE4m3(av[row + 32 * p][16 * blk + i]) * decodeE4m3(bv[col + 32 * p][16 * blk + i]);
      sum += part * ofE8m0(as[row + 32 * blk]) * ofE8m0(bs[col + 32 * blk]);
    }
    c[v] += (float)sum;
  }
  return c;
}
// v_mfma_scale_f32_16x16x128_f8f6f4 on e4m3: lane (row or column l % 16, part l / 16) holds k = 16 part + [0, 16) and 64 + 16 part + [0, 16); the scale of
// k 32 b + [0, 32) is that of part b. C element v of a lane: row 4 part + v, column l % 16.
template <class I8, class F4>
inline F4 mfmaScale16(I8 a, I8 b, F4 c, int sa, int sb) {
  Wave& w = cur->waves[tIdx.x >> 6];
  const unsigned lane = tIdx.x & 63;
  uint8_t av[64][32], bv[64][32];
  int as[64], bs[64];
  {
    const unsigned set = waveOp++ & 1;
    memcpy(&w.opA[set][lane][0], &a, 32);
    memcpy(&w.opB[set][lane][0], &b, 32);
    w.bar->arrive_and_wait();
    memcpy(av, w.opA[set], sizeof(av));
    memcpy(bv, w.opB[set], sizeof(bv));
  }
  {
    const unsigned set = waveOp++ & 1;
    memcpy(&w.opA[set][lane][0], &sa, 4);
    memcpy(&w.opB[set][lane][0], &sb, 4);
    w.bar->arrive_and_wait();
    for(int l = 0; l < 64; l++) {
      memcpy(&as[l], &w.opA[set][l][0], 4);
      memcpy(&bs[l], &w.opB[set][l][0], 4);
    }
  }
  const unsigned col = lane & 15, part = lane >> 4;
  for(int v = 0; v < 4; v++) {
    const unsigned row = 4 * part + v;
    double sum = 0;
    for(int k = 0; k < 128; k++) {
      const int p = k % 64 / 16, i = k / 64 * 16 + k % 16, blk = k / 32;
      sum += (double)decodeE4m3(av[row + 16 * p][i]) * decodeE4m3(bv[col + 16 * p][i]) * ofE8m0(as[row + 16 * blk]) * ofE8m0(bs[col + 16 * blk]);
    }
    c[v] += (float)sum;
  }
  return c;
}
// v_mfma_f32_16x16x32_bf16: lane (row or column l % 16, part l / 16) holds k = 8 part + [0, 8)
template <class V8, class F4>
inline F4 mfma16x16(V8 a, V8 b, F4 c) {
  Wave& w = cur->waves[tIdx.x >> 6];
  const unsigned lane = tIdx.x & 63, set = waveOp++ & 1;
  for(int i = 0; i < 8; i++) {
    w.opA[set][lane][i] = (float)a[i];
    w.opB[set][lane][i] = (float)b[i];
  }
  w.bar->arrive_and_wait();
  for(int v = 0; v < 4; v++) {
    float sum = 0.0f;
    for(int p = 0; p < 4; p++)
      for(int i = 0; i < 8; i++) sum += w.opA[set][4 * (lane >> 4) + v + 16 * p][i] * w.opB[set][(lane & 15) + 16 * p][i];
    c[v] += sum;
  }
  return c;
}
}  // namespace emu
#define __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, hi) emu::cvtPkFp8(a, b, old, hi)
#define __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, scale, hi) emu::cvtBf16Fp8(src, scale, hi)
#define __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, fa, fb, oa, sa, ob, sb) emu::mfmaScale(a, b, c, (int)((unsigned)(sa) >> (8 * (oa))), (int)((unsigned)(sb) >> (8 * (ob))))

#define __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, fa, fb, oa, sa, ob, sb) \
  emu::mfmaScale16(a, b, c, (int)((unsigned)(sa) >> (8 * (oa))), (int)((unsigned)(sb) >> (8 * (ob))))
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) emu::mfma16x16(a, b, c)

#include "../../katago_amd/csrc/norm_quant.hip"
#include "../../katago_amd/csrc/linear8.hip"
#include "../../katago_amd/csrc/rotary.hip"
#include "../../katago_amd/csrc/ops_api.cpp"

#include "emul/emu_runtime.inc"

namespace {
thread_local std::string lastError;
}
namespace kmx {
void hipCheck(hipError_t e, const char* what) {
  if(e != hipSuccess) throw Error(KMX_ERR_DEVICE, what);
}
int apiGuarded(const std::function<void()>& f) {
  try {
    f();
    return KMX_OK;
  }
  catch(const Error& e) {
    lastError = e.what();
    return e.code;
  }
}
}  // namespace kmx
extern "C" const char* kmx_last_error(void) { return lastError.c_str(); }
