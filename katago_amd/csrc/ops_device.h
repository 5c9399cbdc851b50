// ops_device.h — what the kernels of the operators on device buffers share
#ifndef KMX_OPS_DEVICE_H_
#define KMX_OPS_DEVICE_H_

#include "device_common.h"

namespace kmx {

// Has any lane of the wave x?
#ifdef KMX_EMULATED_HIP
inline bool anyLane(bool x) {
  float v = x ? 1.0f : 0.0f;
  for(int o = 1; o < 64; o <<= 1) {
    const float u = __shfl_xor(v, o);
    v = u > v ? u : v;
  }
  return v != 0.0f;
}
#else
__device__ __forceinline__ bool anyLane(bool x) { return __builtin_amdgcn_ballot_w64(x) != 0; }
#endif

}  // namespace kmx
#endif
