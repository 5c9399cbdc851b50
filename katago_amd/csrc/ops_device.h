// ops_device.h — what the kernels of the operators on device buffers share
#ifndef KMX_OPS_DEVICE_H_
#define KMX_OPS_DEVICE_H_

#include <tuple>

#include "device_common.h"

namespace kmx {

// A launch, and ITS error: what an earlier call of the program left for hipGetLastError() stays there, and is not reported as this one's. An error of the
// launch is returned, and not left for others to find.
template <class... P, class... A>
hipError_t launchKernel(void (*kern)(P...), dim3 grid, dim3 block, int lds, hipStream_t stream, const A&... args) {
  static_assert(sizeof...(P) == sizeof...(A), "arguments");
#ifdef KMX_EMULATED_HIP
  hipLaunchKernelGGL(kern, grid, block, lds, stream, args...);
  return hipSuccess;
#else
  std::tuple<P...> copies(args...);
  return std::apply([&](P&... p) {
    void* at[] = {(void*)&p...};
    const hipError_t e = hipLaunchKernel((const void*)kern, grid, block, at, (size_t)lds, stream);
    if(e != hipSuccess) (void)hipGetLastError();
    return e;
  }, copies);
#endif
}

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
