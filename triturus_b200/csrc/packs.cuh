// What the kernels of the operators around the contractions share: vectors of 32- or 16-bit floats moved as one access,
// reductions over a block in a fixed order, launches, and the SM count.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/triturus_b200.h"

namespace tb200 {

// The library's code for a CUDA call.  CUDA keeps an error until it is asked for: one that is reported here is not left for
// a later call to find.
inline int code_of(cudaError_t rc) {
  if (rc == cudaSuccess) return TRITURUS_B200_OK;
  cudaGetLastError();
  return TRITURUS_B200_ELAUNCH;
}
// A launch whose own error is returned, and no earlier one that was left.
template <class... Params, class... Args>
int launch_of(void (*kern)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const cudaLaunchAttribute* attribute, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attribute);
  cfg.numAttrs = attribute != nullptr ? 1 : 0;
  return code_of(cudaLaunchKernelEx(&cfg, kern, static_cast<Args&&>(args)...));
}
inline cudaLaunchAttribute dependent_launch() {
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  return at;
}
inline cudaLaunchAttribute cluster_of(int blocks) {
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(blocks);
  at.val.clusterDim.y = 1;
  at.val.clusterDim.z = 1;
  return at;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

// BYTES / sizeof(T) consecutive elements: one load or store where the address is a multiple of BYTES.
template <class T, int BYTES>
struct alignas(BYTES) Pack {
  static constexpr int N = BYTES / static_cast<int>(sizeof(T));
  T v[N];
};

// The sum over a block of `warps` warps, the same in every thread and always added in the same order.  `part` holds a value
// for each warp; a caller that reduces again before its next barrier uses another array.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* part, int warp, int lane, int warps) {
  v = warp_sum(v);
  if (lane == 0) part[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? part[lane] : 0.f);
}

inline int device_sms() {
  static int sms[64] = {};
  int dev = 0;
  if (code_of(cudaGetDevice(&dev)) != TRITURUS_B200_OK || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) {
    int n = 0;
    sms[dev] = code_of(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev)) == TRITURUS_B200_OK && n > 0 ? n : 148;
  }
  return sms[dev];
}

inline bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0; }

}  // namespace tb200
