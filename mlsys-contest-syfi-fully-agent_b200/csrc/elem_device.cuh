// Element types and small device functions shared by the operators around the shard (norms, balance loss, 4-bit
// products): conversion between the three activation types and fp32, loads of eight elements, sums over a CTA.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/moe_b200.h"
#include "kernels.h"

namespace moe {

// Host side: what a launch returns to the caller, and the checks of types and alignment.
inline int launch_status(cudaError_t e, int launches) {
  if (e != cudaSuccess) {
    set_last_cuda_error(static_cast<int>(e));
    return MOE_B200_ECUDA;
  }
  count_launches(launches);
  return MOE_B200_OK;
}
inline int element_size(int dtype) { return dtype == MOE_B200_F32 ? 4 : 2; }
inline bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// One rounding, to nearest even, where a result leaves fp32.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Eight elements as they lie in memory (16 or 32 bytes).
template <typename T>
struct alignas(16) Pack8 {
  T v[8];
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

// Sums of N values over the CTA, the same bits in every thread.  `red` holds N * 32 floats that no other reduction in
// flight uses: one barrier per call, so consecutive calls alternate between two areas.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* red) {
  const int warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.0f;
    for (int w = 0; w < nwarps; ++w) s += red[i * 32 + w];
    v[i] = s;
  }
}

}  // namespace moe
