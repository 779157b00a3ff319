// Element types and small device functions shared by the operators around the shard (norms, balance loss, 4-bit
// products): conversion between the three activation types and fp32, loads of eight elements, sums over a CTA.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

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
// Lets `kernel` have up to `bytes` of dynamic shared memory on the current device; `done` (a static of the caller, one per
// kernel) remembers the devices where that has been said, a driver call that would cost a small launch a tenth of its time.
template <typename Kernel>
inline cudaError_t allow_smem(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess && device < 64) done.fetch_or(bit, std::memory_order_release);
  return e;
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

// Two fp32 values in a register pair: sm_100's packed instructions do both for one issue slot.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 make_f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 get(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 both(float v) { return make_f2(v, v); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float total(F2 a) {
  const float2 f = get(a);
  return f.x + f.y;
}

// Eight elements as they lie in memory (one or two 16-byte words), and the conversion of all of them at once.
template <typename T>
struct alignas(16) Pack8 {
  uint4 w[sizeof(T) / 2];
};
__device__ __forceinline__ F2 unpack2(uint32_t v, __nv_bfloat16) { return make_f2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
__device__ __forceinline__ F2 unpack2(uint32_t v, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return make_f2(f.x, f.y);
}
__device__ __forceinline__ uint32_t pack2(F2 a, __nv_bfloat16) {
  const float2 f = get(a);
  const __nv_bfloat162 p = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(F2 a, __half) {
  const float2 f = get(a);
  const __half2 p = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <typename T>
__device__ __forceinline__ void unpack8(const Pack8<T>& p, F2 (&v)[4]) {
  v[0] = unpack2(p.w[0].x, T());
  v[1] = unpack2(p.w[0].y, T());
  v[2] = unpack2(p.w[0].z, T());
  v[3] = unpack2(p.w[0].w, T());
}
template <>
__device__ __forceinline__ void unpack8<float>(const Pack8<float>& p, F2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[2 * i] = make_f2(__uint_as_float(p.w[i].x), __uint_as_float(p.w[i].y));
    v[2 * i + 1] = make_f2(__uint_as_float(p.w[i].z), __uint_as_float(p.w[i].w));
  }
}
template <typename T>
__device__ __forceinline__ Pack8<T> pack8(const F2 (&v)[4]) {
  return {{make_uint4(pack2(v[0], T()), pack2(v[1], T()), pack2(v[2], T()), pack2(v[3], T()))}};
}
template <>
__device__ __forceinline__ Pack8<float> pack8<float>(const F2 (&v)[4]) {
  Pack8<float> p;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 lo = get(v[2 * i]), hi = get(v[2 * i + 1]);
    p.w[i] = make_uint4(__float_as_uint(lo.x), __float_as_uint(lo.y), __float_as_uint(hi.x), __float_as_uint(hi.y));
  }
  return p;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

// sum += v, and what the sum's last bit cannot hold goes to `lost` (the error of an addition, after Knuth).  Only for sums of
// sums: the chain of additions is as long as without it.
__device__ __forceinline__ void add_exactly(float& sum, float& lost, float v) {
  const float s = sum + v, b = s - sum;
  lost += (sum - (s - b)) + (v - b);
  sum = s;
}
// The two joined; an infinite or undefined sum has nothing to add.
__device__ __forceinline__ float joined(float sum, float lost) { return isfinite(lost) ? sum + lost : sum; }

// Sums of N values over the CTA, the same bits in every thread.  `red` holds N * 32 floats that no other reduction in
// flight uses: one barrier per call, so consecutive calls alternate between two areas.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < nwarps ? red[i * 32 + lane] : 0.0f);
}

// Asynchronous copies to shared memory (cp.async).  copy16 past the caches' first level, zeros where !there.
__device__ __forceinline__ uint32_t smem_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

}  // namespace moe
