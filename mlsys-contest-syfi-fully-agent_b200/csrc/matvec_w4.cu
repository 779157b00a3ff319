// Matrix-vector products with 4-bit weights and group scales, for decode-sized batches, dense or by chosen experts:
//     out[r, n] = sum_k x[row(r), k] (q[e(r), n, k] - z[e(r), n, k / G]) scale[e(r), n, k / G]
// q: two values a byte, the even k in the low half; z: 8 without a table.  Pair r = (token, choice) reads row r / per_row
// of x and expert experts[r]; a pair whose expert is not held here gives a zero row.  Sums are fp32; q - z is exact and
// the scale multiplies the fp32 sum of its group.
#include "elem_device.cuh"

namespace moe {
namespace {

constexpr int kMaxPairs = 256;
constexpr int kRowWarps = 8;

struct MatvecArgs {
  const void* x;
  int64_t x_stride;
  const uint8_t* q;          // [E, N, K / 2]
  const void* scale;         // [E, N, K / G]
  const uint8_t* zero;       // [E, N, K / G] or null
  const int* experts;        // [pairs] or null
  int pairs, per_row, E, N, K, G, scale_f32;
  void* out;                 // [pairs, N]
};

// One warp per output element; a lane takes eight consecutive weights (four bytes) at a time.
template <typename T, typename O>
__global__ void __launch_bounds__(32 * kRowWarps) matvec_w4_kernel(MatvecArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, n = blockIdx.x * kRowWarps + (threadIdx.x >> 5), r = blockIdx.y;
  if (n >= a.N) return;
  const int e = a.experts ? a.experts[r] : 0;
  float sum = 0.0f;
  if (e >= 0 && e < a.E) {
    const int64_t wrow = static_cast<int64_t>(e) * a.N + n;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(a.q + wrow * (a.K / 2));
    const T* x = static_cast<const T*>(a.x) + (r / a.per_row) * a.x_stride;
    const int groups = a.K / a.G;
    for (int i = lane; i < a.K / 8; i += 32) {
      const uint32_t v = q[i];
      const int64_t g = wrow * groups + i * 8 / a.G;
      const float z = a.zero ? static_cast<float>(a.zero[g]) : 8.0f;
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        part += (static_cast<float>((v >> (4 * j)) & 15u) - z) * to_f32<T>(x[i * 8 + j]);
      sum += part * (a.scale_f32 ? static_cast<const float*>(a.scale)[g] : to_f32<T>(static_cast<const T*>(a.scale)[g]));
    }
    sum = warp_sum(sum);
  }
  if (lane == 0) static_cast<O*>(a.out)[static_cast<int64_t>(r) * a.N + n] = from_f32<O>(sum);
}

template <typename T>
cudaError_t launch_matvec(const MatvecArgs& a, bool out_f32, cudaStream_t stream) {
  const dim3 grid((a.N + kRowWarps - 1) / kRowWarps, a.pairs), block(32 * kRowWarps);
  if (out_f32) return launch_pdl(matvec_w4_kernel<T, float>, grid, block, 0, stream, a);
  return launch_pdl(matvec_w4_kernel<T, T>, grid, block, 0, stream, a);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_fp8_block_scale_matvec_w4(const void* x, int64_t x_stride, int dtype, const uint8_t* qweight,
                                             const void* scale, int scale_f32, const uint8_t* zero, const int32_t* experts,
                                             int pairs, int pairs_per_row, int E, int N, int K, int G, void* out,
                                             int out_f32, void* stream_v) {
  if (pairs < 0 || pairs > kMaxPairs || pairs_per_row < 1 || pairs % pairs_per_row != 0 || E < 1 || N < 1 || K < 1 ||
      (G != 32 && G != 64 && G != 128) || K % G != 0 || (dtype != MOE_B200_BF16 && dtype != MOE_B200_F16) ||
      (!experts && (E != 1 || pairs_per_row != 1)))
    return MOE_B200_EINVAL;
  if (pairs == 0) return MOE_B200_OK;
  if (!x || !qweight || !scale || !out || !aligned(x, 16) || (pairs > pairs_per_row && x_stride % 8 != 0) || !aligned(qweight, 16))
    return MOE_B200_EINVAL;
  MatvecArgs a = {x, x_stride, qweight, scale, zero, experts, pairs, pairs_per_row, E, N, K, G, scale_f32, out};
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  return launch_status(dtype == MOE_B200_BF16 ? launch_matvec<__nv_bfloat16>(a, out_f32 != 0, stream)
                                              : launch_matvec<__half>(a, out_f32 != 0, stream), 1);
}
