// Matrix-vector products with 4-bit weights and group scales, for decode-sized batches, dense or by chosen experts:
//     out[r, n] = sum_k x[row(r), k] (q[e(r), n, k] - z[e(r), n, k / G]) scale[e(r), n, k / G]
// q: two values a byte, the even k in the low half; z: 8 without a table.  Pair r = (token, choice) reads row r / per_row
// of x and expert experts[r]; a pair whose expert is not held here gives a zero row.
//
// Bound by the weights, which are read once per (expert, up to 8 or 16 rows).  The products run on mma.sync m16n8k16 with
// the weights as the 16-row operand, which a lane builds in registers from the bytes it loaded itself: such an operand
// never passes through shared memory or tensor memory, and with at most 16 columns per weight the tensor pipe is idle
// most of the time anyway.  A lane's 16 (8, 4) bytes of a group of 128 (64, 32) weights feed eight (four, two) products in
// whatever order of k suits the unpacking; x is staged in shared memory in that same order.  q - z is exact in the
// activations' type (the bits of 128 + q or 1024 + q minus 128 + z or 1024 + z), products and sums are fp32, and the
// scale multiplies the fp32 sum of its group.
//
// A CTA owns 64 weight rows and a slice of K; its warps split rows and K, the CTAs of a cluster split K, and the partial
// sums meet in shared memory in a fixed order.
#include <cooperative_groups.h>

#include "elem_device.cuh"

namespace moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxPairs = 256;
constexpr int kMaxMatvecExperts = 1024;
constexpr int kThreads = 256;
constexpr int kTileRows = 64;
constexpr int kSliceK = 2048;              // columns of x staged at a time

struct MatvecArgs {
  const void* x;
  int64_t x_stride;
  const uint8_t* q;          // [E, N, K / 2]
  const void* scale;         // [E, N, K / G]
  const uint8_t* zero;       // [E, N, K / G] or null
  const int* experts;        // [pairs] or null
  int pairs, per_row, E, N, K, scale_f32;
  int split;                 // CTAs of a cluster, which divide K
  int slice_units;           // groups staged at a time
  int x_row;                 // 16-byte chunks between staged rows
  void* out;                 // [pairs, N]
};

template <typename T> struct Nibble;
template <> struct Nibble<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;      // 128 + q in both halves
  static __device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Nibble<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;      // 1024 + q
  static __device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// W consecutive words of eight weights each.
template <int W> struct Words;
template <> struct Words<4> { using Type = uint4; };
template <> struct Words<2> { using Type = uint2; };
template <> struct Words<1> { using Type = uint32_t; };

// G: group size.  NT: token tiles of eight columns.  A warp has MT tiles of 16 weight rows.
template <typename T, typename O, int G, int NT>
__global__ void __launch_bounds__(kThreads, 2) matvec_w4_kernel(MatvecArgs a) {
  constexpr int MT = NT, WR = kTileRows / (16 * MT), WK = kThreads / 32 / WR;   // row groups and K parts of the warps
  constexpr int W = G / 32;                        // words a lane loads per row and group
  constexpr int U = (MT == 1 ? 4 : 2) * (4 / W > 2 ? 2 : 4 / W);   // groups in flight
  constexpr int kCols = 8 * NT, kRedRow = kTileRows + 4;
  extern __shared__ uint4 xs[];                    // [kCols][x_row] staged activations
  __shared__ float red[WK][kCols][kRedRow];
  __shared__ int first_of[kMaxMatvecExperts];
  __shared__ int list[kMaxPairs], warp_count[8], chosen, n_list;
  griddep_launch_dependents();
  griddep_wait();

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, quad = lane & 3;
  const int rank = blockIdx.x % a.split, n0 = blockIdx.x / a.split * kTileRows;
  O* out = static_cast<O*>(a.out);

  // Slot y works for the y-th different expert of the batch, in order of first appearance, on all rows that chose it.
  int expert = 0, pairs = a.pairs;
  if (a.experts) {
    const int e = tid < a.pairs ? a.experts[tid] : -1;
    const bool held = e >= 0 && e < a.E;
    if (tid == 0) chosen = -1;
    if (held) first_of[e] = kMaxPairs;
    __syncthreads();
    if (held) atomicMin(first_of + e, tid);
    __syncthreads();
    const bool first = held && first_of[e] == tid;
    const uint32_t firsts = __ballot_sync(0xFFFFFFFFu, first);
    if (lane == 0) warp_count[warp] = __popc(firsts);
    __syncthreads();
    int before = __popc(firsts & ((1u << lane) - 1));
    for (int w = 0; w < warp; ++w) before += warp_count[w];
    if (first && before == blockIdx.y) chosen = e;
    if (rank == 0 && tid < a.pairs && !held && tid % gridDim.y == blockIdx.y) {
      for (int n = n0; n < min(n0 + kTileRows, a.N); ++n) out[static_cast<int64_t>(tid) * a.N + n] = from_f32<O>(0.0f);
    }
    __syncthreads();
    expert = chosen;
    if (expert < 0) return;                        // the same in all CTAs of a cluster
    const uint32_t mine = __ballot_sync(0xFFFFFFFFu, held && e == expert);
    if (lane == 0) warp_count[warp] = __popc(mine);
    __syncthreads();
    before = __popc(mine & ((1u << lane) - 1));
    for (int w = 0; w < warp; ++w) before += warp_count[w];
    if (held && e == expert) list[before] = tid;
    if (tid == 0) {
      int n = 0;
      for (int w = 0; w < 8; ++w) n += warp_count[w];
      n_list = n;
    }
    __syncthreads();
    pairs = n_list;
  }

  const int units = a.K / G, per_rank = (units + a.split - 1) / a.split;
  const int first_unit = min(units, rank * per_rank), end_unit = min(units, first_unit + per_rank);
  const int row_warp = n0 + (warp / WK) * 16 * MT + gid, part = warp % WK;
  // addresses of the lane's rows (rows behind the last read the last one and are not stored)
  int64_t row[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) row[m][h] = static_cast<int64_t>(expert) * a.N + min(row_warp + 16 * m + 8 * h, a.N - 1);

  for (int p0 = 0; p0 < pairs; p0 += kCols) {
    const int cols = min(kCols, pairs - p0);
    float sum[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[m][t][i] = 0.0f;

    for (int s0 = first_unit; s0 < end_unit; s0 += a.slice_units) {
      const int s1 = min(end_unit, s0 + a.slice_units), per_part = (s1 - s0 + WK - 1) / WK;
      const int u0 = s0 + part * per_part, u1 = min(s1, u0 + per_part);
      typename Words<W>::Type w[U][MT][2];
      float sc[U][MT][2];
      uint32_t zp[U][MT][2];
      auto load = [&](int u) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if (u + i >= u1) continue;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              w[i][m][h] = __ldg(reinterpret_cast<const typename Words<W>::Type*>(a.q + row[m][h] * (a.K / 2) +
                                                                                 (u + i) * (G / 2) + quad * (4 * W)));
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if (u + i >= u1) continue;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int64_t at = row[m][h] * units + u + i;
              sc[i][m][h] = a.scale_f32 ? __ldg(static_cast<const float*>(a.scale) + at)
                                        : to_f32<T>(static_cast<const T*>(a.scale)[at]);
              zp[i][m][h] = a.zero ? Nibble<T>::kMagic | __ldg(a.zero + at) * 0x00010001u : Nibble<T>::kMagic | 0x00080008u;
            }
        }
      };
      load(u0);

      // stage x: a 16-byte chunk holds eight k, stored as pairs (k, k + 4); chunk j of quad lane t of a group at 4 j + t
      const int chunks = (s1 - s0) * (G / 8);
      for (int i = tid; i < cols * chunks; i += kThreads) {
        const int c = i / chunks, at = i - c * chunks, in = at % (G / 8);
        const int pair = a.experts ? list[p0 + c] : p0 + c;
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (pair / a.per_row) * a.x_stride +
                                                             static_cast<int64_t>(s0) * G + at * 8));
        xs[c * a.x_row + at - in + (in % W) * 4 + in / W] =
            make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                       __byte_perm(v.y, v.w, 0x7632));
      }
      __syncthreads();

      for (int u = u0; u < u1; u += U) {
        if (u != u0) load(u);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if (u + i >= u1) continue;
          float acc[MT][NT][4];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[m][t][k] = 0.0f;
          const uint4* xu = xs + (u + i - s0) * (G / 8) + quad;
#pragma unroll
          for (int j = 0; j < W; ++j) {
            uint4 b[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              b[t] = make_uint4(0u, 0u, 0u, 0u);
              if (8 * t + gid < cols) b[t] = xu[(8 * t + gid) * a.x_row + 4 * j];
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const uint32_t lo = reinterpret_cast<const uint32_t*>(&w[i][m][0])[j];
              const uint32_t hi = reinterpret_cast<const uint32_t*>(&w[i][m][1])[j];
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                uint32_t frag[4];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const int shift = 4 * (2 * half + k);
                  frag[2 * k] = Nibble<T>::minus(((lo >> shift) & 0x000F000Fu) | Nibble<T>::kMagic, zp[i][m][0]);
                  frag[2 * k + 1] = Nibble<T>::minus(((hi >> shift) & 0x000F000Fu) | Nibble<T>::kMagic, zp[i][m][1]);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  if (t > 0 && cols <= 8 * t) continue;
                  Nibble<T>::mma(acc[m][t], frag, half ? b[t].z : b[t].x, half ? b[t].w : b[t].y);
                }
              }
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int k = 0; k < 4; ++k) sum[m][t][k] += acc[m][t][k] * sc[i][m][k >> 1];
        }
      }
      __syncthreads();                             // the staged rows may be overwritten
    }

    // join: the K parts of the warps, then the CTAs of the cluster, each in order
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          red[part][8 * t + 2 * quad + (k & 1)][(warp / WK) * 16 * MT + 16 * m + 8 * (k >> 1) + gid] = sum[m][t][k];
    __syncthreads();
    if (a.split == 1) {
      for (int i = tid; i < cols * kTileRows; i += kThreads) {
        const int c = i / kTileRows, r = i % kTileRows;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < WK; ++k) v += red[k][c][r];
        const int pair = a.experts ? list[p0 + c] : p0 + c;
        if (n0 + r < a.N) out[static_cast<int64_t>(pair) * a.N + n0 + r] = from_f32<O>(v);
      }
      __syncthreads();
    } else {
      cg::cluster_group cluster = cg::this_cluster();
      for (int i = tid; i < cols * kTileRows; i += kThreads) {
        const int c = i / kTileRows, r = i % kTileRows;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < WK; ++k) v += red[k][c][r];
        red[0][c][r] = v;
      }
      cluster.sync();
      for (int i = tid + rank * kThreads; i < cols * kTileRows; i += kThreads * a.split) {
        const int c = i / kTileRows, r = i % kTileRows;
        float v = 0.0f;
        for (int k = 0; k < a.split; ++k) v += *cluster.map_shared_rank(&red[0][c][r], k);
        const int pair = a.experts ? list[p0 + c] : p0 + c;
        if (n0 + r < a.N) out[static_cast<int64_t>(pair) * a.N + n0 + r] = from_f32<O>(v);
      }
      cluster.sync();                              // nobody reads a neighbour's sums any more
    }
  }
}

template <typename T, typename O, int G, int NT>
cudaError_t launch_kernel(MatvecArgs a, cudaStream_t stream) {
  const int units = a.K / G, tiles = (a.N + kTileRows - 1) / kTileRows;
  const int slots = a.experts ? (a.pairs < a.E ? a.pairs : a.E) : 1;
  // A cluster divides K so that a CTA stages its columns of x once, and further while there are fewer CTAs than SMs and
  // a warp keeps at least one group.
  int split = 1;
  while (split < 8 && a.K > kSliceK * split) split *= 2;
  while (split < 8 && tiles * slots * split < kNumSMs && units >= 2 * split * (NT == 1 ? 2 : 4)) split *= 2;
  a.split = split;
  const int per_rank = (units + split - 1) / split;
  a.slice_units = per_rank < kSliceK / G ? per_rank : kSliceK / G;
  a.x_row = (a.slice_units * (G / 8) + 7) / 8 * 8 + 4;   // rows 64 bytes apart in the banks
  const size_t smem = static_cast<size_t>(8 * NT) * a.x_row * 16;
  constexpr size_t kMost = static_cast<size_t>(8 * NT) * (kSliceK / 8 + 4) * 16;
  static const cudaError_t set = cudaFuncSetAttribute(matvec_w4_kernel<T, O, G, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                      static_cast<int>(kMost));
  if (set != cudaSuccess) return set;
  return launch_cluster(matvec_w4_kernel<T, O, G, NT>, dim3(tiles * split, slots), dim3(kThreads), split, smem, stream, a);
}

template <typename T, typename O>
cudaError_t launch_matvec(const MatvecArgs& a, int G, cudaStream_t stream) {
  // one tile of eight columns where no expert can have more rows (a row chooses an expert once)
  const bool one = a.pairs / a.per_row <= 8;
  if (G == 128) return one ? launch_kernel<T, O, 128, 1>(a, stream) : launch_kernel<T, O, 128, 2>(a, stream);
  if (G == 64) return one ? launch_kernel<T, O, 64, 1>(a, stream) : launch_kernel<T, O, 64, 2>(a, stream);
  return one ? launch_kernel<T, O, 32, 1>(a, stream) : launch_kernel<T, O, 32, 2>(a, stream);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_fp8_block_scale_matvec_w4(const void* x, int64_t x_stride, int dtype, const uint8_t* qweight,
                                             const void* scale, int scale_f32, const uint8_t* zero, const int32_t* experts,
                                             int pairs, int pairs_per_row, int E, int N, int K, int G, void* out,
                                             int out_f32, void* stream_v) {
  if (pairs < 0 || pairs > kMaxPairs || pairs_per_row < 1 || pairs % pairs_per_row != 0 || E < 1 || E > kMaxMatvecExperts ||
      N < 1 || K < 1 || (G != 32 && G != 64 && G != 128) || K % G != 0 || (dtype != MOE_B200_BF16 && dtype != MOE_B200_F16) ||
      (!experts && (E != 1 || pairs_per_row != 1)))
    return MOE_B200_EINVAL;
  if (pairs == 0) return MOE_B200_OK;
  if (!x || !qweight || !scale || !out || !aligned(x, 16) || (pairs > pairs_per_row && x_stride % 8 != 0) || !aligned(qweight, 16))
    return MOE_B200_EINVAL;
  MatvecArgs a = {x, x_stride, qweight, scale, zero, experts, pairs, pairs_per_row, E, N, K, scale_f32, 1, 0, 0, out};
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  cudaError_t e;
  if (dtype == MOE_B200_BF16)
    e = out_f32 ? launch_matvec<__nv_bfloat16, float>(a, G, stream) : launch_matvec<__nv_bfloat16, __nv_bfloat16>(a, G, stream);
  else
    e = out_f32 ? launch_matvec<__half, float>(a, G, stream) : launch_matvec<__half, __half>(a, G, stream);
  return launch_status(e, 1);
}
