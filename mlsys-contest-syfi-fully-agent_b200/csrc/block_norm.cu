// Norms before and after a block, fused with the block's gate and the residual scale.
//
// Forward, per row (x: residual stream, y: the block's output):
//     r1 = rsqrt(mean(y^2) + eps),  n = y r1 w_post            (n = y without w_post)
//     s  = a x + g n                                           (s = x without y)
//     r2 = rsqrt(mean(s^2) + eps),  h = s r2 w_pre
// h leaves as activations or as the shard's input: e4m3 with one fp32 scale per 128 columns, [H / 128, T].
// Everything between the loads and the stores is fp32; s is rounded once when it is stored, h is computed from the
// unrounded s, and the e4m3 values are rounded from the unrounded h.
//
// Backward, per row, with D = dL/ds, u = gh w_pre, sh = s r2, yh = y r1, n = yh w_post:
//     D  = gs + r2 (u - sh mean(u sh)),      dx = a D,      dg = D n (summed over what the gate is broadcast along)
//     dy = r1 (D g w_post - yh mean(D g w_post yh))         (D g without w_post)
//     dw_pre = sum_t gh sh,   dw_post = sum_t D g yh
// s is formed again from x and y (two rows read instead of the rounded s and y), r1 and r2 come from the forward.
#include <cuda_fp8.h>

#include "elem_device.cuh"

namespace moe {
namespace {

constexpr int kMaxWidth = 16384;
constexpr int kNormThreads = 512;

enum GateKind : int { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

struct NormArgs {
  const void *x, *y, *gate, *pre_w, *post_w;
  int64_t x_stride, y_stride, gate_stride;   // elements between rows
  int T, H, gate_kind;
  int pre_f32, post_f32, gate_f32;           // parameter is fp32 whatever the activations' type is
  float a, eps;
  void *s, *h;                               // [T, H]
  uint8_t* q;                                // [T, H] e4m3 and
  float* q_scale;                            // [H / 128, T], both or neither
  float* rstd;                               // [T, 2]
  // backward
  const void *gh, *gs;
  int64_t gh_stride, gs_stride;
  void *dx, *dy, *dgate_rows;                // dgate_rows: [T, 1] or [T, H]
  float* partial;                            // [gridDim.x][n_sums][H] column sums
  int n_sums, sum_post, sum_gate;            // rows of `partial`: 0 is dw_pre; -1: not wanted
};

// Which column a thread's j-th element of chunk c is: eight neighbours where rows can be read 16 bytes at a time,
// else columns blockDim.x apart, so that single-element loads of a warp are adjacent.
template <bool VEC>
__device__ __forceinline__ int column(int c, int j) {
  return VEC ? (c * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8 + j
             : (c * 8 + j) * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int c, int H, float (&v)[8]) {
  if (VEC) {
    const int col = column<VEC>(c, 0);
    Pack8<T> raw;
    if (col < H) {
      raw = *reinterpret_cast<const Pack8<T>*>(p + col);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(raw.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = column<VEC>(c, j);
      v[j] = col < H ? to_f32<T>(p[col]) : 0.0f;
    }
  }
}

// A parameter row (weight or gate) in the activations' type or in fp32.
template <typename T, bool VEC>
__device__ __forceinline__ void load8_param(const void* p, int f32, int64_t row_offset, int c, int H, float (&v)[8]) {
  if (f32)
    load8<float, VEC>(static_cast<const float*>(p) + row_offset, c, H, v);
  else
    load8<T, VEC>(static_cast<const T*>(p) + row_offset, c, H, v);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int c, int H, const float (&v)[8]) {
  if (VEC) {
    const int col = column<VEC>(c, 0);
    if (col >= H) return;
    Pack8<T> raw;
#pragma unroll
    for (int j = 0; j < 8; ++j) raw.v[j] = from_f32<T>(v[j]);
    *reinterpret_cast<Pack8<T>*>(p + col) = raw;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = column<VEC>(c, j);
      if (col < H) p[col] = from_f32<T>(v[j]);
    }
  }
}

// One CTA per row; a thread keeps CH groups of eight columns in registers from the loads to the stores.
template <typename T, int CH, bool VEC, bool QUANT>
__global__ void __launch_bounds__(kNormThreads) block_norm_kernel(NormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float red[2][32];
  const int H = a.H;
  const float inv_h = 1.0f / static_cast<float>(H);
  for (int row = blockIdx.x; row < a.T; row += gridDim.x) {
    float s[CH][8];
    float r1 = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) load8<T, VEC>(static_cast<const T*>(a.x) + row * a.x_stride, c, H, s[c]);
    if (a.y) {
      float n[CH][8];
#pragma unroll
      for (int c = 0; c < CH; ++c) load8<T, VEC>(static_cast<const T*>(a.y) + row * a.y_stride, c, H, n[c]);
      if (a.post_w) {
        float sum[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[0] += n[c][j] * n[c][j];
        block_sum(sum, red[0]);
        r1 = rsqrtf(sum[0] * inv_h + a.eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float w[8];
          load8_param<T, VEC>(a.post_w, a.post_f32, 0, c, H, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) n[c][j] = n[c][j] * r1 * w[j];
        }
      }
      if (a.gate_kind == kGateToken) {
        const int64_t at = row * a.gate_stride;
        const float g = a.gate_f32 ? static_cast<const float*>(a.gate)[at] : to_f32<T>(static_cast<const T*>(a.gate)[at]);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j) n[c][j] *= g;
      } else if (a.gate_kind != kGateNone) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float g[8];
          load8_param<T, VEC>(a.gate, a.gate_f32, a.gate_kind == kGateFull ? row * a.gate_stride : 0, c, H, g);
#pragma unroll
          for (int j = 0; j < 8; ++j) n[c][j] *= g[j];
        }
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[c][j] = a.a * s[c][j] + n[c][j];
        store8<T, VEC>(static_cast<T*>(a.s) + static_cast<int64_t>(row) * H, c, H, s[c]);
      }
    }
    float sum[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[0] += s[c][j] * s[c][j];
    block_sum(sum, red[1]);
    const float r2 = rsqrtf(sum[0] * inv_h + a.eps);
    if (threadIdx.x == 0) {
      a.rstd[2 * static_cast<int64_t>(row)] = r1;
      a.rstd[2 * static_cast<int64_t>(row) + 1] = r2;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float w[8];
      load8_param<T, VEC>(a.pre_w, a.pre_f32, 0, c, H, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[c][j] = s[c][j] * r2 * w[j];
      if (QUANT) {
        // sixteen lanes hold a block of 128 columns; scale = max(|h|, 1e-10) / 448 and e4m3(h / scale), the rule of the
        // activation quantiser
        const int col = column<true>(c, 0);
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(s[c][j]));
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
        const float scale = __fdiv_rn(fmaxf(amax, 1e-10f), 448.0f);
        uint32_t packed[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          packed[j >> 2] |= static_cast<uint32_t>(__nv_cvt_float_to_fp8(__fdiv_rn(s[c][j], scale), __NV_SATFINITE, __NV_E4M3))
                            << (8 * (j & 3));
        if (col < H) {
          *reinterpret_cast<uint2*>(a.q + static_cast<int64_t>(row) * H + col) = make_uint2(packed[0], packed[1]);
          if ((threadIdx.x & 15) == 0) a.q_scale[static_cast<int64_t>(col / kBlock) * a.T + row] = scale;
        }
      } else {
        store8<T, VEC>(static_cast<T*>(a.h) + static_cast<int64_t>(row) * H, c, H, s[c]);
      }
    }
    // red[0] of the next row is written only after every thread has passed the barrier of red[1], and without a first
    // sum red[1] would be written again while a slow thread reads it
    if (!a.post_w) __syncthreads();
  }
}

// Rows are dealt to the CTAs round-robin; the column sums of a CTA's rows stay in shared memory (every thread owns its
// columns) and leave once, as one partial row per CTA, which column_sum_kernel adds in CTA order: no atomics, the same
// bits every time.  The dot products of a row need one reduction: with A = sum u sh, B = sum (gs + r2 u) v and
// C = sum sh v for v = n (its gate g_t left out of a per-token gate's gradient) everything follows linearly.
template <typename T, int CH, bool VEC>
__global__ void __launch_bounds__(kNormThreads) block_norm_backward_kernel(NormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  extern __shared__ float acc[];             // [n_sums][CH * 8][blockDim.x], thread-private columns
  __shared__ float red[2][96];
  const int H = a.H, nt = blockDim.x, tid = threadIdx.x;
  const float inv_h = 1.0f / static_cast<float>(H);
  for (int i = 0; i < a.n_sums * CH * 8; ++i) acc[i * nt + tid] = 0.0f;
  int flip = 0;
  for (int row = blockIdx.x; row < a.T; row += gridDim.x, flip ^= 1) {
    const float r1 = a.rstd[2 * static_cast<int64_t>(row)], r2 = a.rstd[2 * static_cast<int64_t>(row) + 1];
    float gt = 1.0f;
    if (a.gate_kind == kGateToken) {
      const int64_t at = row * a.gate_stride;
      gt = a.gate_f32 ? static_cast<const float*>(a.gate)[at] : to_f32<T>(static_cast<const T*>(a.gate)[at]);
    }
    float u[CH][8], sh[CH][8], d[CH][8], yh[CH][8];
    float sums[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float w[8], g[8], wp[8];
      load8<T, VEC>(static_cast<const T*>(a.x) + row * a.x_stride, c, H, sh[c]);
      load8<T, VEC>(static_cast<const T*>(a.gh) + row * a.gh_stride, c, H, u[c]);
      load8_param<T, VEC>(a.pre_w, a.pre_f32, 0, c, H, w);
      if (a.gs) {
        load8<T, VEC>(static_cast<const T*>(a.gs) + row * a.gs_stride, c, H, d[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[c][j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) { g[j] = gt; wp[j] = 1.0f; yh[c][j] = 0.0f; }
      if (a.y) {
        load8<T, VEC>(static_cast<const T*>(a.y) + row * a.y_stride, c, H, yh[c]);
        if (a.post_w) {
          load8_param<T, VEC>(a.post_w, a.post_f32, 0, c, H, wp);
#pragma unroll
          for (int j = 0; j < 8; ++j) yh[c][j] *= r1;
        }
        if (a.gate_kind == kGateChannel || a.gate_kind == kGateFull)
          load8_param<T, VEC>(a.gate, a.gate_f32, a.gate_kind == kGateFull ? row * a.gate_stride : 0, c, H, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) sh[c][j] = a.a * sh[c][j] + g[j] * (yh[c][j] * wp[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sh[c][j] *= r2;
        acc[(c * 8 + j) * nt + tid] += u[c][j] * sh[c][j];            // dw_pre
        u[c][j] *= w[j];
        d[c][j] += r2 * u[c][j];
        const float v = yh[c][j] * wp[j] * (a.gate_kind == kGateToken ? 1.0f : g[j]);
        sums[0] += u[c][j] * sh[c][j];
        sums[1] += d[c][j] * v;
        sums[2] += sh[c][j] * v;
      }
    }
    block_sum(sums, red[flip]);
    const float k2 = r2 * (sums[0] * inv_h);                          // D = d - sh k2
    const float dv = sums[1] - k2 * sums[2];                          // sum_h D v
    if (a.gate_kind == kGateToken && tid == 0) {
      if (a.gate_f32) static_cast<float*>(a.dgate_rows)[row] = dv;
      else static_cast<T*>(a.dgate_rows)[row] = from_f32<T>(dv);
    }
    const float k1 = dv * gt * inv_h;                                 // mean(D g w_post yh)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float g[8], wp[8], out[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        d[c][j] -= sh[c][j] * k2;
        out[j] = a.y ? a.a * d[c][j] : d[c][j];
        g[j] = gt;
        wp[j] = 1.0f;
      }
      store8<T, VEC>(static_cast<T*>(a.dx) + static_cast<int64_t>(row) * H, c, H, out);
      if (!a.y) continue;
      if (a.gate_kind == kGateChannel || a.gate_kind == kGateFull)
        load8_param<T, VEC>(a.gate, a.gate_f32, a.gate_kind == kGateFull ? row * a.gate_stride : 0, c, H, g);
      if (a.post_w) load8_param<T, VEC>(a.post_w, a.post_f32, 0, c, H, wp);
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = d[c][j] * (yh[c][j] * wp[j]);
      if (a.gate_kind == kGateFull) {
        if (a.gate_f32) store8<float, VEC>(static_cast<float*>(a.dgate_rows) + static_cast<int64_t>(row) * H, c, H, out);
        else store8<T, VEC>(static_cast<T*>(a.dgate_rows) + static_cast<int64_t>(row) * H, c, H, out);
      } else if (a.sum_gate >= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[(a.sum_gate * CH * 8 + c * 8 + j) * nt + tid] += out[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float dn = d[c][j] * g[j];
        out[j] = dn;
        if (a.post_w) {
          acc[(a.sum_post * CH * 8 + c * 8 + j) * nt + tid] += dn * yh[c][j];
          out[j] = r1 * (dn * wp[j] - yh[c][j] * k1);
        }
      }
      store8<T, VEC>(static_cast<T*>(a.dy) + static_cast<int64_t>(row) * H, c, H, out);
    }
  }
  for (int k = 0; k < a.n_sums; ++k) {
    float* dst = a.partial + (static_cast<int64_t>(blockIdx.x) * a.n_sums + k) * H;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = column<VEC>(c, j);
        if (col < H) dst[col] = acc[(k * CH * 8 + c * 8 + j) * nt + tid];
      }
  }
}

struct ColumnSumArgs {
  const float* partial;    // [n_parts][n_sums][H]
  int n_parts, n_sums, H;
  void* out[3];
  int f32[3];
};

constexpr int kSumStrips = 8;

// out[k][col] = sum over the parts in order, in eight interleaved strips that are joined in order.
template <typename T>
__global__ void __launch_bounds__(32 * kSumStrips) column_sum_kernel(ColumnSumArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float strip[kSumStrips][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, k = blockIdx.y;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (col < a.H) {
#pragma unroll 4
    for (int p = w; p < a.n_parts; p += kSumStrips) s += a.partial[(static_cast<int64_t>(p) * a.n_sums + k) * a.H + col];
  }
  strip[w][lane] = s;
  __syncthreads();
  if (w == 0 && col < a.H) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kSumStrips; ++i) t += strip[i][lane];
    if (a.f32[k]) static_cast<float*>(a.out[k])[col] = t;
    else static_cast<T*>(a.out[k])[col] = from_f32<T>(t);
  }
}

// Threads and groups of eight columns per thread for a row of H columns.
struct Shape {
  int ch, threads;
};
Shape shape_of(int H) {
  const int groups = (H + 7) / 8;
  const int ch = groups <= 256 ? 1 : groups <= 2 * kNormThreads ? 2 : 4;
  return {ch, ((groups + ch - 1) / ch + 31) / 32 * 32};
}

// Rows can be moved 16 bytes at a time.
bool rows_aligned(const void* p, int64_t stride, int size) {
  return !p || (aligned(p, 16) && stride * size % 16 == 0);
}

bool vector_rows(const NormArgs& a, int dtype) {
  const int size = element_size(dtype);
  return a.H % 8 == 0 && rows_aligned(a.x, a.x_stride, size) && rows_aligned(a.y, a.y_stride, size) &&
         (a.gate_kind == kGateToken || rows_aligned(a.gate, a.gate_kind == kGateFull ? a.gate_stride : 0, a.gate_f32 ? 4 : size)) &&
         rows_aligned(a.pre_w, 0, 1) && rows_aligned(a.post_w, 0, 1) && rows_aligned(a.gh, a.gh_stride, size) &&
         rows_aligned(a.gs, a.gs_stride, size) && rows_aligned(a.s, a.H, size) && rows_aligned(a.h, a.H, size) &&
         rows_aligned(a.dx, a.H, size) && rows_aligned(a.dy, a.H, size) &&
         (a.gate_kind != kGateFull || rows_aligned(a.dgate_rows, a.H, a.gate_f32 ? 4 : size)) && aligned(a.q, 8);
}

bool bad_common(const NormArgs& a, int dtype, int param_f32) {
  return a.T < 0 || a.H < 1 || a.H > kMaxWidth || dtype < MOE_B200_F32 || dtype > MOE_B200_F16 || (param_f32 & ~7) ||
         a.gate_kind < kGateNone || a.gate_kind > kGateFull || (a.gate_kind != kGateNone && (!a.gate || !a.y)) ||
         (a.post_w && !a.y);
}

int grid_rows(int T, int per_sm) { return T < kNumSMs * per_sm ? T : kNumSMs * per_sm; }

template <typename T, int CH>
cudaError_t launch_forward(const NormArgs& a, bool vec, int threads, cudaStream_t stream) {
  const dim3 grid(grid_rows(a.T, 8)), block(threads);
  if (a.q) return launch_pdl(block_norm_kernel<T, CH, true, true>, grid, block, 0, stream, a);
  if (vec) return launch_pdl(block_norm_kernel<T, CH, true, false>, grid, block, 0, stream, a);
  return launch_pdl(block_norm_kernel<T, CH, false, false>, grid, block, 0, stream, a);
}

template <typename T>
cudaError_t launch_forward(const NormArgs& a, bool vec, cudaStream_t stream) {
  const Shape sh = shape_of(a.H);
  if (sh.ch == 1) return launch_forward<T, 1>(a, vec, sh.threads, stream);
  if (sh.ch == 2) return launch_forward<T, 2>(a, vec, sh.threads, stream);
  return launch_forward<T, 4>(a, vec, sh.threads, stream);
}

template <typename T, int CH, bool VEC>
cudaError_t launch_backward(const NormArgs& a, int grid, int threads, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(a.n_sums) * CH * 8 * threads * sizeof(float);
  cudaError_t e = cudaFuncSetAttribute(block_norm_backward_kernel<T, CH, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  return launch_pdl(block_norm_backward_kernel<T, CH, VEC>, dim3(grid), dim3(threads), smem, stream, a);
}

template <typename T>
cudaError_t launch_backward(const NormArgs& a, const ColumnSumArgs& cs, bool vec, cudaStream_t stream) {
  const Shape sh = shape_of(a.H);
  const int grid = cs.n_parts, nt = sh.threads;
  cudaError_t e;
  if (sh.ch == 1) e = vec ? launch_backward<T, 1, true>(a, grid, nt, stream) : launch_backward<T, 1, false>(a, grid, nt, stream);
  else if (sh.ch == 2) e = vec ? launch_backward<T, 2, true>(a, grid, nt, stream) : launch_backward<T, 2, false>(a, grid, nt, stream);
  else e = vec ? launch_backward<T, 4, true>(a, grid, nt, stream) : launch_backward<T, 4, false>(a, grid, nt, stream);
  if (e != cudaSuccess) return e;
  return launch_pdl(column_sum_kernel<T>, dim3((a.H + 31) / 32, cs.n_sums), dim3(32 * kSumStrips), 0, stream, cs);
}

int backward_parts(int T) { return grid_rows(T, 1); }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_fp8_block_scale_block_norm(const void* x, int64_t x_stride, const void* y, int64_t y_stride,
                                              const void* gate, int64_t gate_stride, int gate_kind,
                                              const void* pre_weight, const void* post_weight, int T, int H, int dtype,
                                              int param_f32, float residual_scale, float eps, void* stream_out, void* h,
                                              float* h_scale, float* rstd, void* stream_v) {
  NormArgs a = {};
  a.x = x; a.y = y; a.gate = gate; a.pre_w = pre_weight; a.post_w = post_weight;
  a.x_stride = x_stride; a.y_stride = y_stride; a.gate_stride = gate_stride;
  a.T = T; a.H = H; a.gate_kind = gate_kind;
  a.pre_f32 = param_f32 & 1; a.post_f32 = (param_f32 >> 1) & 1; a.gate_f32 = (param_f32 >> 2) & 1;
  a.a = residual_scale; a.eps = eps; a.s = stream_out; a.rstd = rstd;
  if (h_scale) {
    a.q = static_cast<uint8_t*>(h);
    a.q_scale = h_scale;
  } else {
    a.h = h;
  }
  if (bad_common(a, dtype, param_f32) || !(eps > 0.0f)) return MOE_B200_EINVAL;
  if (T == 0) return MOE_B200_OK;
  if (!x || !pre_weight || !h || !rstd || (y && !stream_out)) return MOE_B200_EINVAL;
  const bool vec = vector_rows(a, dtype);
  if (h_scale && (H % kBlock != 0 || !vec)) return MOE_B200_EINVAL;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  cudaError_t e;
  if (dtype == MOE_B200_F32) e = launch_forward<float>(a, vec, stream);
  else if (dtype == MOE_B200_BF16) e = launch_forward<__nv_bfloat16>(a, vec, stream);
  else e = launch_forward<__half>(a, vec, stream);
  return launch_status(e, 1);
}

extern "C" size_t moe_fp8_block_scale_block_norm_backward_workspace_bytes(int T, int H) {
  if (T < 0 || H < 1 || H > kMaxWidth) return 0;
  return static_cast<size_t>(backward_parts(T)) * 3 * H * sizeof(float);
}

extern "C" int moe_fp8_block_scale_block_norm_backward(
    const void* x, int64_t x_stride, const void* y, int64_t y_stride, const void* gate, int64_t gate_stride, int gate_kind,
    const void* pre_weight, const void* post_weight, int T, int H, int dtype, int param_f32, float residual_scale,
    const float* rstd, const void* grad_h, int64_t grad_h_stride, const void* grad_stream, int64_t grad_stream_stride,
    void* grad_x, void* grad_y, void* grad_gate, void* grad_pre_weight, void* grad_post_weight, void* workspace,
    size_t workspace_bytes, void* stream_v) {
  NormArgs a = {};
  a.x = x; a.y = y; a.gate = gate; a.pre_w = pre_weight; a.post_w = post_weight;
  a.x_stride = x_stride; a.y_stride = y_stride; a.gate_stride = gate_stride;
  a.T = T; a.H = H; a.gate_kind = gate_kind;
  a.pre_f32 = param_f32 & 1; a.post_f32 = (param_f32 >> 1) & 1; a.gate_f32 = (param_f32 >> 2) & 1;
  a.a = residual_scale; a.rstd = const_cast<float*>(rstd);
  a.gh = grad_h; a.gh_stride = grad_h_stride; a.gs = grad_stream; a.gs_stride = grad_stream_stride;
  a.dx = grad_x; a.dy = grad_y;
  if (bad_common(a, dtype, param_f32)) return MOE_B200_EINVAL;
  if (T == 0) return MOE_B200_OK;
  if (!x || !pre_weight || !rstd || !grad_h || !grad_x || !grad_pre_weight || (y && !grad_y) ||
      (post_weight && !grad_post_weight) || (gate_kind != kGateNone && !grad_gate) || !workspace || !aligned(workspace, 16))
    return MOE_B200_EINVAL;
  if (workspace_bytes < moe_fp8_block_scale_block_norm_backward_workspace_bytes(T, H)) return MOE_B200_EWORKSPACE;
  ColumnSumArgs cs = {};
  a.sum_post = a.sum_gate = -1;
  cs.out[0] = grad_pre_weight;
  cs.f32[0] = a.pre_f32;
  a.n_sums = 1;
  if (post_weight) {
    a.sum_post = a.n_sums++;
    cs.out[a.sum_post] = grad_post_weight;
    cs.f32[a.sum_post] = a.post_f32;
  }
  if (gate_kind == kGateChannel) {
    a.sum_gate = a.n_sums++;
    cs.out[a.sum_gate] = grad_gate;
    cs.f32[a.sum_gate] = a.gate_f32;
  } else {
    a.dgate_rows = grad_gate;
  }
  a.partial = static_cast<float*>(workspace);
  cs.partial = a.partial;
  cs.n_parts = backward_parts(T);
  cs.n_sums = a.n_sums;
  cs.H = H;
  const bool vec = vector_rows(a, dtype);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  cudaError_t e;
  if (dtype == MOE_B200_F32) e = launch_backward<float>(a, cs, vec, stream);
  else if (dtype == MOE_B200_BF16) e = launch_backward<__nv_bfloat16>(a, cs, vec, stream);
  else e = launch_backward<__half>(a, cs, vec, stream);
  return launch_status(e, 2);
}
