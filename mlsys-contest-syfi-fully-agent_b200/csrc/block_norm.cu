// Norms before and after a block, fused with the block's gate and the residual scale.
//
// Forward, per row (x: residual stream, y: the block's output):
//     r1 = rsqrt(mean(y^2) + eps),  n = y r1 w_post            (n = y without w_post)
//     s  = a x + g n                                           (s = x without y)
//     r2 = rsqrt(mean(s^2) + eps),  h = s r2 w_pre
// h leaves as activations or as the shard's input: e4m3 with one fp32 scale per 128 columns, [H / 128, T].
// Everything between the loads and the stores is fp32; s is rounded once when it is stored, h is computed from the
// unrounded s, and the e4m3 values are rounded from the unrounded h.
#include <cuda_fp8.h>

#include "block_norm.cuh"

namespace moe {
namespace {

// Bound by HBM (x, y in; s, h out), so the loads must never wait for the two reductions of a row: persistent CTAs bring
// the rows of x, y (and a full gate) that they will need through a ring of up to three stages (cp.async).  Every thread
// copies exactly the sixteen-byte pieces that it will read itself, so the ring needs no barrier.  Weights come from the
// first-level cache, which the copies pass by.  A thread has sixteen columns of a row of 4096 and more: two CTAs of 448
// threads at 7168 columns, whose barriers fill each other's gaps.
// Measured, 4096 x 7168 bf16: join and norm 47 us (5.0 TB/s), with e4m3 output 51 us (4.1 TB/s: 61 % of the issue slots
// are taken, the conversion's maximum and products among them); without the ring 79 us.  4096 x 5001 (kEdges) 44 us, with
// rows 5006 apart (kShifted) 59 us, element by element 180 us.
//
// GATE: where the gate and the parameters' types are known (all of the activations' type), else kAnyGate.
constexpr int kAnyGate = -1;

template <typename T, int CH, RowMode MODE, bool QUANT, int GATE>
__global__ void __launch_bounds__(CH == 1 ? 256 : kNormThreads, CH == 1 ? 3 : CH == 2 ? 2 : 1) block_norm_kernel(NormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr bool VEC = by_block(MODE);
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2][32];
  const int H = a.H;
  const int gate_kind = GATE == kAnyGate ? a.gate_kind : GATE == kGateNone && a.gate_kind == kGateToken ? kGateToken : GATE;
  const float inv_h = 1.0f / static_cast<float>(H);
  // a full gate of another type than the activations' is read directly
  const bool full_in_ring = GATE == kGateFull || (GATE == kAnyGate && gate_kind == kGateFull && !(a.gate_f32 && sizeof(T) == 2));
  const int span = span_bytes(H, sizeof(T));
  const int off = has_edges(MODE) ? static_cast<int>(blockIdx.x * static_cast<int64_t>(H) % (16 / static_cast<int>(sizeof(T)))) : 0;
  const uint32_t stage_bytes = static_cast<uint32_t>(a.arrays * (VEC ? CH * blockDim.x * sizeof(Pack8<T>) : span));
  auto param = [&](const void* p, int f32, int64_t offset, int c, F2 (&v)[4]) {
    if (has_edges(MODE)) take8<T, CH>(ring + a.ring * stage_bytes, p == a.pre_w ? 0 : p == a.post_w ? 1 : 2, c, v);
    else if (GATE == kAnyGate) load8_param<T, VEC>(p, f32, offset, c, H, v);
    else load8<T, VEC>(static_cast<const T*>(p) + offset, c, H, v);
  };
  // rows still to be fetched and to be stored
  int64_t fetch_at = blockIdx.x;
  const T* fetch_x = static_cast<const T*>(a.x) + fetch_at * a.x_stride;
  const T* fetch_y = static_cast<const T*>(a.y) + fetch_at * a.y_stride;
  const T* fetch_g = static_cast<const T*>(a.gate) + fetch_at * a.gate_stride;
  const int64_t step = gridDim.x;
  auto fetch = [&](uint32_t stage) {
    if (fetch_at < a.T) {
      if (VEC) {
        fetch_row<T, CH, MODE>(stage, 0, fetch_x, H, off);
        if (a.y) fetch_row<T, CH, MODE>(stage, 1, fetch_y, H, off);
        if (full_in_ring) fetch_row<T, CH, MODE>(stage, 2, fetch_g, H, off);
      } else {
        fetch_span(stage, fetch_x, H);
        if (a.y) fetch_span(stage + span, fetch_y, H);
        if (full_in_ring) fetch_span(stage + 2 * span, fetch_g, H);
      }
    }
    fetch_at += step;
    fetch_x += step * a.x_stride;
    fetch_y += step * a.y_stride;
    fetch_g += step * a.gate_stride;
    copies_close();
  };
  // rows being worked on, for where they begin in their blocks
  const T *row_x = fetch_x, *row_y = fetch_y, *row_g = fetch_g;
  auto take = [&](const uint8_t* stage, int array, const T* from, int c, F2 (&v)[4]) {
    if (VEC) take8<T, CH>(stage, array, c, v);
    else if (MODE == kShifted) take_shifted8<T>(stage + array * span + row_low(from), group_column(c, off), H, v);
    else take_span8<T>(stage + array * span + row_low(from), c, H, v);
    if (MODE == kEdges && partial(group_column(c, off), H)) clip8(group_column(c, off), H, v);
  };
  if (has_edges(MODE)) {                           // the parameters at the thread's columns, behind the ring
    const void* const from[3] = {a.pre_w, a.post_w, gate_kind == kGateChannel ? a.gate : nullptr};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (!from[k]) continue;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        F2 w[4];
        load8_at<T>(static_cast<const T*>(from[k]), group_column(c, off), H, 0.0f, w);
        put8<T, CH>(ring + a.ring * stage_bytes, k, c, w);
      }
    }
  }
  if (MODE == kAligned) clear_ring_ends<T, CH>(ring, stage_bytes, a.ring, a.arrays, H);
  for (int i = 0; i < a.ring; ++i) fetch(smem_address(ring) + i * stage_bytes);
  T* s_out = static_cast<T*>(a.s) + blockIdx.x * static_cast<int64_t>(H);
  T* h_out = static_cast<T*>(a.h) + blockIdx.x * static_cast<int64_t>(H);
  uint8_t* q_out = a.q + blockIdx.x * static_cast<int64_t>(H);
  const int64_t step_h = step * H;
  float next_gate = gate_kind == kGateToken && blockIdx.x < a.T ? token_gate<T>(a, blockIdx.x) : 1.0f;   // loaded a row ahead
  int slot = 0;
  for (int row = blockIdx.x; row < a.T; row += gridDim.x) {
    const uint8_t* const stage = ring + slot * stage_bytes;
    const float gate = next_gate;
    if (gate_kind == kGateToken && row + step < a.T) next_gate = token_gate<T>(a, row + step);
    ring_wait(a.ring);
    if (!VEC) __syncthreads();
    F2 s[CH][4];
    float r1 = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) take(stage, 0, row_x, c, s[c]);
    if (a.y) {
      F2 n[CH][4];
      F2 g[4];
      float k = gate;                              // what a whole row of y is multiplied by
#pragma unroll
      for (int c = 0; c < CH; ++c) take(stage, 1, row_y, c, n[c]);
      if (a.post_w) {
        F2 square = both(0.0f);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) square = fma2(n[c][j], n[c][j], square);
        float sum[1] = {total(square)};
        block_sum(sum, red[0]);
        r1 = rsqrtf(sum[0] * inv_h + a.eps);
        k *= r1;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          param(a.post_w, a.post_f32, 0, c, g);
#pragma unroll
          for (int j = 0; j < 4; ++j) n[c][j] = mul2(n[c][j], g[j]);
        }
      }
      if (gate_kind == kGateChannel || gate_kind == kGateFull) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          if (full_in_ring) take(stage, 2, row_g, c, g);
          else param(a.gate, a.gate_f32, gate_kind == kGateFull ? row * a.gate_stride : 0, c, g);
#pragma unroll
          for (int j = 0; j < 4; ++j) n[c][j] = mul2(n[c][j], g[j]);
        }
      }
      const F2 kk = both(k), aa = both(a.a);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[c][j] = fma2(aa, s[c][j], mul2(kk, n[c][j]));
        store_row8<T, MODE>(s_out, c, H, off, s[c]);
      }
    }
    if (VEC) fetch(smem_address(stage));
    F2 square = both(0.0f);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) square = fma2(s[c][j], s[c][j], square);
    float sum[1] = {total(square)};
    block_sum(sum, red[1]);
    if (!VEC) {                                    // everybody has read the stage
      fetch(smem_address(stage));
      row_x += step * a.x_stride;
      row_y += step * a.y_stride;
      row_g += step * a.gate_stride;
    }
    slot = slot + 1 == a.ring ? 0 : slot + 1;
    const float r2 = rsqrtf(sum[0] * inv_h + a.eps);
    if (threadIdx.x == 0) *reinterpret_cast<float2*>(a.rstd + 2 * static_cast<int64_t>(row)) = make_float2(r1, r2);
    const F2 rr = both(r2);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 w[4];
      param(a.pre_w, a.pre_f32, 0, c, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[c][j] = mul2(mul2(s[c][j], rr), w[j]);
      if (QUANT) {
        // sixteen lanes hold a block of 128 columns; scale = max(|h|, 1e-10) / 448 and e4m3(h / scale), the rule of the
        // activation quantiser and the same values (a zero loses its sign).  Both quotients are products with a reciprocal,
        // corrected by what they leave of the dividend.  For the constant that is the rounded quotient of every fp32 value
        // (checked for all mantissas; the method is Brisebarre, Muller and Raina's of 2004); for the values it is but for
        // ties of fp32, and no quotient of fp32 values lies that close to a tie of e4m3 without being one
        const int col = column<true>(c, 0);
        float amax = 1e-10f;
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(get(s[c][j]).x), fabsf(get(s[c][j]).y)));
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
        const float about = amax * (1.0f / 448.0f);
        const bool finite = about < INFINITY;              // an infinite block: zeros, NaN where it is infinite
        const float scale = finite ? fmaf(fmaf(-448.0f, about, amax), 1.0f / 448.0f, about) : about;
        const F2 inverse = both(__fdividef(1.0f, scale)), minus = both(finite ? -scale : 0.0f);
        uint32_t packed[2];
        float2 quotient[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const F2 near = mul2(s[c][j], inverse);
          quotient[j] = get(fma2(fma2(minus, near, s[c][j]), inverse, near));
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
          packed[j] = __nv_cvt_float2_to_fp8x2(quotient[2 * j], __NV_SATFINITE, __NV_E4M3) |
                      static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(quotient[2 * j + 1], __NV_SATFINITE, __NV_E4M3)) << 16;
        if (col < H) {
          *reinterpret_cast<uint2*>(q_out + col) = make_uint2(packed[0], packed[1]);
          if ((threadIdx.x & 15) == 0) a.q_scale[static_cast<int64_t>(col / kBlock) * a.T + row] = scale;
        }
      } else {
        store_row8<T, MODE>(h_out, c, H, off, s[c]);
      }
    }
    s_out += step_h;
    h_out += step_h;
    q_out += step_h;
    // red[0] of the next row is written only after every thread has passed the barrier of red[1], and without a first
    // sum red[1] would be written again while a slow thread reads it
    if (VEC && !a.post_w) __syncthreads();
  }
}

// Activations that a row's ring stage holds: x, y and a full gate of the same type.
int forward_arrays(const NormArgs& a, int size) {
  return 1 + (a.y ? 1 : 0) + (a.gate_kind == kGateFull && (!a.gate_f32 || size == 4) ? 1 : 0);
}

template <typename T, int CH, RowMode MODE, bool QUANT, int GATE>
cudaError_t launch_forward(NormArgs a, int threads, cudaStream_t stream) {
  const auto kernel = block_norm_kernel<T, CH, MODE, QUANT, GATE>;
  a.arrays = forward_arrays(a, sizeof(T));
  const size_t stage = static_cast<size_t>(a.arrays) * (by_block(MODE) ? CH * threads * sizeof(Pack8<T>) : span_bytes(a.H, sizeof(T)));
  const size_t weights = has_edges(MODE) ? 3 * CH * threads * sizeof(Pack8<T>) : 0;
  // as many CTAs as the registers are cut for, or fewer where their rings do not fit; two stages at least, if that can be
  // had
  int per_sm = 896 / threads > 0 ? 896 / threads : 1;
  while (per_sm > 1 && (2 * stage + weights) * per_sm > kRingMost) per_sm /= 2;
  a.ring = static_cast<int>((kRingMost / per_sm - weights) / stage);
  if (a.ring > kMaxRing) a.ring = kMaxRing;
  const size_t smem = a.ring * stage + weights;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(kernel, kSmemMost, done);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(grid_rows(a.T, per_sm, MODE)), dim3(threads), smem, stream, a);
}

template <typename T, int CH, RowMode MODE, bool QUANT>
cudaError_t launch_forward(const NormArgs& a, int threads, cudaStream_t stream) {
  if (a.gate_kind == kGateChannel) return launch_forward<T, CH, MODE, QUANT, kGateChannel>(a, threads, stream);
  if (a.gate_kind == kGateFull) return launch_forward<T, CH, MODE, QUANT, kGateFull>(a, threads, stream);
  return launch_forward<T, CH, MODE, QUANT, kGateNone>(a, threads, stream);
}

// `known`: the gate is compiled in (parameters have the activations' type and a thread has at most 16 columns).
template <typename T, int CH>
cudaError_t launch_forward(const NormArgs& a, RowMode mode, bool known, int threads, cudaStream_t stream) {
  constexpr int kCh = CH <= 2 ? CH : 1;
  if (mode == kEdges) return launch_forward<T, kCh, kEdges, false>(a, threads, stream);
  if (mode == kShifted) return launch_forward<T, kCh, kShifted, false>(a, threads, stream);
  if (mode == kSpan) return launch_forward<T, CH, kSpan, false, kAnyGate>(a, threads, stream);
  if (known) return a.q ? launch_forward<T, kCh, kAligned, true>(a, threads, stream) : launch_forward<T, kCh, kAligned, false>(a, threads, stream);
  return a.q ? launch_forward<T, CH, kAligned, true, kAnyGate>(a, threads, stream)
             : launch_forward<T, CH, kAligned, false, kAnyGate>(a, threads, stream);
}

template <typename T>
cudaError_t launch_forward(const NormArgs& a, RowMode mode, cudaStream_t stream) {
  const Shape sh = shape_of(counted_width(a.H, mode));
  const bool known = sh.ch <= 2 && (sizeof(T) == 4 || !(a.pre_f32 || a.post_f32 || a.gate_f32));
  if (sh.ch == 1) return launch_forward<T, 1>(a, mode, known, sh.threads, stream);
  if (sh.ch == 2) return launch_forward<T, 2>(a, mode, known, sh.threads, stream);
  return launch_forward<T, 4>(a, mode, known, sh.threads, stream);
}
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
  if (!x || !pre_weight || !h || !rstd || !aligned(rstd, 8) || !aligned(h_scale, 4) || (y && !stream_out)) return MOE_B200_EINVAL;
  const RowMode mode = row_mode(a, dtype);
  if (h_scale && (H % kBlock != 0 || mode != kAligned)) return MOE_B200_EINVAL;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  cudaError_t e;
  if (dtype == MOE_B200_F32) e = launch_forward<float>(a, mode, stream);
  else if (dtype == MOE_B200_BF16) e = launch_forward<__nv_bfloat16>(a, mode, stream);
  else e = launch_forward<__half>(a, mode, stream);
  return launch_status(e, 1);
}
