// Gradients of the norms before and after a block (block_norm.cu has the forward and its formulas).
//
// Backward, per row, with D = dL/ds, u = gh w_pre, sh = s r2, yh = y r1, n = yh w_post:
//     D  = gs + r2 (u - sh mean(u sh)),      dx = a D,      dg = D n (summed over what the gate is broadcast along)
//     dy = r1 (D g w_post - yh mean(D g w_post yh))         (D g without w_post)
//     dw_pre = sum_t gh sh,   dw_post = sum_t D g yh
// s is formed again from x and y (two rows read instead of the rounded s and y), r1 and r2 come from the forward.
#include "block_norm.cuh"

namespace moe {
namespace {

// Rows are dealt to the CTAs round-robin; the column sums of a CTA's rows stay with the thread that owns the columns and
// leave once, as one partial row per CTA, which column_sum_kernel adds in CTA order: no atomics, the same bits every time.
// The dot products of a row need one reduction: with D = d - sh k2, d = gs + r2 u and v = n (times a gate per column),
//     k2 = r2 mean(u sh),   sum_h D v = sum d v - k2 sum sh v,   mean(D g w_post yh) = that (times a gate per token) / H.
//
// Two kernels: this one for all cases, with its column sums in shared memory ...
template <typename T, int CH, bool VEC>
__global__ void __launch_bounds__(kNormThreads) block_norm_backward_kernel(NormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  extern __shared__ float acc[];             // [n_sums][CH * 8][blockDim.x], thread-private columns
  __shared__ float red[2][96];
  const int H = a.H, nt = blockDim.x, tid = threadIdx.x;
  const float inv_h = 1.0f / static_cast<float>(H);
  auto add_to = [&](int sum, int c, int j, F2 v) {
    float* at = acc + (sum * CH * 8 + c * 8 + 2 * j) * nt + tid;
    const float2 f = get(v);
    at[0] += f.x;
    at[nt] += f.y;
  };
  for (int i = 0; i < a.n_sums * CH * 8; ++i) acc[i * nt + tid] = 0.0f;
  int flip = 0;
  for (int row = blockIdx.x; row < a.T; row += gridDim.x, flip ^= 1) {
    const float r1 = a.rstd[2 * static_cast<int64_t>(row)], r2 = a.rstd[2 * static_cast<int64_t>(row) + 1];
    const float gt = a.gate_kind == kGateToken ? token_gate<T>(a, row) : 1.0f;
    F2 sh[CH][4], d[CH][4], yh[CH][4];
    F2 dots[3] = {both(0.0f), both(0.0f), both(0.0f)};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 u[4], w[4], g[4], wp[4];
      load8<T, VEC>(static_cast<const T*>(a.x) + row * a.x_stride, c, H, sh[c]);
      load8<T, VEC>(static_cast<const T*>(a.gh) + row * a.gh_stride, c, H, u);
      load8_param<T, VEC>(a.pre_w, a.pre_f32, 0, c, H, w);
      if (a.gs) {
        load8<T, VEC>(static_cast<const T*>(a.gs) + row * a.gs_stride, c, H, d[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[c][j] = both(0.0f);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) { g[j] = wp[j] = both(1.0f); yh[c][j] = both(0.0f); }
      if (a.y) {
        load8<T, VEC>(static_cast<const T*>(a.y) + row * a.y_stride, c, H, yh[c]);
        if (a.post_w) {
          load8_param<T, VEC>(a.post_w, a.post_f32, 0, c, H, wp);
#pragma unroll
          for (int j = 0; j < 4; ++j) yh[c][j] = mul2(yh[c][j], both(r1));
        }
        if (a.gate_kind == kGateChannel || a.gate_kind == kGateFull)
          load8_param<T, VEC>(a.gate, a.gate_f32, a.gate_kind == kGateFull ? row * a.gate_stride : 0, c, H, g);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const F2 v = mul2(mul2(yh[c][j], wp[j]), g[j]);
        if (a.y) sh[c][j] = fma2(both(a.a), sh[c][j], mul2(both(gt), v));
        sh[c][j] = mul2(sh[c][j], both(r2));
        add_to(0, c, j, mul2(u[j], sh[c][j]));            // dw_pre
        u[j] = mul2(u[j], w[j]);
        d[c][j] = fma2(both(r2), u[j], d[c][j]);
        dots[0] = fma2(u[j], sh[c][j], dots[0]);
        dots[1] = fma2(d[c][j], v, dots[1]);
        dots[2] = fma2(sh[c][j], v, dots[2]);
      }
    }
    float sums[3] = {total(dots[0]), total(dots[1]), total(dots[2])};
    block_sum(sums, red[flip]);
    const float k2 = r2 * (sums[0] * inv_h);
    const float dv = sums[1] - k2 * sums[2];
    if (a.gate_kind == kGateToken && tid == 0) {
      if (a.gate_f32) static_cast<float*>(a.dgate_rows)[row] = dv;
      else static_cast<T*>(a.dgate_rows)[row] = from_f32<T>(dv);
    }
    const float k1 = dv * gt * inv_h;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 g[4], wp[4], out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[c][j] = fma2(both(-k2), sh[c][j], d[c][j]);
        out[j] = a.y ? mul2(both(a.a), d[c][j]) : d[c][j];
        g[j] = both(gt);
        wp[j] = both(1.0f);
      }
      store8<T, VEC>(static_cast<T*>(a.dx) + static_cast<int64_t>(row) * H, c, H, out);
      if (!a.y) continue;
      if (a.gate_kind == kGateChannel || a.gate_kind == kGateFull)
        load8_param<T, VEC>(a.gate, a.gate_f32, a.gate_kind == kGateFull ? row * a.gate_stride : 0, c, H, g);
      if (a.post_w) load8_param<T, VEC>(a.post_w, a.post_f32, 0, c, H, wp);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = mul2(d[c][j], mul2(yh[c][j], wp[j]));
      if (a.gate_kind == kGateFull) {
        if (a.gate_f32) store8<float, VEC>(static_cast<float*>(a.dgate_rows) + static_cast<int64_t>(row) * H, c, H, out);
        else store8<T, VEC>(static_cast<T*>(a.dgate_rows) + static_cast<int64_t>(row) * H, c, H, out);
      } else if (a.sum_gate >= 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) add_to(a.sum_gate, c, j, out[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const F2 dn = mul2(d[c][j], g[j]);
        out[j] = dn;
        if (a.post_w) {
          add_to(a.sum_post, c, j, mul2(dn, yh[c][j]));
          out[j] = mul2(both(r1), fma2(both(-k1), yh[c][j], mul2(dn, wp[j])));
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

// ... and this one where parameters have the activations' type and a row fits 16 columns a thread and the ring: the
// rows come through a ring like the forward's, the column sums stay in registers as fp32, and the weights, which leave no
// registers for themselves, in shared memory behind the ring (an SM's quarter has 128 registers for each of four warps).
// Missing parts are neutral values (y = 0, w_post = 1, gate = 1) instead of branches.  Bound by HBM at many rows (x, y, gh,
// gs in; dx, dy out).  Measured, 16384 x 7168 bf16 with a gate per channel: 305 us (4.6 TB/s) for both kernels, 809 us with
// the kernel above; 4096 x 7168 with a full gate 98 us (4.8 TB/s); 4096 x 5001 97 us.
template <typename T, int CH, RowMode MODE, int GATE>
__global__ void __launch_bounds__(kNormThreads) block_norm_backward_ring_kernel(NormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr bool VEC = by_block(MODE);
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2][96];
  const int H = a.H;
  const float inv_h = 1.0f / static_cast<float>(H), scale = a.y ? a.a : 1.0f;
  const int span = span_bytes(H, sizeof(T));
  const int off = has_edges(MODE) ? static_cast<int>(blockIdx.x * static_cast<int64_t>(H) % (16 / static_cast<int>(sizeof(T)))) : 0;
  const uint32_t stage_bytes = static_cast<uint32_t>(a.arrays * (VEC ? CH * blockDim.x * sizeof(Pack8<T>) : span));
  auto fetch_one = [&](uint32_t stage, int array, const void* p, int64_t at) {
    if (VEC) fetch_row<T, CH, MODE>(stage, array, static_cast<const T*>(p) + at, H, off);
    else fetch_span(stage + array * span, static_cast<const T*>(p) + at, H);
  };
  // arrays of a stage: x, grad_h, grad_stream, y, gate; what the call lacks is never copied and stays zero
  auto fetch = [&](int64_t row, uint32_t stage) {
    if (row < a.T) {
      fetch_one(stage, 0, a.x, row * a.x_stride);
      fetch_one(stage, 1, a.gh, row * a.gh_stride);
      if (a.gs) fetch_one(stage, 2, a.gs, row * a.gs_stride);
      if (a.y) fetch_one(stage, 3, a.y, row * a.y_stride);
      if (GATE == kGateFull) fetch_one(stage, 4, a.gate, row * a.gate_stride);
    }
    copies_close();
  };
  for (uint32_t i = threadIdx.x * 16; i < a.ring * stage_bytes; i += blockDim.x * 16) *reinterpret_cast<uint4*>(ring + i) = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  for (int i = 0; i < a.ring - (VEC ? 0 : 1); ++i) fetch(blockIdx.x + static_cast<int64_t>(i) * gridDim.x, smem_address(ring) + i * stage_bytes);

  auto take = [&](const uint8_t* stage, int array, const void* p, int64_t at, int c, F2 (&v)[4]) {
    if (VEC) take8<T, CH>(stage, array, c, v);
    else if (p) take_shifted8<T>(stage + array * span + row_low(static_cast<const T*>(p) + at), group_column(c, off), H, v);
    else v[0] = v[1] = v[2] = v[3] = both(0.0f);
    if (MODE == kEdges && partial(group_column(c, off), H)) clip8(group_column(c, off), H, v);
  };
  uint8_t* const weights = ring + a.ring * stage_bytes;    // w_pre, w_post, gate per channel: the thread's own pieces
  F2 sum_pre[CH][4], sum_post[CH][4], sum_gate[GATE == kGateChannel ? CH : 1][4];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const void* const from[3] = {a.pre_w, a.post_w, GATE == kGateChannel ? a.gate : nullptr};
#pragma unroll
    for (int k = 0; k < (GATE == kGateChannel ? 3 : 2); ++k) {
      F2 w[4] = {both(1.0f), both(1.0f), both(1.0f), both(1.0f)};
      if (from[k]) {
        if (has_edges(MODE)) load8_at<T>(static_cast<const T*>(from[k]), group_column(c, off), H, 1.0f, w);
        else load8<T, true>(static_cast<const T*>(from[k]), c, H, w);
      }
      put8<T, CH>(weights, k, c, w);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum_pre[c][j] = sum_post[c][j] = both(0.0f);
      if (GATE == kGateChannel) sum_gate[c][j] = both(0.0f);
    }
  }

  // a row's statistics and gate are loaded a row ahead
  auto stats = [&](int64_t row, float& r1, float& r2, float& gt) {
    r1 = r2 = gt = 1.0f;
    if (row >= a.T) return;
    const float2 r = *reinterpret_cast<const float2*>(a.rstd + 2 * row);
    r2 = r.y;
    if (a.post_w) r1 = r.x;
    if (GATE == kGateNone && a.gate_kind == kGateToken) gt = token_gate<T>(a, row);
  };
  float next_r1, next_r2, next_gt;
  stats(blockIdx.x, next_r1, next_r2, next_gt);
  int flip = 0, slot = 0;
  for (int row = blockIdx.x; row < a.T; row += gridDim.x, flip ^= 1) {
    const uint8_t* const stage = ring + slot * stage_bytes;
    const float r1 = next_r1, r2 = next_r2, gt = next_gt;
    stats(row + static_cast<int64_t>(gridDim.x), next_r1, next_r2, next_gt);
    if (VEC) {
      ring_wait(a.ring);
    } else {
      // the stage of the row before is free once all threads are here: a ring of n stages runs n - 1 rows ahead
      if (a.ring == 3) copies_wait<1>();
      else copies_wait<0>();
      __syncthreads();
      fetch(row + static_cast<int64_t>(a.ring - 1) * gridDim.x, smem_address(ring) + (slot == 0 ? a.ring - 1 : slot - 1) * stage_bytes);
    }
    F2 sh[CH][4], d[CH][4];
    F2 dots[3] = {both(0.0f), both(0.0f), both(0.0f)};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 u[4], w[4], g[4], wp[4], yh[4];
      take(stage, 0, a.x, row * a.x_stride, c, sh[c]);
      take(stage, 1, a.gh, row * a.gh_stride, c, u);
      take(stage, 2, a.gs, row * a.gs_stride, c, d[c]);
      take(stage, 3, a.y, row * a.y_stride, c, yh);
      take8<T, CH>(weights, 0, c, w);
      take8<T, CH>(weights, 1, c, wp);
      if (GATE == kGateChannel) take8<T, CH>(weights, 2, c, g);
      if (GATE == kGateFull) take(stage, 4, a.gate, row * a.gate_stride, c, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        F2 v = mul2(mul2(yh[j], both(r1)), wp[j]);
        if (GATE != kGateNone) v = mul2(v, g[j]);
        sh[c][j] = mul2(fma2(both(scale), sh[c][j], GATE == kGateNone ? mul2(both(gt), v) : v), both(r2));
        sum_pre[c][j] = fma2(u[j], sh[c][j], sum_pre[c][j]);
        u[j] = mul2(u[j], w[j]);
        d[c][j] = fma2(both(r2), u[j], d[c][j]);
        dots[0] = fma2(u[j], sh[c][j], dots[0]);
        dots[1] = fma2(d[c][j], v, dots[1]);
        dots[2] = fma2(sh[c][j], v, dots[2]);
      }
    }
    float sums[3] = {total(dots[0]), total(dots[1]), total(dots[2])};
    block_sum(sums, red[flip]);
    const float k2 = r2 * (sums[0] * inv_h);
    const float dv = sums[1] - k2 * sums[2];
    if (GATE == kGateNone && a.gate_kind == kGateToken && threadIdx.x == 0) static_cast<T*>(a.dgate_rows)[row] = from_f32<T>(dv);
    const float k1 = a.post_w ? dv * gt * inv_h * r1 : 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 g[4], wp[4], out[4], yh[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[c][j] = fma2(both(-k2), sh[c][j], d[c][j]);
        out[j] = mul2(both(scale), d[c][j]);
      }
      store_row8<T, MODE>(static_cast<T*>(a.dx) + static_cast<int64_t>(row) * H, c, H, off, out);
      if (!a.y) continue;
      take(stage, 3, a.y, row * a.y_stride, c, yh);               // read again: registers are what this kernel is short of
      take8<T, CH>(weights, 1, c, wp);
#pragma unroll
      for (int j = 0; j < 4; ++j) yh[j] = mul2(yh[j], both(r1));
      if (GATE == kGateChannel) take8<T, CH>(weights, 2, c, g);
      if (GATE == kGateFull) take(stage, 4, a.gate, row * a.gate_stride, c, g);
      if (GATE != kGateNone) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const F2 n = mul2(yh[j], wp[j]);
          if (GATE == kGateChannel) sum_gate[c][j] = fma2(d[c][j], n, sum_gate[c][j]);
          else out[j] = mul2(d[c][j], n);
        }
        if (GATE == kGateFull) store_row8<T, MODE>(static_cast<T*>(a.dgate_rows) + static_cast<int64_t>(row) * H, c, H, off, out);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const F2 dn = mul2(d[c][j], GATE == kGateNone ? both(gt) : g[j]);
        sum_post[c][j] = fma2(dn, yh[j], sum_post[c][j]);
        out[j] = fma2(both(-k1), yh[j], mul2(mul2(dn, wp[j]), both(r1)));
      }
      store_row8<T, MODE>(static_cast<T*>(a.dy) + static_cast<int64_t>(row) * H, c, H, off, out);
    }
    if (VEC) fetch(row + static_cast<int64_t>(a.ring) * gridDim.x, smem_address(stage));
    slot = slot + 1 == a.ring ? 0 : slot + 1;
  }
  float* dst = a.partial + static_cast<int64_t>(blockIdx.x) * a.n_sums * H;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    store_row8<float, MODE>(dst, c, H, off, sum_pre[c], false);
    if (a.sum_post >= 0) store_row8<float, MODE>(dst + static_cast<int64_t>(a.sum_post) * H, c, H, off, sum_post[c], false);
    if (GATE == kGateChannel) store_row8<float, MODE>(dst + static_cast<int64_t>(a.sum_gate) * H, c, H, off, sum_gate[c], false);
  }
}

struct ColumnSumArgs {
  const float* partial;    // [n_parts][n_sums][H]
  int n_parts, n_sums, H;
  void* out[3];
  int f32[3];
};

constexpr int kSumStrips = 8, kSumAhead = 20;

// out[k][col] = sum over the parts in order, in eight interleaved strips that are joined in order.  A long or a narrow batch
// has thousands of parts, so what the additions lose is kept beside the sums.  Loads go out twenty at a time, all of a strip
// in one wave of CTAs (16384 x 512, 1184 parts: 36 us for both kernels, 41 with eight).
template <typename T>
__global__ void __launch_bounds__(32 * kSumStrips) column_sum_kernel(ColumnSumArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float strip[2][kSumStrips][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, k = blockIdx.y;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.0f, lost = 0.0f;
  if (col < a.H) {
    const float* const from = a.partial + static_cast<int64_t>(k) * a.H + col;
    const int64_t row = static_cast<int64_t>(a.n_sums) * a.H;
    for (int p = w; p < a.n_parts; p += kSumStrips * kSumAhead) {
      float v[kSumAhead];
#pragma unroll
      for (int i = 0; i < kSumAhead; ++i) v[i] = p + i * kSumStrips < a.n_parts ? from[(p + i * kSumStrips) * row] : 0.0f;
#pragma unroll
      for (int i = 0; i < kSumAhead; ++i) add_exactly(s, lost, v[i]);
    }
  }
  strip[0][w][lane] = s;
  strip[1][w][lane] = lost;
  __syncthreads();
  if (w == 0 && col < a.H) {
    float t = 0.0f, low = 0.0f;
#pragma unroll
    for (int i = 0; i < kSumStrips; ++i) {
      add_exactly(t, low, strip[0][i][lane]);
      low += strip[1][i][lane];
    }
    t = joined(t, low);
    if (a.f32[k]) static_cast<float*>(a.out[k])[col] = t;
    else static_cast<T*>(a.out[k])[col] = from_f32<T>(t);
  }
}

// CTAs of the backward pass, one partial row of column sums each: as many as the registers hold, or a multiple of that, one
// wave after another, so that none has more than kSumRows rows.  A sum in fp32 over more would lose the terms below its last
// bit; over kSumRows it is off by 256 * 2^-24 / 2 = 2^-17 of the terms' magnitudes at most.  A wave costs some 20 us (the
// ring fills again): 65536 x 7168 takes two and 1197 us, where sums over all rows took 1173.  (Partial rows written inside
// the loop over the rows save half of that and cost batches of one wave up to 20 %: the loop has no registers left.)
constexpr int kSumRows = 256;
int backward_parts(int T, int H, RowMode mode) {
  const Shape sh = backward_shape_of(counted_width(H, mode));
  const int at_once = grid_rows(T, sh.ch > 1 ? 1 : 512 / sh.threads, mode);
  return at_once > 0 ? at_once * ((T - 1) / (at_once * kSumRows) + 1) : 0;
}

template <typename T, int CH, bool VEC>
cudaError_t launch_backward(const NormArgs& a, int grid, int threads, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(a.n_sums) * CH * 8 * threads * sizeof(float);
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(block_norm_backward_kernel<T, CH, VEC>, kSmemMost, done);
  if (e != cudaSuccess) return e;
  return launch_pdl(block_norm_backward_kernel<T, CH, VEC>, dim3(grid), dim3(threads), smem, stream, a);
}

// Whether the ring kernel takes this call (a longer row or a mixed call goes to the other one), its stages and memory.
template <typename T>
bool ring_plan(NormArgs& a, RowMode mode, size_t* smem) {
  const Shape sh = backward_shape_of(counted_width(a.H, mode));
  if (mode == kSpan || sh.ch > 2 || (sizeof(T) == 2 && (a.pre_f32 || a.post_f32 || a.gate_f32))) return false;
  a.arrays = a.gate_kind == kGateFull ? 5 : 4;
  const size_t array = static_cast<size_t>(sh.ch) * sh.threads * sizeof(Pack8<T>), weights = 3 * array;
  const size_t stage = a.arrays * (by_block(mode) ? array : span_bytes(a.H, sizeof(T)));
  const size_t room = 220 * 1024 / (sh.ch == 1 ? 512 / sh.threads : 1) - 2048;
  a.ring = room > weights ? static_cast<int>((room - weights) / stage) : 0;
  if (a.ring > kMaxRing) a.ring = kMaxRing;
  *smem = a.ring * stage + weights;
  return a.ring >= 2;
}
template <typename T>
bool ring_fits(NormArgs a, RowMode mode) {
  size_t smem;
  return ring_plan<T>(a, mode, &smem);
}

template <typename T, int CH, RowMode MODE, int GATE>
cudaError_t launch_ring(const NormArgs& a, int grid, int threads, size_t smem, cudaStream_t stream) {
  const auto kernel = block_norm_backward_ring_kernel<T, CH, MODE, GATE>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(kernel, kSmemMost, done);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(grid), dim3(threads), smem, stream, a);
}

template <typename T, int CH, RowMode MODE>
cudaError_t launch_ring(const NormArgs& a, int grid, int threads, size_t smem, cudaStream_t stream) {
  if (a.gate_kind == kGateChannel) return launch_ring<T, CH, MODE, kGateChannel>(a, grid, threads, smem, stream);
  if (a.gate_kind == kGateFull) return launch_ring<T, CH, MODE, kGateFull>(a, grid, threads, smem, stream);
  return launch_ring<T, CH, MODE, kGateNone>(a, grid, threads, smem, stream);
}

template <typename T, int CH>
cudaError_t launch_ring(const NormArgs& a, RowMode mode, int grid, int threads, size_t smem, cudaStream_t stream) {
  if (mode == kAligned) return launch_ring<T, CH, kAligned>(a, grid, threads, smem, stream);
  if (mode == kEdges) return launch_ring<T, CH, kEdges>(a, grid, threads, smem, stream);
  return launch_ring<T, CH, kShifted>(a, grid, threads, smem, stream);
}

template <typename T>
cudaError_t launch_backward(NormArgs a, ColumnSumArgs cs, RowMode mode, cudaStream_t stream) {
  if (has_edges(mode) && !ring_fits<T>(a, mode)) mode = kSpan;
  const Shape sh = backward_shape_of(counted_width(a.H, mode));
  cs.n_parts = backward_parts(a.T, a.H, mode);
  const int grid = cs.n_parts, nt = sh.threads;
  size_t smem = 0;
  const bool vec = mode == kAligned;
  cudaError_t e;
  if (ring_plan<T>(a, mode, &smem)) {
    e = sh.ch == 1 ? launch_ring<T, 1>(a, mode, grid, nt, smem, stream) : launch_ring<T, 2>(a, mode, grid, nt, smem, stream);
  } else if (sh.ch == 1) {
    e = vec ? launch_backward<T, 1, true>(a, grid, nt, stream) : launch_backward<T, 1, false>(a, grid, nt, stream);
  } else if (sh.ch == 2) {
    e = vec ? launch_backward<T, 2, true>(a, grid, nt, stream) : launch_backward<T, 2, false>(a, grid, nt, stream);
  } else {
    e = vec ? launch_backward<T, 4, true>(a, grid, nt, stream) : launch_backward<T, 4, false>(a, grid, nt, stream);
  }
  if (e != cudaSuccess) return e;
  return launch_pdl(column_sum_kernel<T>, dim3((a.H + 31) / 32, cs.n_sums), dim3(32 * kSumStrips), 0, stream, cs);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_fp8_block_scale_block_norm_backward_workspace_bytes(int T, int H) {
  if (T < 0 || H < 1 || H > kMaxWidth) return 0;
  int parts = 0;
  for (RowMode mode : {kSpan, kEdges}) {
    const int n = backward_parts(T, H, mode);
    parts = n > parts ? n : parts;
  }
  return static_cast<size_t>(parts) * 3 * H * sizeof(float);
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
  if (!x || !pre_weight || !rstd || !aligned(rstd, 8) || !grad_h || !grad_x || !grad_pre_weight || (y && !grad_y) ||
      (post_weight && !grad_post_weight) || (gate_kind != kGateNone && !grad_gate) || !workspace || !aligned(workspace, 16))
    return MOE_B200_EINVAL;
  const int size = element_size(dtype);
  if (!aligned(grad_pre_weight, a.pre_f32 ? 4 : size) || !aligned(grad_post_weight, a.post_f32 ? 4 : size) ||
      !aligned(grad_gate, a.gate_f32 ? 4 : size))
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
  cs.n_sums = a.n_sums;
  cs.H = H;
  const RowMode mode = row_mode(a, dtype);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  cudaError_t e;
  if (dtype == MOE_B200_F32) e = launch_backward<float>(a, cs, mode, stream);
  else if (dtype == MOE_B200_BF16) e = launch_backward<__nv_bfloat16>(a, cs, mode, stream);
  else e = launch_backward<__half>(a, cs, mode, stream);
  return launch_status(e, 2);
}
