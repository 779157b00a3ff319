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
constexpr int kMostTokens = 1 << 30;       // row indexes and a grid's step stay within an int
constexpr int kNormThreads = 512;

enum GateKind : int { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

struct NormArgs {
  const void *x, *y, *gate, *pre_w, *post_w;
  int64_t x_stride, y_stride, gate_stride;   // elements between rows
  int T, H, gate_kind;
  int arrays, ring;                          // activations that go through the ring, its stages
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

// How rows are read and written.  kAligned: every row starts on 16 bytes.  kEdges: all row arrays are off by the same in
// every row (an odd width, strides that differ from it by whole 16 bytes, aligned bases): blocks of 16 bytes are still
// shared by loads and stores, the first and last one of a row are partial.  With a grid that is a multiple of eight, or
// one row per CTA, a CTA's rows are all off by the same, so that its threads keep their columns.  kShifted: the results are
// such rows, the inputs start anywhere: they come as the aligned blocks that cover them and are shifted when they are read.
// kSpan: anything else, element by element.
enum RowMode : int { kSpan = 0, kAligned = 1, kEdges = 2, kShifted = 3 };
__host__ __device__ constexpr bool by_block(RowMode m) { return m == kAligned || m == kEdges; }     // a thread reads what it copied
__host__ __device__ constexpr bool has_edges(RowMode m) { return m == kEdges || m == kShifted; }    // columns begin in front of the row

// Which column a thread's j-th element of chunk c is: eight neighbours where rows can be read 16 bytes at a time,
// else columns blockDim.x apart, so that single-element loads of a warp are adjacent.
template <bool VEC>
__device__ __forceinline__ int column(int c, int j) {
  return VEC ? (c * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8 + j
             : (c * 8 + j) * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
}

// Eight columns of a row as four pairs, zeros behind the row's end.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int c, int H, F2 (&v)[4]) {
  if (VEC) {
    const int col = column<VEC>(c, 0);
    if (col < H) {
      unpack8<T>(*reinterpret_cast<const Pack8<T>*>(p + col), v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = both(0.0f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c0 = column<VEC>(c, 2 * j), c1 = column<VEC>(c, 2 * j + 1);
      v[j] = make_f2(c0 < H ? to_f32<T>(p[c0]) : 0.0f, c1 < H ? to_f32<T>(p[c1]) : 0.0f);
    }
  }
}

// A parameter row (weight or gate) in the activations' type or in fp32.
template <typename T, bool VEC>
__device__ __forceinline__ void load8_param(const void* p, int f32, int64_t row_offset, int c, int H, F2 (&v)[4]) {
  if (f32)
    load8<float, VEC>(static_cast<const float*>(p) + row_offset, c, H, v);
  else
    load8<T, VEC>(static_cast<const T*>(p) + row_offset, c, H, v);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int c, int H, const F2 (&v)[4]) {
  if (VEC) {
    const int col = column<VEC>(c, 0);
    if (col < H) *reinterpret_cast<Pack8<T>*>(p + col) = pack8<T>(v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c0 = column<VEC>(c, 2 * j), c1 = column<VEC>(c, 2 * j + 1);
      const float2 f = get(v[j]);
      if (c0 < H) p[c0] = from_f32<T>(f.x);
      if (c1 < H) p[c1] = from_f32<T>(f.y);
    }
  }
}

template <typename T>
__device__ __forceinline__ float token_gate(const NormArgs& a, int64_t row) {
  const int64_t at = row * a.gate_stride;
  return a.gate_f32 ? static_cast<const float*>(a.gate)[at] : to_f32<T>(static_cast<const T*>(a.gate)[at]);
}

// ---- Forward
//
// Bound by HBM (x, y in; s, h out), so the loads must never wait for the two reductions of a row: persistent CTAs bring
// the rows of x, y (and a full gate) that they will need through a ring of up to three stages (cp.async).  Every thread
// copies exactly the sixteen-byte pieces that it will read itself, so the ring needs no barrier.  Weights come from the
// first-level cache, which the copies pass by.  A thread has sixteen columns of a row of 4096 and more: two CTAs of 448
// threads at 7168 columns, whose barriers fill each other's gaps.
// Measured, 4096 x 7168 bf16: join and norm 47 us (5.0 TB/s), with e4m3 output 50 us (4.2 TB/s: 61 % of the issue slots
// are taken, the conversion's maximum and products among them); without the ring 79 us.  4096 x 5001 (kEdges) 44 us, with
// rows 5006 apart (kShifted) 59 us, element by element 180 us.
constexpr int kMaxRing = 3;

// Until the oldest of `ring` stages in flight has landed.
__device__ __forceinline__ void ring_wait(int ring) {
  if (ring == 3) copies_wait<2>();
  else if (ring == 2) copies_wait<1>();
  else copies_wait<0>();
}

// The row's share of one thread in a stage: CH groups of eight columns of every array.
template <typename T, int CH>
__device__ __forceinline__ uint32_t piece(int array, int c) {
  return (array * CH + c) * blockDim.x * sizeof(Pack8<T>) + threadIdx.x * 16;
}

// First column of a thread's group c where rows begin `off` elements behind 16 bytes.
__device__ __forceinline__ int group_column(int c, int off) { return column<true>(c, 0) - off; }

template <typename T, int CH, RowMode MODE>
__device__ __forceinline__ void fetch_row(uint32_t stage, int array, const T* row, int H, int off) {
  constexpr int kBlockElems = 16 / static_cast<int>(sizeof(T));
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = group_column(c, off);
    if (col >= H) continue;
#pragma unroll
    for (int half = 0; half < static_cast<int>(sizeof(T)) / 2; ++half) {
      const uint32_t to = stage + piece<T, CH>(array, c) + half * 16 * blockDim.x;
      const int first = col + half * kBlockElems;
      if (MODE == kAligned) copy16(to, row + first, true);
      else if (first < H)    // the row's bytes and, in its first block, those in front of it
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(row + first),
                     "r"(min(kBlockElems, H - first) * static_cast<int>(sizeof(T))) : "memory");
    }
  }
}

// Zeros where a group of eight columns from `col` lies outside the row.
__device__ __forceinline__ void clip8(int col, int H, F2 (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = get(v[j]);
    v[j] = make_f2(col + 2 * j >= 0 && col + 2 * j < H ? f.x : 0.0f, col + 2 * j + 1 >= 0 && col + 2 * j + 1 < H ? f.y : 0.0f);
  }
}
__device__ __forceinline__ bool partial(int col, int H) { return col < 0 || col + 8 > H; }

// Eight columns from `col` on of a row that starts at p, outside it `fill`.
template <typename T>
__device__ __forceinline__ void load8_at(const T* p, int col, int H, float fill, F2 (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c0 = col + 2 * j, c1 = c0 + 1;
    v[j] = make_f2(c0 >= 0 && c0 < H ? to_f32<T>(p[c0]) : fill, c1 >= 0 && c1 < H ? to_f32<T>(p[c1]) : fill);
  }
}

template <typename T, RowMode MODE>
__device__ __forceinline__ void store_row8(T* p, int c, int H, int off, const F2 (&v)[4], bool whole_blocks = true) {
  if (!has_edges(MODE)) {
    store8<T, MODE == kAligned>(p, c, H, v);
    return;
  }
  const int col = group_column(c, off);
  if (whole_blocks && !partial(col, H)) {
    *reinterpret_cast<Pack8<T>*>(p + col) = pack8<T>(v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = get(v[j]);
    if (col + 2 * j >= 0 && col + 2 * j < H) p[col + 2 * j] = from_f32<T>(f.x);
    if (col + 2 * j + 1 >= 0 && col + 2 * j + 1 < H) p[col + 2 * j + 1] = from_f32<T>(f.y);
  }
}

template <typename T, int CH>
__device__ __forceinline__ void take8(const uint8_t* stage, int array, int c, F2 (&v)[4]) {
  Pack8<T> raw;
#pragma unroll
  for (int half = 0; half < static_cast<int>(sizeof(T)) / 2; ++half)
    raw.w[half] = *reinterpret_cast<const uint4*>(stage + piece<T, CH>(array, c) + half * 16 * blockDim.x);
  unpack8<T>(raw, v);
}

template <typename T, int CH>
__device__ __forceinline__ void put8(uint8_t* stage, int array, int c, const F2 (&v)[4]) {
  const Pack8<T> raw = pack8<T>(v);
#pragma unroll
  for (int half = 0; half < static_cast<int>(sizeof(T)) / 2; ++half)
    *reinterpret_cast<uint4*>(stage + piece<T, CH>(array, c) + half * 16 * blockDim.x) = raw.w[half];
}

// Pieces behind the end of an aligned row are never copied: they hold zeros.  (Rows with edges are clipped when they are read.)
template <typename T, int CH>
__device__ __forceinline__ void clear_ring_ends(uint8_t* ring, uint32_t stage_bytes, int stages, int arrays, int H) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (group_column(c, 0) < H) continue;
    for (int i = 0; i < stages * arrays; ++i)
      for (int half = 0; half < static_cast<int>(sizeof(T)) / 2; ++half)
        *reinterpret_cast<uint4*>(ring + i / arrays * stage_bytes + piece<T, CH>(i % arrays, c) + half * 16 * blockDim.x) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// Rows that start anywhere go through the ring as the aligned blocks that cover them; the last one brings only the row's
// bytes, so that nothing behind the row is read, and the bytes in front of the row lie in the same 16 bytes of the same
// allocation.  A thread then reads what others copied: these kernels have a barrier after the wait.
__host__ __device__ constexpr int span_bytes(int H, int size) { return (H * size + 15) / 16 * 16 + 16; }

template <typename T>
__device__ __forceinline__ void fetch_span(uint32_t to, const T* row, int H) {
  const uintptr_t from = reinterpret_cast<uintptr_t>(row) & ~uintptr_t(15);
  const int bytes = static_cast<int>(reinterpret_cast<uintptr_t>(row) - from) + H * static_cast<int>(sizeof(T));
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i), "l"(from + i), "r"(min(16, bytes - i)) : "memory");
}

template <typename T>
__device__ __forceinline__ int row_low(const T* row) { return static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15); }

// Eight columns from `col` on of a row in shared memory that starts at `row`, on any element.
__device__ __forceinline__ void shifted8(const uint8_t* at, F2 (&v)[4], float) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = make_f2(reinterpret_cast<const float*>(at)[2 * j], reinterpret_cast<const float*>(at)[2 * j + 1]);
}
template <typename T>
__device__ __forceinline__ void shifted8(const uint8_t* at, F2 (&v)[4], T) {
  const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 2) * 8;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(at - odd / 8);
  uint32_t w[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) w[j] = words[j];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = unpack2(__funnelshift_r(w[j], w[j + 1], odd), T());
}
template <typename T>
__device__ __forceinline__ void take_shifted8(const uint8_t* row, int col, int H, F2 (&v)[4]) {
  if (partial(col, H)) load8_at<T>(reinterpret_cast<const T*>(row), col, H, 0.0f, v);
  else shifted8(row + col * static_cast<int>(sizeof(T)), v, T());
}

template <typename T>
__device__ __forceinline__ void take_span8(const uint8_t* row, int c, int H, F2 (&v)[4]) {
  load8<T, false>(reinterpret_cast<const T*>(row), c, H, v);
}

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
        // activation quantiser, with products of reciprocals (errors of 2^-22 before the rounding to e4m3's 2^-4)
        const int col = column<true>(c, 0);
        float amax = 1e-10f;
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(get(s[c][j]).x), fabsf(get(s[c][j]).y)));
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
        const float scale = amax * (1.0f / 448.0f);
        const F2 inverse = both(__fdividef(1.0f, scale));
        uint32_t packed[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          packed[j] = __nv_cvt_float2_to_fp8x2(get(mul2(s[c][2 * j], inverse)), __NV_SATFINITE, __NV_E4M3) |
                      static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(get(mul2(s[c][2 * j + 1], inverse)), __NV_SATFINITE, __NV_E4M3)) << 16;
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

// ---- Backward
//
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
#pragma unroll 8
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

// The backward kernels hold more per column: one group a thread up to 512 threads.
Shape backward_shape_of(int H) {
  const int groups = (H + 7) / 8;
  const int ch = groups <= kNormThreads ? 1 : groups <= 2 * kNormThreads ? 2 : 4;
  return {ch, ((groups + ch - 1) / ch + 31) / 32 * 32};
}

// How the rows of this call can be moved; for kEdges parameters need the activations' type too.
RowMode row_mode(const NormArgs& a, int dtype) {
  const int size = element_size(dtype), block = 16 / size;
  struct { const void* p; int64_t stride; int size; } const rows[] = {
      {a.x, a.x_stride, size}, {a.y, a.y_stride, size}, {a.gh, a.gh_stride, size}, {a.gs, a.gs_stride, size},
      {a.s, a.H, size}, {a.h, a.H, size}, {a.dx, a.H, size}, {a.dy, a.H, size},
      {a.gate_kind == kGateFull ? a.gate : nullptr, a.gate_stride, a.gate_f32 ? 4 : size},
      {a.gate_kind == kGateFull ? a.dgate_rows : nullptr, a.H, a.gate_f32 ? 4 : size}};
  bool all = a.H % 8 == 0, congruent = true, results = true;
  for (const auto& r : rows) {
    if (!r.p) continue;
    const bool base = aligned(r.p, 16);
    all = all && base && r.stride * r.size % 16 == 0;
    congruent = congruent && base && (r.stride - a.H) % block == 0 && r.size == size;
  }
  for (const void* p : {static_cast<const void*>(a.s), static_cast<const void*>(a.h), static_cast<const void*>(a.dx),
                        static_cast<const void*>(a.dy), a.gate_kind == kGateFull ? static_cast<const void*>(a.dgate_rows) : nullptr})
    results = results && aligned(p, 16);
  const bool params = aligned(a.pre_w, 16) && aligned(a.post_w, 16) && (a.gate_kind != kGateChannel || aligned(a.gate, 16));
  if (all && params && aligned(a.q, 8)) return kAligned;
  const bool own_type = size == 4 || !(a.pre_f32 || a.post_f32 || a.gate_f32);
  if (!own_type || a.q || !results || shape_of(a.H + 7).ch > 2) return kSpan;
  return congruent ? kEdges : kShifted;
}

// Width by which threads are counted: with edges a row has up to one block more.
int counted_width(int H, RowMode mode) { return has_edges(mode) ? H + 7 : H; }

bool bad_common(const NormArgs& a, int dtype, int param_f32) {
  if (dtype < MOE_B200_F32 || dtype > MOE_B200_F16) return true;
  const int size = element_size(dtype);
  const void* const rows[] = {a.x, a.y, a.gh, a.gs, a.s, a.h, a.dx, a.dy};
  for (const void* p : rows)
    if (!aligned(p, size)) return true;
  if (!aligned(a.pre_w, a.pre_f32 ? 4 : size) || !aligned(a.post_w, a.post_f32 ? 4 : size) || !aligned(a.gate, a.gate_f32 ? 4 : size))
    return true;
  return a.T < 0 || a.T > kMostTokens || a.H < 1 || a.H > kMaxWidth || (param_f32 & ~7) ||
         a.gate_kind < kGateNone || a.gate_kind > kGateFull || (a.gate_kind != kGateNone && (!a.gate || !a.y)) ||
         (a.post_w && !a.y);
}

constexpr size_t kSmemMost = 224 * 1024;          // dynamic shared memory a kernel here may have
constexpr size_t kRingMost = 208 * 1024;          // shared memory of an SM for rings; the rest is first-level cache

int grid_rows(int T, int per_sm, RowMode mode) {
  if (T <= kNumSMs * per_sm) return T;
  return has_edges(mode) ? kNumSMs * per_sm / 8 * 8 : kNumSMs * per_sm;
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

// CTAs of the backward pass, one partial row of column sums each: as many as the registers hold.
int backward_parts(int T, int H, RowMode mode) {
  const Shape sh = backward_shape_of(counted_width(H, mode));
  return grid_rows(T, sh.ch > 1 ? 1 : 512 / sh.threads, mode);
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
  if (!x || !pre_weight || !h || !rstd || !aligned(rstd, 8) || (y && !stream_out)) return MOE_B200_EINVAL;
  const RowMode mode = row_mode(a, dtype);
  if (h_scale && (H % kBlock != 0 || mode != kAligned)) return MOE_B200_EINVAL;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  cudaError_t e;
  if (dtype == MOE_B200_F32) e = launch_forward<float>(a, mode, stream);
  else if (dtype == MOE_B200_BF16) e = launch_forward<__nv_bfloat16>(a, mode, stream);
  else e = launch_forward<__half>(a, mode, stream);
  return launch_status(e, 1);
}

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
