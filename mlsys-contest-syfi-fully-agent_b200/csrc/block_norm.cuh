// What the forward and the backward of the block norms (block_norm.cu, block_norm_backward.cu) share: arguments, how rows are
// moved, rings, and the host's choice between the ways of moving rows.
#pragma once
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

// Threads and groups of eight columns per thread for a row of H columns.
struct Shape {
  int ch, threads;
};
inline Shape shape_of(int H) {
  const int groups = (H + 7) / 8;
  const int ch = groups <= 256 ? 1 : groups <= 2 * kNormThreads ? 2 : 4;
  return {ch, ((groups + ch - 1) / ch + 31) / 32 * 32};
}

// The backward kernels hold more per column: one group a thread up to 512 threads.
inline Shape backward_shape_of(int H) {
  const int groups = (H + 7) / 8;
  const int ch = groups <= kNormThreads ? 1 : groups <= 2 * kNormThreads ? 2 : 4;
  return {ch, ((groups + ch - 1) / ch + 31) / 32 * 32};
}

// How the rows of this call can be moved; for kEdges parameters need the activations' type too.
inline RowMode row_mode(const NormArgs& a, int dtype) {
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
inline int counted_width(int H, RowMode mode) { return has_edges(mode) ? H + 7 : H; }

inline bool bad_common(const NormArgs& a, int dtype, int param_f32) {
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

inline int grid_rows(int T, int per_sm, RowMode mode) {
  if (T <= kNumSMs * per_sm) return T;
  return has_edges(mode) ? kNumSMs * per_sm / 8 * 8 : kNumSMs * per_sm;
}
}  // namespace
}  // namespace moe
